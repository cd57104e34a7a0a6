// Losses over a vocabulary, and their gradients, without the logits in memory:
//
//     z[n, v] = x[n] . weight[v] / temperature,   lse[n] = log sum_v exp(z[n, v])
//     loss[n] = lse[n] - z[n, label[n]],  or  sum_k q[n, k] (log q[n, k] - z[n, word[n, k]] + lse[n])
//     G[n, v] = dloss[n] / temperature (exp(z[n, v] - lse[n]) - q[n, v]),   dx = G weight,   dweight = G' x
//
// The forward pass forms tiles of z and leaves of each the maximum and the sum of a token's exponentials and the
// logit of its label, or the sum of its targets' q z.  The backward pass goes over the vocabulary in pieces: a piece's part of G is formed from z again and kept,
// in the type of x, for the two products that read it.
#include <algorithm>
#include <optional>

#include "token_layout.h"

namespace {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr int kNoWord = 0x7fffffff;
constexpr int kMostTop = 256;
constexpr long long kMostRows = 1 << 20, kMostChannels = 1 << 20;

__device__ __forceinline__ long long word_at(const void* p, int wide, long long i) {
    return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// ------------------------------------------------------------------------- a teacher's shares
// A wave takes a row: shares of its entries, sorted by word, equal words added up, so that a tile finds its targets in one
// range and no element of G has two.  A logit is taken off the row's largest before the temperature divides it: the lowest
// value of 32 bits over a temperature below one would be -inf, which is no entry.
struct Shares {
    const void *words, *logits;
    int wide, logits_type, top, n_words;
    long long rows;
    float per_temperature;
    int* word;      // [rows, top], kNoWord behind the last
    float* share;
    float* self;    // sum q log q
    int* flag;      // 0: the row counts, -1: it has no entries
    unsigned short* first;  // [rows, blocks]: entries below the first word of each block of `block` words
    int blocks, block;
};

template <int Q> __global__ __launch_bounds__(NHIP_WG) void shares_kernel(Shares a) {
    constexpr int kMost = Q * NHIP_WAVE;
    __shared__ int s_word[4][kMost], s_sorted[4][kMost], s_merged[4][kMost];
    __shared__ float s_share[4][kMost], s_sorted_share[4][kMost];
    const int wave = threadIdx.x / NHIP_WAVE, lane = threadIdx.x % NHIP_WAVE;
    const long long row = (long long)blockIdx.x * 4 + wave, r = min(row, a.rows - 1);
    int id[Q];
    float t[Q];
    float most = -INFINITY;
    bool nan = false;
    int any = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int e = lane + q * NHIP_WAVE;
        id[q] = kNoWord;
        t[q] = -INFINITY;
        if (e < a.top) {
            const long long w = word_at(a.words, a.wide, r * a.top + e);
            const float v = sel_element(a.logits, a.logits_type, r * a.top + e);
            if (w >= 0 && w < a.n_words && !(v == -INFINITY)) {
                id[q] = (int)w;
                t[q] = v;
                any = 1;
            }
        }
        nan |= t[q] != t[q];
        most = fmaxf(most, t[q]);
    }
#pragma unroll
    for (int d = 1; d < NHIP_WAVE; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    any = __any(any);
    nan = __any(nan);
    float sum = 0.0f, x[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        t[q] = (t[q] - most) * a.per_temperature;
        x[q] = id[q] == kNoWord ? 0.0f : sel_exp(t[q]);
        sum += x[q];
    }
    sum = sel_wave_sum(sum);
    if (nan) sum = NAN;
    const float log_sum = logf(sum);
    float self = 0.0f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int e = lane + q * NHIP_WAVE;
        const float share = id[q] == kNoWord ? 0.0f : x[q] / sum;
        self += share == 0.0f ? 0.0f : share * (t[q] - log_sum);
        s_word[wave][e] = id[q];
        s_share[wave][e] = x[q] = share;
    }
    self = sel_wave_sum(self);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int e = lane + q * NHIP_WAVE;
        int rank = 0;
        for (int o = 0; o < kMost; ++o) {
            const int w = s_word[wave][o];
            rank += w < id[q] || (w == id[q] && o < e);
        }
        s_sorted[wave][rank] = id[q];
        s_sorted_share[wave][rank] = x[q];
    }
    __syncthreads();
    if (row >= a.rows) return;  // (a wave: what follows is within waves, whose LDS accesses stay in their order)
    int before = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int e = lane + q * NHIP_WAVE, w = s_sorted[wave][e];
        const bool first = w != kNoWord && (e == 0 || s_sorted[wave][e - 1] != w);
        const unsigned long long all = __ballot(first);
        if (first) {
            float share = s_sorted_share[wave][e];
            for (int o = e + 1; o < kMost && s_sorted[wave][o] == w; ++o) share += s_sorted_share[wave][o];
            const int at = before + __popcll(all & ((1ULL << lane) - 1));
            s_merged[wave][at] = w;
            a.word[row * a.top + at] = w;
            a.share[row * a.top + at] = share;
        }
        before += __popcll(all);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int e = lane + q * NHIP_WAVE;
        if (e >= before && e < a.top) {
            a.word[row * a.top + e] = kNoWord;
            a.share[row * a.top + e] = 0.0f;
        }
    }
    if (lane == 0) {
        a.self[row] = self;
        a.flag[row] = any ? 0 : -1;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int b = lane; b < a.blocks; b += NHIP_WAVE) {
        int lo = 0, hi = before;  // (b times block stays below 2^31: so do the words)
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (s_merged[wave][mid] < b * a.block) lo = mid + 1;
            else hi = mid;
        }
        a.first[row * a.blocks + b] = (unsigned short)lo;
    }
}

// ------------------------------------------------------------------------------ rows that count
// The rows whose label is a word move together, rows of whole stages.  A group takes some rows and counts those before them itself
// (8192 labels are 64 KB in the L2; a launch of its own for the sums would take longer).
struct Gather {
    const void *x, *labels;
    int wide_labels, n_words, type, wide;
    long long ld, rows;
    int channels, out_ld;
    void* out;
    int *row, *where, *label, *count;  // [rows padded], [rows], [rows padded], 1
    float *loss, *lse;                 // zeros where a row does not count; NULL in the backward pass
    int per;                           // rows of a group
};
constexpr int kMostPer = 1024;
// Rows of a group: as few as give every compute unit some, more where counting would cost more than moving
int gather_rows(long long rows) { return rows <= 1024 * 8 ? 8 : rows <= 1024 * 64 ? 64 : kMostPer; }
static_assert(kMostRows <= 1024 * kMostPer, "");

template <class T> __global__ __launch_bounds__(NHIP_WG) void gather_kernel(Gather a) {
    constexpr int V = 16 / (int)sizeof(T);
    __shared__ int s_sum[4], s_at[kMostPer];
    const int wave = threadIdx.x / NHIP_WAVE, lane = threadIdx.x % NHIP_WAVE;
    const long long r0 = (long long)blockIdx.x * a.per;
    auto label_of = [&](long long r) {
        const long long w = word_at(a.labels, a.wide_labels, r);
        return w >= 0 && w < a.n_words ? (int)w : -1;
    };
    int sum = 0;
    for (long long r = threadIdx.x; r < r0; r += 8 * NHIP_WG) {
        int some[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) some[e] = label_of(min(r + e * NHIP_WG, r0 - 1));
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += some[e] >= 0 && r + e * NHIP_WG < r0;
    }
#pragma unroll
    for (int d = 1; d < NHIP_WAVE; d *= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    if (wave == 0) {
        int before = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        for (int k = lane; k < a.per; k += NHIP_WAVE) {
            const long long r = r0 + k;
            const int label = r < a.rows ? label_of(r) : -1;
            const unsigned long long all = __ballot(label >= 0);
            const int at = before + __popcll(all & ((1ULL << lane) - 1));
            s_at[k] = label >= 0 ? at : -1;
            if (label >= 0) {
                a.row[at] = (int)r;
                a.label[at] = label;
            }
            if (r < a.rows) {
                a.where[r] = label >= 0 ? at : -1;
                if (a.loss && label < 0) a.loss[r] = a.lse[r] = 0.0f;
            }
            before += __popcll(all);
        }
        if (blockIdx.x == gridDim.x - 1 && lane == 0) *a.count = before;
    }
    __syncthreads();
    if (r0 >= a.rows) return;
    // loads are unconditional, from places that exist: those under a condition are waited for one by one
    const int packs = a.out_ld / V, all = a.per * packs;
    for (int q = threadIdx.x; q < all; q += 4 * NHIP_WG) {
        SelPack<T, V> v[4];
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            const int k = min(q + o * NHIP_WG, all - 1), c = k % packs * V;
            const T* const from = static_cast<const T*>(a.x) + min(r0 + k / packs, a.rows - 1) * a.ld;
            if (a.wide && a.channels % V == 0) {
                v[o] = *reinterpret_cast<const SelPack<T, V>*>(from + min(c, a.channels - V));
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) v[o].v[e] = from[min(c + e, a.channels - 1)];
            }
        }
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            const int k = q + o * NHIP_WG, c = k % packs * V;
            const int at = k < all ? s_at[k / packs] : -1;
            if (at < 0) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) v[o].v[e] = c + e < a.channels ? v[o].v[e] : (T)0.0f;
            *reinterpret_cast<SelPack<T, V>*>(static_cast<T*>(a.out) + (long long)at * a.out_ld + c) = v[o];
        }
    }
}

// What G is scaled by in 16 bits, and the reverse: `most` over the largest magnitude of the tokens' dloss.  Where all tokens have
// the same one (a mean), the targets' elements, p - 1 times one, lose next to nothing when they are rounded; and
// in float16 (2^14) the gradient of a mean over many tokens stays in the type's range.
__global__ __launch_bounds__(1024) void scale_kernel(const float* dloss, const int* where, long long rows, float per_temperature,
                                                     float most, float* scale) {
    __shared__ float s[16];
    float top = 0.0f;
    for (long long r = threadIdx.x; r < rows; r += 4 * 1024) {
        float v[4];
        int at[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = dloss[min(r + e * 1024, rows - 1)];
            at[e] = where[min(r + e * 1024, rows - 1)];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float m = fabsf(v[e] * per_temperature);
            if (at[e] >= 0 && m < INFINITY) top = fmaxf(top, m);
        }
    }
#pragma unroll
    for (int d = 1; d < NHIP_WAVE; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    if (threadIdx.x % NHIP_WAVE == 0) s[threadIdx.x / NHIP_WAVE] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) top = fmaxf(top, s[w]);
        top = top > 0.0f ? fminf(fmaxf(top, 0x1p-100f), 0x1p100f) : most;
        scale[0] = most / top;
        scale[1] = top / most;
    }
}

// ----------------------------------------------------------------------------------- tiles of z
struct Targets {
    const void* label;  // [live], or
    const int* word;    // [rows, top], sorted, with
    const float* share;
    const int* row;     // of a live token; NULL: tokens are rows, of which not all count
    const unsigned short* first;
    int top, blocks, block, wide_label, n_words;
    const int* flag;    // [rows] with `row` NULL and a teacher: below zero where a row does not count
    __device__ __forceinline__ int row_of(long long n) const { return row ? row[n] : (int)n; }
    __device__ __forceinline__ int label_of(long long n) const {  // -1: the token does not count
        const long long w = word_at(label, wide_label, n);
        return w >= 0 && w < n_words ? (int)w : -1;
    }
    // where the entries of words w0 ... w1 - 1 (and some around them, to whole blocks) begin and end among a row's
    __device__ __forceinline__ void range(long long r, int w0, int w1, int& lo, int& hi) const {
        const unsigned short* const of = first + r * blocks;
        lo = of[min(w0 / block, blocks - 1)];
        hi = of[min((w1 + block - 1) / block, blocks - 1)];
    }
};

// Forward: of each token in the tile the maximum of z and the sum of exp(z - maximum), in powers of two, and the logit of
// its label, or the sum of its targets' q z.  (4096 tokens, 32000 words, 64 of them targets, 1024 channels: without targets the
// kernel would take 45 us less of 265.  A wave waits for row, range and first target, one after the other; loaded while
// the tile is multiplied they need registers that there are not: 13 spilled, 60 us more.)
template <bool TOP> struct Statistics {
    Targets targets;
    float2* part;      // [tiles of the whole vocabulary, ld]
    float* picked;     // [live]: the label's logit; of each tile the sum of shares and logits of a teacher's targets, as `part`
    long long ld;
    int words, word0, tile0;  // words of the piece, its first word, its first tile
    float per_temperature;

    template <class T, class S> __device__ __forceinline__ void run(const TokPlace& at, sel_f4 (&acc)[S::MI][S::NI]) const {
        float2* const s_part = reinterpret_cast<float2*>(at.lds);  // [WM][BN]
        float* const s_picked = reinterpret_cast<float*>(s_part + S::WM * S::BN);
        static_assert(12 * S::WM * S::BN <= S::kEpilogue, "");
        const long long n0 = (long long)at.n_tile * S::BN;
        const int m0 = at.m_tile * S::BM + at.wave_m * S::kWaveM + 4 * at.g;  // within the piece
        const int w0 = word0 + at.m_tile * S::BM + at.wave_m * S::kWaveM;
        if (S::WM > 1) __syncthreads();  // (the tile before is done with the LDS)
        const float c = kLog2e * per_temperature;
        // what the tokens have, before it is needed: loads under a condition are waited for one by one
        int lo[S::NI], hi[S::NI], row[S::NI], word[S::NI];
        float share[S::NI];
        auto token = [&](int j) { return n0 + at.wave_n * S::kWaveN + 16 * j + at.l; };
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            const long long n = min(token(j), at.live - 1LL);
            row[j] = TOP ? targets.row_of(n) : targets.label_of(n);
        }
        if constexpr (TOP) {
#pragma unroll
            for (int j = 0; j < S::NI; ++j) targets.range(row[j], w0, w0 + S::kWaveM, lo[j], hi[j]);
#pragma unroll
            for (int j = 0; j < S::NI; ++j) {
                const long long e = (long long)row[j] * targets.top + min(lo[j], targets.top - 1);
                word[j] = targets.word[e];
                share[j] = targets.share[e];
            }
        }
        auto go = [&](auto whole) {
            auto is = [&](int i, int r) { return decltype(whole)::value || m0 + 16 * i + r < words; };
#pragma unroll
            for (int j = 0; j < S::NI; ++j) {
                const int local = at.wave_n * S::kWaveN + 16 * j + at.l;
                const long long n = n0 + local;
                float most = -INFINITY;
#pragma unroll
                for (int i = 0; i < S::MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) most = is(i, r) ? fmaxf(most, acc[i][j][r]) : most;
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                float top2 = most * c;
                if (!(fabsf(top2) < INFINITY)) top2 = 0.0f;  // (infinities then reach the sum as they are)
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < S::MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], c, -top2));
                        sum += is(i, r) ? e : 0.0f;
                    }
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
                if constexpr (S::WM > 1) {
                    if (at.g == 0) s_part[at.wave_m * S::BN + local] = float2{top2, sum};
                } else {
                    if (at.g == 0 && n < at.live) part[(long long)(tile0 + at.m_tile) * ld + n] = float2{top2, sum};
                }
            }
        };
        if ((at.m_tile + 1) * S::BM <= words) go(std::true_type());
        else go(std::false_type());
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            const long long n = token(j);
            auto is_mine = [&](int rel) { return rel >= 0 && rel < S::kWaveM && (rel & 15) < 4; };
            auto logit = [&](int rel) {
                float z = 0.0f;
#pragma unroll
                for (int i = 0; i < S::MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z = rel == 16 * i + r ? acc[i][j][r] : z;
                return z * per_temperature;
            };
            if constexpr (TOP) {
                float sum = 0.0f;
                // (the first target's loads are under no condition: the compiler would wait for each of them)
                asm volatile("" : "+v"(word[j]), "+v"(share[j]));
                const long long from = (long long)row[j] * targets.top;
                float q = n < at.live && lo[j] < hi[j] ? share[j] : 0.0f;
                int rel = word[j] - word0 - m0;
                for (int k = lo[j];;) {
                    if (!is_mine(rel)) q = 0.0f;
                    if (__any(q != 0.0f)) sum = q != 0.0f ? fmaf(q, logit(rel), sum) : sum;
                    const bool more = n < at.live && ++k < hi[j];
                    if (!__any(more)) break;
                    q = more ? targets.share[from + k] : 0.0f;
                    rel = more ? targets.word[from + k] - word0 - m0 : -1;
                }
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
                if (at.g == 0) {
                    if (S::WM > 1) s_picked[at.wave_m * S::BN + (int)(n - n0)] = sum;
                    else if (n < at.live) picked[(long long)(tile0 + at.m_tile) * ld + n] = sum;
                }
            } else if (n < at.live && is_mine(row[j] - word0 - m0)) {
                picked[n] = logit(row[j] - word0 - m0);
            }
        }
        if constexpr (S::WM > 1) {
            __syncthreads();
            for (int k = threadIdx.x; k < S::BN; k += S::kThreads) {
                float2 a = s_part[k];
                float sum = TOP ? s_picked[k] : 0.0f;
#pragma unroll
                for (int w = 1; w < S::WM; ++w) {
                    a = joined(a, s_part[w * S::BN + k]);
                    if (TOP) sum += s_picked[w * S::BN + k];
                }
                if (n0 + k >= at.live) continue;
                part[(long long)(tile0 + at.m_tile) * ld + n0 + k] = a;
                if (TOP) picked[(long long)(tile0 + at.m_tile) * ld + n0 + k] = sum;
            }
        }
    }
    // of two parts, neither of which is more than infinite
    static __device__ __forceinline__ float2 joined(float2 a, float2 b) {
        if (b.y == 0.0f) return a;
        if (a.y == 0.0f) return b;
        const float top = fmaxf(a.x, b.x);
        const float x = a.y == INFINITY ? a.y : a.y * __builtin_amdgcn_exp2f(a.x - top);
        const float y = b.y == INFINITY ? b.y : b.y * __builtin_amdgcn_exp2f(b.x - top);
        return float2{top, x + y};
    }
};

// loss and lse of the live tokens: 64 lanes to a token
constexpr int kFinishLanes = 64;
struct Finish {
    const float2* part;
    const float* picked;
    Targets targets;
    const float* self;
    const int* count;  // NULL: `rows`
    long long ld;
    int tiles, rows;
    float *loss, *lse;
};

__global__ __launch_bounds__(16 * kFinishLanes) void finish_kernel(Finish a) {
    __shared__ float3 s[16][16];
    const int k = threadIdx.x % 16, q = threadIdx.x / 16, live = a.count ? *a.count : a.rows;
    if ((long long)blockIdx.x * 16 >= live) return;
    const int n = min((int)blockIdx.x * 16 + k, live - 1), row = a.targets.row_of(n);
    const bool is = a.targets.row || (a.targets.top ? a.targets.flag[n] : a.targets.label_of(n)) >= 0;
    float2 v = {0.0f, 0.0f};
    float loss = 0.0f;  // sum q z
    for (int t = q; t < a.tiles; t += 8 * kFinishLanes) {
        float2 some[8];
        float z[8];
#pragma unroll
        for (int o = 0; o < 8; ++o) {
            const long long at = (long long)min(t + o * kFinishLanes, a.tiles - 1) * a.ld + n;
            some[o] = a.part[at];
            z[o] = a.targets.top ? a.picked[at] : 0.0f;
        }
#pragma unroll
        for (int o = 0; o < 8; ++o)
            if (t + o * kFinishLanes < a.tiles) {
                v = Statistics<false>::joined(v, some[o]);
                loss += z[o];
            }
    }
    // four lanes of a wave have one token, then 16 waves; always in the same order
    auto join = [&](int d) {
        v = Statistics<false>::joined(v, float2{__shfl_xor(v.x, d), __shfl_xor(v.y, d)});
        loss += __shfl_xor(loss, d);
    };
    join(16);
    join(32);
    if (q % 4 == 0) s[q / 4][k] = float3{v.x, v.y, loss};
    __syncthreads();
    if (threadIdx.x >= NHIP_WAVE) return;
    v = float2{s[q][k].x, s[q][k].y};
    loss = s[q][k].z;
#pragma unroll
    for (int o = 4; o < 16; o += 4) {
        v = Statistics<false>::joined(v, float2{s[q + o][k].x, s[q + o][k].y});
        loss += s[q + o][k].z;
    }
    join(16);
    join(32);
    if (q || (int)blockIdx.x * 16 + k >= live) return;
    const float lse = (v.x + __builtin_amdgcn_logf(v.y)) * kLn2;
    a.loss[row] = !is ? 0.0f : a.targets.top ? a.self[row] + (lse - loss) : lse - a.picked[n];  // (the shares' sum is one)
    a.lse[row] = is ? lse : 0.0f;
}

// Backward: G of the tile, rounded to the type of x, in which the matrix cores multiply it with x and the weights: once, to half a
// step, of numbers that `scale` brings near one (in float16 to its range).  A gradient in bfloat16 is off by 0.0022 to 0.0023 of its
// norm for it, where the rounding of the result makes 0.0017; G in two parts would save that and double two of the three products.
template <bool TOP> struct Gradient {
    Targets targets;
    const float *dloss, *lse, *scale;
    void *g, *gt;             // [live, g_ld], [words, gt_ld] (or NULL)
    long long g_ld, gt_ld;
    int words, word0;
    float per_temperature;

    template <class T, class S> __device__ __forceinline__ void run(const TokPlace& at, sel_f4 (&acc)[S::MI][S::NI]) const {
        const long long n0 = (long long)at.n_tile * S::BN;
        const int m0 = at.m_tile * S::BM + at.wave_m * S::kWaveM + 4 * at.g, w0 = word0 + at.m_tile * S::BM + at.wave_m * S::kWaveM;
        const float c = kLog2e * per_temperature, k = scale ? *scale * per_temperature : per_temperature;
        // what the tokens have, before it is needed: loads under a condition are waited for one by one
        int row[S::NI], label[S::NI], lo[S::NI], hi[S::NI];
        float d[S::NI], lse2[S::NI];
        auto token = [&](int j) { return n0 + at.wave_n * S::kWaveN + 16 * j + at.l; };
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            row[j] = targets.row_of(min(token(j), at.live - 1LL));
            if constexpr (!TOP) label[j] = targets.label_of(min(token(j), at.live - 1LL));
        }
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            d[j] = dloss[row[j]] * k;
            lse2[j] = lse[row[j]] * kLog2e;
            if constexpr (TOP) targets.range(row[j], w0, w0 + S::kWaveM, lo[j], hi[j]);
        }
        // of a teacher's targets in the tile the first is taken before the element is stored: most tiles have no second of a token
        // (4096 tokens, 32000 words, 64 of them targets, 1024 channels: 697 us; 680 so, 687 with two)
        constexpr int kTaken = TOP ? 1 : 0;
        int place[S::NI][kTaken + 1];
        float share[S::NI][kTaken + 1];
#pragma unroll
        for (int j = 0; j < S::NI; ++j)
#pragma unroll
            for (int t = 0; t < kTaken; ++t) {
                const long long e = (long long)row[j] * targets.top + min(lo[j] + t, targets.top - 1);
                place[j][t] = lo[j] + t < hi[j] ? targets.word[e] - word0 - m0 : -1;
                share[j][t] = targets.share[e] * d[j];
            }
        const bool whole = (at.m_tile + 1) * S::BM <= words;
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            const long long n = token(j);
            const bool counts = n < at.live;
            int taken = 0;  // of the wave: so many targets at most has a token of the column
#pragma unroll
            for (int t = 0; t < kTaken; ++t) {
                if (!counts) place[j][t] = -1;
                if (__any(place[j][t] >= 0 && place[j][t] < S::kWaveM)) taken = t + 1;
            }
            auto value = [&](int i, float(&v)[4]) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = d[j] * __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], c, -lse2[j]));
                    v[r] = counts && (whole || m0 + 16 * i + r < words) ? p : 0.0f;
                }
#pragma unroll
                for (int t = 0; t < kTaken; ++t)
                    if (t < taken) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] -= place[j][t] == 16 * i + r ? share[j][t] : 0.0f;
                    }
            };
            bool stored = false;
            if constexpr (sizeof(T) == 2 && S::MI % 4 == 0) {
                if (!gt) {
                    stored = true;
#pragma unroll
                    for (int i = 0; i < S::MI; i += 4)
                        tok_put<T>(at, static_cast<T*>(g) + (n - at.l) * g_ld + m0 - 4 * at.g + 16 * i, g_ld, 16, 64,
                                   [&](int e, float(&v)[4]) { value(i + e, v); });
                }
            }
            if (!stored) {
#pragma unroll
                for (int i = 0; i < S::MI; ++i) {
                    float v[4];
                    value(i, v);
                    tok_store_both<T>(static_cast<T*>(g), g_ld, static_cast<T*>(gt), gt_ld, n, m0 + 16 * i, v);
                }
            }
            // the targets' elements once more, when what the wave has stored there has arrived
            auto take = [&](int word, float share) {
                const int rel = word - word0 - m0;
                if (rel < 0 || rel >= S::kWaveM || (rel & 15) >= 4) return;
                float z = 0.0f;
#pragma unroll
                for (int i = 0; i < S::MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z = rel == 16 * i + r ? acc[i][j][r] : z;
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                const T v = (T)(d[j] * (__builtin_amdgcn_exp2f(fmaf(z, c, -lse2[j])) - share));
                static_cast<T*>(g)[n * g_ld + m0 + rel] = v;
                if (gt) static_cast<T*>(gt)[(m0 + rel) * gt_ld + n] = v;
            };
            if (counts) {
                if constexpr (TOP) {
                    const long long from = (long long)row[j] * targets.top;
                    for (int e = lo[j] + kTaken; e < hi[j]; ++e) take(targets.word[from + e], targets.share[from + e]);
                } else {
                    take(label[j], 1.0f);
                }
            }
        }
    }
};

// --------------------------------------------------------------------------------------- host
int check(const nhip_loss_args* a) {
    if (!a || a->channels <= 0 || a->words <= 0 || a->rows < 0 || a->top < 0) return NHIP_E_BADARG;
    if (a->type < NHIP_F32 || a->type > NHIP_F16 || a->rows > kMostRows || a->top > kMostTop) return NHIP_E_BADARG;
    if (a->top && (a->logits_type < NHIP_F32 || a->logits_type > NHIP_F16)) return NHIP_E_BADARG;
    if (!(a->temperature >= 0x1p-126f) || !(a->temperature <= 0x1p126f)) return NHIP_E_BADARG;  // (its reciprocal is one of 32 bits)
    if (a->words > kNoWord - 4096 || a->channels > kMostChannels) return NHIP_E_BADARG;
    return 0;
}

bool wide_weight(const nhip_loss_args& a) {
    const long long size = sel_size(a.type);
    return tok_rows_wide(a.weight, a.weight_stride * size, a.channels * size);
}

struct Space : TokSpace {
    long long padded, x_ld, piece;
    long long row, where, label, count, flag, word, share, self, first, blocks, block, x, weight, part, picked;
    std::optional<TokGradient> gradient;
    Space(const nhip_loss_args& a, bool grad) {
        const long long size = sel_size(a.type), rows = a.rows > 0 ? a.rows : 1, top = a.top;
        padded = tok_round(rows, TOK_MOST_TILE);
        x_ld = tok_round(a.channels, 64);
        row = take(padded * 4);
        where = take(rows * 4);
        label = take(padded * 4);
        count = take(256);
        flag = word = share = self = first = blocks = block = 0;
        if (top) {
            flag = take(rows * 4);
            word = take(rows * top * 4);
            share = take(rows * top * 4);
            self = take(rows * 4);
            // as fine as the tiles: those of the kernels for few columns, or of the others
            block = !grad && a.rows <= TOK_FEW ? TOK_LEAST_BM : 128;
            blocks = (a.words + block - 1) / block + 1;  // (the last one: all entries)
            first = take(rows * blocks * 2);
        }
        x = take(padded * x_ld * size);
        if (grad) {
            gradient.emplace(*this, a.rows, a.channels, a.words, size);
            piece = gradient->piece;
        } else {
            // as many words as a launch's tiles reach (256 tokens: 2^28), and where they are copied as fit 512 MB
            piece = (1LL << 21) / (padded / 256) * 128;
            if (!wide_weight(a)) piece = std::min(piece, std::max(256LL, (512LL << 20) / (x_ld * size) / 256 * 256));
            piece = std::min(piece, tok_round(a.words, 256));
            const long long tiles = tok_round(a.words, piece) / (a.rows <= TOK_FEW ? TOK_LEAST_BM : 128);
            part = take(tiles * padded * 8);
            picked = take((top ? tiles : 1) * padded * 4);
        }
        weight = wide_weight(a) ? 0 : take(piece * x_ld * size);
    }
};

#define TOK_TRY(call) do { if (int e_ = (call)) return e_; } while (0)

// The rows that count (or all, as they are), and the targets of all rows
template <class T>
int prepare(hipStream_t st, const nhip_loss_args& a, const Space& s, char* w, bool grad, bool as_they_are, Targets& t) {
    t = Targets{w + s.label, reinterpret_cast<int*>(w + s.word), reinterpret_cast<float*>(w + s.share),
                reinterpret_cast<int*>(w + s.row), reinterpret_cast<unsigned short*>(w + s.first), a.top, (int)s.blocks, (int)s.block,
                0, a.words, reinterpret_cast<int*>(w + s.flag)};
    Gather gather{a.x, a.targets, a.wide_targets, a.words, a.type, 0, a.x_stride, a.rows, a.channels, (int)s.x_ld, w + s.x,
                  reinterpret_cast<int*>(w + s.row), reinterpret_cast<int*>(w + s.where), reinterpret_cast<int*>(w + s.label),
                  reinterpret_cast<int*>(w + s.count), grad ? nullptr : a.loss, grad ? nullptr : a.lse, gather_rows(a.rows)};
    gather.wide = tok_rows_wide(a.x, a.x_stride * (long long)sizeof(T), 16);
    if (a.top && a.rows) {
        Shares sh{a.targets, a.target_logits, a.wide_targets, a.logits_type, a.top, a.words, a.rows, 1.0f / a.temperature,
                  reinterpret_cast<int*>(w + s.word), reinterpret_cast<float*>(w + s.share), reinterpret_cast<float*>(w + s.self),
                  reinterpret_cast<int*>(w + s.flag), reinterpret_cast<unsigned short*>(w + s.first), (int)s.blocks, (int)s.block};
        const dim3 grid((unsigned)((a.rows + 3) / 4));
        if (a.top <= 64) TOK_LAUNCH(false, (shares_kernel<1>), grid, dim3(NHIP_WG), 0, st, sh);
        else if (a.top <= 128) TOK_LAUNCH(false, (shares_kernel<2>), grid, dim3(NHIP_WG), 0, st, sh);
        else TOK_LAUNCH(false, (shares_kernel<4>), grid, dim3(NHIP_WG), 0, st, sh);
        NHIP_LAUNCH_CHECK();
        gather.labels = w + s.flag;  // 0 or -1
        gather.wide_labels = 0;
    }
    if (as_they_are) {
        t.row = nullptr;
        t.label = a.targets;
        t.wide_label = a.wide_targets;
        return 0;
    }
    const long long groups = (a.rows + gather.per - 1) / gather.per;
    TOK_LAUNCH(false, (gather_kernel<T>), dim3((unsigned)(groups ? groups : 1)), dim3(NHIP_WG), 0, st, gather);
    NHIP_LAUNCH_CHECK();
    return 0;
}

// The rows of a piece of the weights as the products read them
template <class T> int piece_rows(hipStream_t st, const nhip_loss_args& a, const Space& s, char* w, long long v0, long long words,
                                  TokRows& rows) {
    const T* const from = static_cast<const T*>(a.weight) + v0 * a.weight_stride;
    rows = TokRows{reinterpret_cast<const char*>(from), nullptr, a.weight_stride * (long long)sizeof(T), words};
    if (s.weight) {
        TOK_TRY(tok_pad<T>(st, TokPad{from, a.weight_stride, w + s.weight, s.x_ld, words, a.channels}));
        rows.p = w + s.weight;
        rows.ld = s.x_ld * (long long)sizeof(T);
    }
    return 0;
}

template <class T> int forward(hipStream_t st, const nhip_loss_args& a, const Space& s) {
    char* const w = static_cast<char*>(a.workspace);
    Targets t;
    // few rows are computed all, where they lie: to bring together those that count would take a launch
    const bool all = a.rows <= TOK_FEW && tok_rows_wide(a.x, a.x_stride * (long long)sizeof(T), a.channels * (long long)sizeof(T));
    TOK_TRY(prepare<T>(st, a, s, w, false, all, t));
    const int* const count = all ? nullptr : reinterpret_cast<int*>(w + s.count);
    const TokRows x = all ? TokRows{static_cast<const char*>(a.x), nullptr, a.x_stride * (long long)sizeof(T), a.rows}
                          : TokRows{w + s.x, nullptr, s.x_ld * (long long)sizeof(T), a.rows};
    int tiles = 0;
    for (long long v0 = 0; v0 < a.words; v0 += s.piece) {
        const long long words = a.words - v0 < s.piece ? a.words - v0 : s.piece;
        TokRows rows;
        TOK_TRY(piece_rows<T>(st, a, s, w, v0, words, rows));
        TokProduct p{rows, x, count, nullptr, a.channels * (long long)sizeof(T), 0, 0, 1};
        auto go = [&](auto top) {
            Statistics<decltype(top)::value> e{t, reinterpret_cast<float2*>(w + s.part), reinterpret_cast<float*>(w + s.picked),
                                               s.padded, (int)words, (int)v0, tiles, 1.0f / a.temperature};
            if (a.rows <= TOK_FEW) {
                tiles += (int)((words + TOK_LEAST_BM - 1) / TOK_LEAST_BM);
                return tok_few<T, TOK_LEAST_BM / 16, 0>(st, p, e);
            }
            return tok_with_many(words, a.rows, sizeof(T), 1, [&](auto shape) {
                using S = decltype(shape);
                p.m_tiles = (int)((words + S::BM - 1) / S::BM);
                p.n_tiles = (int)((a.rows + S::BN - 1) / S::BN);
                tiles += p.m_tiles;
                return tok_product<T, S, 0>(st, p, e);
            });
        };
        TOK_TRY(a.top ? go(std::true_type()) : go(std::false_type()));
    }
    if (!a.rows) return 0;
    Finish f{reinterpret_cast<float2*>(w + s.part), reinterpret_cast<float*>(w + s.picked), t, reinterpret_cast<float*>(w + s.self),
             count, s.padded, tiles, (int)a.rows, a.loss, a.lse};
    TOK_LAUNCH(true, finish_kernel, dim3((unsigned)((a.rows + 15) / 16)), dim3(16 * kFinishLanes), 0, st, f);
    NHIP_LAUNCH_CHECK();
    return 0;
}

template <class T> int backward(hipStream_t st, const nhip_loss_args& a, const Space& s) {
    constexpr long long size = sizeof(T);
    char* const w = static_cast<char*>(a.workspace);
    Targets t;
    TOK_TRY(prepare<T>(st, a, s, w, true, false, t));
    const int* const count = reinterpret_cast<int*>(w + s.count);
    const TokGradient& gr = *s.gradient;
    TOK_TRY(gr.lay_out_x<T>(st, w, w + s.x, s.x_ld, count));
    float* scale = nullptr;
    if (sizeof(T) == 2 && a.rows) {
        scale = reinterpret_cast<float*>(w + s.count) + 16;
        TOK_LAUNCH(false, scale_kernel, dim3(1), dim3(1024), 0, st, a.dloss, reinterpret_cast<int*>(w + s.where), a.rows,
                    1.0f / a.temperature, std::is_same<T, _Float16>::value ? 0x1p14f : 1.0f, scale);
        NHIP_LAUNCH_CHECK();
    }
    const long long d = a.channels;
    for (long long v0 = 0; v0 < a.words; v0 += s.piece) {
        const long long words = a.words - v0 < s.piece ? a.words - v0 : s.piece;
        TokRows rows;
        TOK_TRY(piece_rows<T>(st, a, s, w, v0, words, rows));
        const TokRows x{w + s.x, nullptr, s.x_ld * size, a.rows};
        TOK_TRY(tok_with_shape(words, a.rows, sizeof(T), 1, [&](auto shape) {
            using S = decltype(shape);
            TokProduct p{rows, x, count, nullptr, d * size,
                         (int)((words + S::BM - 1) / S::BM), (int)((a.rows + S::BN - 1) / S::BN), 1};
            auto go = [&](auto top) {
                Gradient<decltype(top)::value> e{t, a.dloss, a.lse, scale, w + gr.g, gr.gt_of<T>(w), gr.g_ld, gr.gt_ld, (int)words, (int)v0,
                                                 1.0f / a.temperature};
                return tok_product<T, S, 0>(st, p, e);
            };
            return a.top ? go(std::true_type()) : go(std::false_type());
        }));
        TOK_TRY(gr.weights<T>(st, w, x, count, words, words, 0, static_cast<T*>(a.dweight) + v0 * d, static_cast<T*>(nullptr),
                              scale ? scale + 1 : nullptr));
        TOK_TRY(gr.inputs<T>(st, w, rows, count, words, words, 0, v0 > 0));
    }
    return gr.finish<T>(st, w, reinterpret_cast<int*>(w + s.where), count, scale ? scale + 1 : nullptr, a.dx);
}

int run(void* stream, const nhip_loss_args* args, bool grad) {
    if (int e = check(args)) return e;
    const nhip_loss_args& a = *args;
    if (!a.weight || (a.rows && (!a.x || !a.targets || (a.top && !a.target_logits) || !a.lse))) return NHIP_E_BADARG;
    if (grad ? !a.dweight || (a.rows && (!a.dloss || !a.dx)) : a.rows && !a.loss) return NHIP_E_BADARG;
    const Space s(a, grad);
    if (s.bytes > a.workspace_bytes) return NHIP_E_TOOBIG;
    if (!a.workspace || !sel_aligned(a.workspace, 256)) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        rc = grad ? backward<T>(static_cast<hipStream_t>(stream), a, s) : forward<T>(static_cast<hipStream_t>(stream), a, s);
    });
    return tok_end(static_cast<hipStream_t>(stream), rc);
}

}  // namespace

extern "C" int nhip_vocabulary_loss_workspace(const nhip_loss_args* args, long long* bytes_out) {
    if (int e = check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    *bytes_out = Space(*args, false).bytes;
    return 0;
}

extern "C" int nhip_vocabulary_loss(void* stream, const nhip_loss_args* args) { return run(stream, args, false); }

extern "C" int nhip_vocabulary_loss_grad_workspace(const nhip_loss_args* args, long long* bytes_out) {
    if (int e = check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    *bytes_out = Space(*args, true).bytes;
    return 0;
}

extern "C" int nhip_vocabulary_loss_grad(void* stream, const nhip_loss_args* args) { return run(stream, args, true); }
