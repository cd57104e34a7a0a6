// The matrix product behind the operators over tokens (gated projection, losses over a vocabulary):
//
//     D[m, n] = sum_k A[m, k] B[n, k],     rows of A and B along k, sums in 32 bits
//
// and what becomes of D is the caller's: an epilogue gets it in registers.  A work-group forms a tile of BM x BN; tiles of A
// and B of 128 bytes along k (a stage) go straight from memory into one of two places in the LDS.  While half a stage is
// multiplied the next half is read into registers; a place is filled again as soon as it has been read.
//
// D lies as the matrix instructions leave it: tile (i, j) of 16 x 16 of a wave holds column n = 16 j + lane % 16 and
// rows m = 16 i + 4 (lane / 16) + r in its four registers.  So m runs along what is contiguous in the result, and a
// reduction over m (the softmax over a vocabulary) is one within a lane, up to four lanes.
#pragma once

#include <type_traits>

#include "selective_common.h"

typedef unsigned tok_u4 __attribute__((ext_vector_type(4)));
typedef __bf16 tok_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 tok_h8 __attribute__((ext_vector_type(8)));
typedef __bf16 sel_b4 __attribute__((ext_vector_type(4)));

// An entry point's first launch carries the start event, the one that is known to be its last (`last`) the stop event; where that
// is not launched (no rows) the stop event is recorded behind the others.
#define TOK_LAUNCH(last, kernel, grid, block, lds, stream, ...)                              \
    do {                                                                                     \
        const hipEvent_t start_ = nhip_launch_events.start;                                  \
        const hipEvent_t stop_ = (last) ? nhip_launch_events.stop : nullptr;                 \
        if (start_ || stop_) {                                                               \
            nhip_launch_events = NhipLaunchEvents{nullptr, stop_ ? nullptr : nhip_launch_events.stop}; \
            hipExtLaunchKernelGGL(kernel, grid, block, lds, stream, start_, stop_, 0, __VA_ARGS__);    \
        } else {                                                                             \
            hipLaunchKernelGGL(kernel, grid, block, lds, stream, __VA_ARGS__);               \
        }                                                                                    \
    } while (0)
static inline int tok_end(hipStream_t stream, int rc) {
    const NhipLaunchEvents left = nhip_launch_events;
    if (left.start || !left.stop) return rc;
    nhip_launch_events = NhipLaunchEvents{nullptr, nullptr};
    const int e = (int)hipEventRecord(left.stop, stream);
    return rc ? rc : e;
}

#define TOK_MOST_LD (1 << 23)  // 256 rows lie within 2^31 bytes
#define TOK_KB 128  // bytes of k in a stage: 64 elements of 16 bits, 32 of 32

// acc += a b over 64 bytes of k: lane group g = lane / 16 holds k = 8 g ... 8 g + 7 (16 bits), or four products of
// k = 4 g + part, which the hardware sums over g (32 bits; both operands agree on the order).
template <class T> __device__ __forceinline__ void tok_mma(sel_f4& acc, tok_u4 a, tok_u4 b, int part) {
    if constexpr (std::is_same<T, __bf16>::value) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(tok_b8, a), __builtin_bit_cast(tok_b8, b), acc, 0, 0, 0);
    } else if constexpr (std::is_same<T, _Float16>::value) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(tok_h8, a), __builtin_bit_cast(tok_h8, b), acc, 0, 0, 0);
    } else {
        const sel_f4 x = __builtin_bit_cast(sel_f4, a), y = __builtin_bit_cast(sel_f4, b);
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[part], y[part], acc, 0, 0, 0);
    }
}

#define TOK_PUT 2048  // bytes of the LDS that tok_put has to a wave

// An operand: rows of `ld` bytes at p (multiples of 16 both; TOK_MOST_LD at most).  HALF != 0: two matrices side by side, the
// second at p2; of every 2 HALF rows of a tile the first half are the first one's, so that a wave holds equal rows of both.
struct TokRows {
    const char *p, *p2;
    long long ld;
    long long rows;  // that there are (of each): those beyond are read as the last one
    // An operand that lies across (16 bits, tiles of 256): rows along m (n), one to a k, of `across` bytes; what lies beyond them
    // is read as their last 16.  p2: the rows from k = `second` on (a multiple of 64) are those at p2, k_rows of each matrix.
    long long across = 0, second = 0, k_rows = 0;
};

struct TokProduct {
    TokRows a, b;
    const int* live;   // how many rows of B count (device), or NULL: b.rows
    const int* k_live; // how many elements of k count (device), or NULL
    long long k_bytes; // of a row
    int m_tiles, n_tiles;
    int splits;        // parts that k is cut into: so many, or
    bool last = false; // the entry point's last launch
    int slots = 0;     // (not zero) as many as let the tiles of rows that count take so many work-groups, up to `splits`
};

// How many parts k has: where rows do not count, whose number the host does not know, tiles are fewer and parts more
static __host__ __device__ __forceinline__ int tok_parts(int slots, int tiles, int most) {
    const int n = slots / (tiles > 0 ? tiles : 1);
    return n < 1 ? 1 : n < most ? n : most;
}

template <int BM_, int BN_, int WM_, int WN_> struct TokShape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;     // tile, waves along m and n
    static constexpr int kWaves = WM * WN, kThreads = kWaves * NHIP_WAVE;
    static constexpr int kWaveM = BM / WM, kWaveN = BN / WN, MI = kWaveM / 16, NI = kWaveN / 16;
    static constexpr int kStage = (BM + BN) * TOK_KB;
    // an epilogue has 8 bytes per column and wave of m, or TOK_PUT to a wave
    static constexpr int kEpilogue = 8 * WM * BN > TOK_PUT * kWaves ? 8 * WM * BN : TOK_PUT * kWaves, kLds = 2 * kStage + kEpilogue;
    static constexpr bool kPair = kWaves == 8;
    // work-groups to a compute unit, by the LDS and by the registers: two waves to a SIMD
    static constexpr int kAtOnce = (160 << 10) / kLds < 8 / kWaves ? (160 << 10) / kLds : 8 / kWaves;
    static_assert(kWaveM % 16 == 0 && kWaveN % 16 == 0 && MI * NI <= 32, "waves hold whole tiles, in half of a SIMD's registers");
};

// Where a work-group's wave is
struct TokPlace {
    int m_tile, n_tile, split;
    int wave_m, wave_n, l, g;   // lane % 16, lane / 16
    int live;                   // rows of B that count
    char* lds;                  // S::kEpilogue bytes, the epilogue's own
    int wave;
};

static __device__ const tok_u4 tok_zeros = {0, 0, 0, 0};  // what lies behind the end of a row

// 16 bytes to a lane, straight into the LDS: lane i's to `to` + 16 i.  (The builtin of this has the compiler wait for all such
// loads before reads of the LDS that it cannot tell apart from them: half of what was under way had to arrive a turn early.  The
// kernel waits by their number instead, tok_wait and the turns; no register is written.)
static __device__ __forceinline__ void tok_load_lds(const char* from, char* to) {
    const unsigned at = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)to;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory", "m0");
}

// One operand's part of a stage: instruction i of a wave brings rows 8 i ... 8 i + 7.  Row r's 16 bytes c lie at c ^ (r % 8),
// so that 8 rows' same bytes lie in different banks.  Every wave has as many instructions (where there are fewer rows several
// bring the same ones), so that it knows by their number which have arrived.
template <int ROWS, int WAVES, int HALF> struct TokLoader {
    static constexpr int kAll = ROWS / 8, kMine = (kAll + WAVES - 1) / WAVES;
    const char* at[kMine];

    static __device__ __forceinline__ int part(int lane) { return 16 * ((lane % 8) ^ (lane / 8)); }
    static __device__ __forceinline__ int instruction(int wave, int q) {
        const int i = wave + q * WAVES;
        return kAll % WAVES == 0 ? i : min(i, kAll - 1);
    }
    static __device__ __forceinline__ const char* row_at(const TokRows& t, long long row0, int row, long long k0) {
        const long long first = HALF ? row0 / 2 : row0;
        const int last = (int)min((long long)ROWS, t.rows - first) - 1;
        const char* p = t.p;
        if constexpr (HALF > 0) {
            p = row / HALF % 2 ? t.p2 : t.p;
            row = row / (2 * HALF) * HALF + row % HALF;
        }
        return p + first * t.ld + k0 + (unsigned)min(row, last) * (unsigned)t.ld;
    }
    __device__ __forceinline__ void begin(const TokRows& t, long long row0, int wave, int lane, long long k0) {
#pragma unroll
        for (int q = 0; q < kMine; ++q) at[q] = row_at(t, row0, 8 * instruction(wave, q) + lane / 8, k0) + part(lane);
    }
    // The last `left` bytes of k: what lies behind the end of a row is read from elsewhere
    __device__ __forceinline__ void cut(int lane, int left) {
#pragma unroll
        for (int q = 0; q < kMine; ++q) at[q] = part(lane) < left ? at[q] : reinterpret_cast<const char*>(&tok_zeros);
    }
    __device__ __forceinline__ void load(char* to, int wave, int q) {
        tok_load_lds(at[q], to + instruction(wave, q) * 1024);
        at[q] += TOK_KB;
    }
};

// The same for an operand that lies across: a stage is 64 rows of 512 bytes, one to a k.  Instruction i of a wave brings rows 2 i
// and 2 i + 1.  Reads of 4 k by 16 columns (ds_read_b64_tr_b16) take rows 8 g + 4 h + 0 ... 3 of all four lane groups g at
// once: these lie next to each other in the LDS, 32 bytes between two instructions' rows.  (Rows 2 i and 2 i + 1 meet in the same
// banks.  With the odd rows' units exchanged they do not, and the gradient of 8192 x 65536 logits took 4110 us, not 4080: the
// LDS is not what it waits for.)
#define TOK_ACROSS 1056  // bytes of two rows in the LDS
template <int WAVES> struct TokAcross {
    static constexpr int kMine = 32 / WAVES;
    static_assert(WAVES == 8, "");
    const char* at[kMine];
    static __device__ __forceinline__ int place(int wave, int q) {
        return (8 * (wave / 2 % 2) + 2 * (wave / 4) + wave % 2 + 16 * (q / 2) + 4 * (q % 2)) * TOK_ACROSS;
    }
    __device__ __forceinline__ void begin(const TokRows& t, long long col0, int wave, int lane, long long k0) {
        const long long c = min(2 * col0 + 16 * (lane % 32), t.across - 16);
        const bool other = t.p2 && k0 >= t.second;
#pragma unroll
        for (int q = 0; q < kMine; ++q)
            at[q] = (other ? t.p2 : t.p) + (k0 - (other ? t.second : 0) + 2 * (wave + q * WAVES) + lane / 32) * t.ld + c;
    }
    __device__ __forceinline__ void cut(int wave, int lane, long long left) {  // rows of k that are left
#pragma unroll
        for (int q = 0; q < kMine; ++q)
            at[q] = 2 * (wave + q * WAVES) + lane / 32 < left ? at[q] : reinterpret_cast<const char*>(&tok_zeros);
    }
    __device__ __forceinline__ void load(char* to, int wave, int q, long long ld) {
        tok_load_lds(at[q], to + place(wave, q));
        at[q] += 64 * ld;
    }
};

// 8 k (from half a stage, s) of column l of a unit of 16 columns: `from` is the lane's place in unit 0
static __device__ __forceinline__ tok_u4 tok_read_across(const char* from, int s, int unit) {
    typedef __attribute__((address_space(3))) sel_b4* lds;
    typedef unsigned pair __attribute__((ext_vector_type(2)));
    const char* const p = from + s * 16 * TOK_ACROSS + unit * 32;
    const pair lo = __builtin_bit_cast(pair, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds)p));
    const pair hi = __builtin_bit_cast(pair, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds)(p + 8 * TOK_ACROSS)));
    return tok_u4{lo.x, lo.y, hi.x, hi.y};
}

// A wave's part of half a stage, 64 bytes of k
template <class S> struct TokPart {
    static constexpr int kReads = S::MI + S::NI;
    tok_u4 a[S::MI], b[S::NI];
    // its q-th 16 rows: those of B, which all of A's meet, come first
    __device__ __forceinline__ void read_one(int q, const char* from_a, const char* from_b, int c) {
        if (q < S::NI) b[q] = *reinterpret_cast<const tok_u4*>(from_b + c + q * 16 * TOK_KB);
        else a[q - S::NI] = *reinterpret_cast<const tok_u4*>(from_a + c + (q - S::NI) * 16 * TOK_KB);
    }
    __device__ __forceinline__ void read(const char* from_a, const char* from_b, int c) {
#pragma unroll
        for (int q = 0; q < kReads; ++q) read_one(q, from_a, from_b, c);
    }
    // products q of n, in steps
    template <class T> __device__ __forceinline__ void multiply(sel_f4 (&acc)[S::MI][S::NI], int q, int n) const {
        constexpr int kProducts = S::MI * S::NI * (sizeof(T) == 2 ? 1 : 4);
#pragma unroll
        for (int e = q * kProducts / n; e < (q + 1) * kProducts / n; ++e) {
            const int part = e / (S::MI * S::NI), i = e / S::NI % S::MI, j = e % S::NI;
            tok_mma<T>(acc[i][j], a[i], b[j], part);
        }
    }
};

// Tile `id` of m_tiles x n_tiles: bands of 8 tiles of m, so that the tiles under way at once on a die share rows in its L2
static __device__ __forceinline__ void tok_tile(int id, int m_tiles, int n_tiles, int& m, int& n) {
    constexpr int kBand = 8;
    const int band = id / (kBand * n_tiles), first = band * kBand;
    const int wide = min(kBand, m_tiles - first), at = id - band * kBand * n_tiles;
    m = first + at % wide;
    n = at / wide;
}

// Waits until the products before it are done: a result that is read behind the loop's branch needs it (see sel_settle).
template <int MI, int NI> __device__ __forceinline__ void tok_settle(sel_f4 (&acc)[MI][NI]) {
    auto touch = [&] {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) asm volatile("" : "+v"(acc[i][j]));
    };
    touch();
    asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");
    touch();
}

template <int N> __device__ __forceinline__ void tok_wait() {  // until all but the last N loads have come, and all is read
    static_assert(N < 64, "what the counter holds");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// As many work-groups as run at once go over the tiles, those of a die over neighbouring ones; tiles of rows that do not count
// are no tiles.  The stages of all its tiles are one stream to a work-group: what is on its way does not stop at a
// tile's end.
// ACROSS: bit 0: A lies across, bit 1: B does
template <class T, class S, int HALF, int ACROSS, class Epilogue>
__global__ __launch_bounds__(S::kThreads, S::kAtOnce * S::kWaves / 4) void tok_product_kernel(TokProduct p, Epilogue epilogue) {
    extern __shared__ __attribute__((aligned(16))) char tok_lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NHIP_WAVE), lane = threadIdx.x % NHIP_WAVE;
    static_assert(ACROSS == 0 || (S::kPair && sizeof(T) == 2 && HALF == 0), "");
    constexpr bool kAX = ACROSS & 1, kBX = ACROSS & 2;
    constexpr int kBytesA = kAX ? 32 * TOK_ACROSS : S::BM * TOK_KB, kStage = kBytesA + (kBX ? 32 * TOK_ACROSS : S::BN * TOK_KB);
    TokPlace at;
    at.live = (int)(p.live ? min((long long)*p.live, p.b.rows) : p.b.rows);
    at.wave = wave;
    at.wave_m = wave % S::WM;
    at.wave_n = wave / S::WM;
    at.l = lane % 16;
    at.g = lane / 16;
    at.lds = tok_lds + 2 * kStage;
    const int n_tiles = (at.live + S::BN - 1) / S::BN, tiles = p.m_tiles * n_tiles;
    const int splits = p.slots ? tok_parts(p.slots, tiles, p.splits) : p.splits, total = tiles * splits;
    const long long bytes = p.k_live ? (long long)*p.k_live * (int)sizeof(T) : p.k_bytes;
    const int all = (int)((bytes + TOK_KB - 1) / TOK_KB), per = (all + splits - 1) / splits;
    const int dies = NHIP_NXCD, die = blockIdx.x % dies, step = (int)gridDim.x / dies;  // (the grid is a multiple of it)
    const int end = (int)((long long)total * (die + 1) / dies);
    int id = (int)((long long)total * die / dies) + blockIdx.x / dies;

    struct Tile {
        int m, n, split, k0, stages;
    };
    auto tile = [&](int i) {
        Tile t;
        t.split = i / max(tiles, 1);
        tok_tile(i - t.split * tiles, p.m_tiles, n_tiles, t.m, t.n);
        t.k0 = min(all, t.split * per);
        t.stages = min(all, t.k0 + per) - t.k0;
        return t;
    };
    // the stream: what is sent for next
    using LoaderA = typename std::conditional<kAX, TokAcross<8>, TokLoader<S::BM, S::kWaves, HALF>>::type;
    using LoaderB = typename std::conditional<kBX, TokAcross<8>, TokLoader<S::BN, S::kWaves, 0>>::type;
    constexpr int kLoads = LoaderA::kMine + LoaderB::kMine;
    LoaderA la;
    LoaderB lb;
    int coming = id - step, coming_left = 0;  // its tile, the stages of it that are left
    int coming_m = 0;
    long long left = 0;                       // bytes of k
    auto load = [&](int q, int place) {
        char* const to = tok_lds + place * kStage;
        if (q < LoaderA::kMine) {
            if constexpr (kAX) la.load(to, wave, q, p.a.ld);
            else la.load(to, wave, q);
        } else {
            if constexpr (kBX) lb.load(to + kBytesA, wave, q - LoaderA::kMine, p.b.ld);
            else lb.load(to + kBytesA, wave, q - LoaderA::kMine);
        }
    };
    auto sent = [&] {
        left -= TOK_KB;
        --coming_left;
    };
    auto prepare = [&] {  // where a stage's rows are; behind the last stage there are zeros to send for
        if (coming_left == 0) {
            while (coming < end && coming_left == 0) {
                coming += step;
                if (coming < end) coming_left = tile(coming).stages;
            }
            if (coming >= end) {
                left = 0;
                coming_left = 1;
            } else {
                const Tile t = tile(coming);
                const long long k0 = (long long)t.k0 * TOK_KB;
                left = bytes - k0;
                la.begin(p.a, (long long)t.m * S::BM, wave, lane, kAX ? k0 / (int)sizeof(T) : k0);
                lb.begin(p.b, (long long)t.n * S::BN, wave, lane, kBX ? k0 / (int)sizeof(T) : k0);
                coming_m = t.m;
            }
        }
        if constexpr (kAX)
            if (p.a.p2 && left > 0) {  // two matrices: the second one's rows begin, the rows of one end
                const long long k = (bytes - left) / (int)sizeof(T);
                if (k == p.a.second) la.begin(p.a, (long long)coming_m * S::BM, wave, lane, k);
                const long long rest = p.a.k_rows - (k < p.a.second ? k : k - p.a.second);
                if (rest < 64) la.cut(wave, lane, rest);
            }
        if (left < TOK_KB) {  // (a stage of zeros is `left` below zero for the next one: that is cut, too)
            if constexpr (kAX) la.cut(wave, lane, left / (int)sizeof(T));
            else la.cut(lane, (int)left);
            if constexpr (kBX) lb.cut(wave, lane, left / (int)sizeof(T));
            else lb.cut(lane, (int)left);
        }
    };

    if (id >= end) return;
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
        prepare();
#pragma unroll
        for (int q = 0; q < kLoads; ++q)
            if (!S::kPair || s == 0 || q < kLoads / 2) load(q, s);  // (pairs of groups: half of the second one, as always)
        if (!S::kPair || s == 0) sent();
    }
    tok_wait<0>();
    constexpr int kSteps = TokPart<S>::kReads;
    const int c0 = (at.g ^ (at.l & 7)) * 16 + at.l * TOK_KB, c1 = c0 ^ 64;
    const int cx = (2 * at.g + at.l / 8) * TOK_ACROSS + at.l / 4 % 2 * 512 + at.l % 4 * 8;  // across
    int place = 0;  // of the stage that is multiplied next
    for (; id < end; id += step) {
        const Tile now = tile(id);
        at.m_tile = now.m;
        at.n_tile = now.n;
        at.split = now.split;
        sel_f4 acc[S::MI][S::NI];
#pragma unroll
        for (int i = 0; i < S::MI; ++i)
#pragma unroll
            for (int j = 0; j < S::NI; ++j) acc[i][j] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
        const char* const a0 = tok_lds + (kAX ? at.wave_m * S::kWaveM * 2 + cx : at.wave_m * S::kWaveM * TOK_KB);
        const char* const b0 = tok_lds + kBytesA + (kBX ? at.wave_n * S::kWaveN * 2 + cx : at.wave_n * S::kWaveN * TOK_KB);
        if constexpr (S::kPair) {
            // Two groups of four waves, one of each to a SIMD, take turns: while one multiplies a quarter of its tile by a stage,
            // the other reads its next quarter's operands and sends for more.  The second group is half a turn behind, which
            // the barriers before and behind the tile bring about and undo.
            constexpr int HM = S::MI / 2, HN = S::NI / 2;
            tok_u4 a[2][HM], b[2][2][HN];
            auto read_a = [&](int h) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int i = 0; i < HM; ++i) {
                        if constexpr (kAX) a[s][i] = tok_read_across(a0 + place * kStage, s, h * HM + i);
                        else a[s][i] = *reinterpret_cast<const tok_u4*>(a0 + place * kStage + (s ? c1 : c0) + (h * HM + i) * 16 * TOK_KB);
                    }
            };
            auto read_b = [&](int h) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int j = 0; j < HN; ++j) {
                        if constexpr (kBX) b[h][s][j] = tok_read_across(b0 + place * kStage, s, h * HN + j);
                        else b[h][s][j] = *reinterpret_cast<const tok_u4*>(b0 + place * kStage + (s ? c1 : c0) + (h * HN + j) * 16 * TOK_KB);
                    }
            };
            auto turn = [&] {
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
            };
            auto multiply = [&](int hm, int hn) {
                turn();
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int e = 0; e < (sizeof(T) == 2 ? 1 : 4); ++e)
#pragma unroll
                        for (int i = 0; i < HM; ++i)
#pragma unroll
                            for (int j = 0; j < HN; ++j) tok_mma<T>(acc[hm * HM + i][hn * HN + j], a[s][i], b[hn][s][j], e);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
                turn();
            };
            auto loads = [&](int from, int to, int where) {
#pragma unroll
                for (int q = 0; q < kLoads; ++q)
                    if (q >= from && q < to) load(q, where);
            };
            const bool behind = wave >= S::kWaves / 2;
            if (behind) turn();
            for (int k = 0; k < now.stages; ++k) {
                read_a(0);
                read_b(0);
                loads(kLoads / 2, kLoads * 3 / 4, place ^ 1);
                multiply(0, 0);
                read_b(1);
                loads(kLoads * 3 / 4, kLoads, place ^ 1);
                sent();
                multiply(0, 1);
                read_a(1);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (all of this stage's place is read)
                multiply(1, 1);
                prepare();
                loads(0, kLoads / 2, place);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads / 2) : "memory");  // the next stage has come
                multiply(1, 0);
                place ^= 1;
            }
            if (!behind) turn();
        } else {
            TokPart<S> first, second;
            if (now.stages > 0) first.read(a0 + place * kStage, b0 + place * kStage, c0);
            // Half a stage: `next` is read, and `loads` are sent for, between the products.  (Products first: the compiler waits for
            // all reads before the first one, which have come then; and no read among the last quarter, whose time a read takes.)
            auto half = [&](const TokPart<S>& mine, TokPart<S>& next, int from, int c, auto&& loads) {
#pragma unroll
                for (int q = 0; q < kSteps; ++q) {
                    mine.template multiply<T>(acc, q, kSteps);
#pragma unroll
                    for (int o = 4 * q / 3; o < 4 * (q + 1) / 3 && o < kSteps; ++o)
                        next.read_one(o, a0 + from * kStage, b0 + from * kStage, c);
                    loads(q);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            auto stage = [&] {
                half(first, second, place, c1, [](int) {});
                tok_wait<0>();  // the other stage has come, this one is read
                half(second, first, place ^ 1, c0, [&](int q) {  // (behind the tile's last stage `first` is read for nothing)
#pragma unroll
                    for (int o = 2 * q * kLoads / kSteps; o < 2 * (q + 1) * kLoads / kSteps && o < kLoads; ++o) load(o, place);
                });
                place ^= 1;
                sent();
            };
            // whole stages of this tile are sent for without a branch; its last one, and those of the next tiles, in a loop of their own
            int k = 0;
            for (; k + 3 < now.stages; ++k) stage();
            for (; k < now.stages; ++k) {
                prepare();
                stage();
            }
        }
        tok_settle(acc);
        TokPlace here = at;
        asm volatile("" : "+v"(here.l), "+v"(here.g));  // (or what an epilogue forms of them is kept over all tiles, and spilled)
        epilogue.template run<T, S>(here, acc);
    }
    tok_wait<0>();  // (nothing arrives in the LDS of a work-group that has ended)
}

// Up to 16 columns: nothing is read twice, so that all is the time that A takes to arrive.  A work-group has MT tiles of 16 rows;
// its four waves have a quarter of k each, straight from memory into registers, U steps of 64 bytes of k under way while as
// many are multiplied, and add up their sums in the LDS.  (One row, 2048 channels, 2 x 5504 features in bfloat16: 45 MB in 13 us,
// 205 MB of a vocabulary in 36, part of it from the last cache; tiles of 128 rows through the LDS, 86 work-groups, took 18.)
template <int MT_> struct TokFew {
    static constexpr int MT = MT_, kWaves = 4, U = 8 / MT_;
    using Shape = TokShape<16 * MT_, 16, 1, 1>;  // what an epilogue sees: a wave has a tile of 16 columns
};

template <class T, class F, int HALF, class Epilogue>
__global__ __launch_bounds__(F::kWaves * NHIP_WAVE, 2) void tok_few_kernel(TokProduct p, Epilogue epilogue) {
    constexpr int MT = F::MT, U = F::U;
    __shared__ sel_f4 s_sum[F::kWaves][MT][NHIP_WAVE];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NHIP_WAVE), lane = threadIdx.x % NHIP_WAVE;
    TokPlace at;
    at.m_tile = nhip_xcd_remap(blockIdx.x, gridDim.x);
    at.n_tile = at.split = at.wave_m = at.wave_n = at.wave = 0;
    at.l = lane % 16;
    at.g = lane / 16;
    at.live = (int)(p.live ? min((long long)*p.live, p.b.rows) : p.b.rows);
    at.lds = nullptr;
    if (at.live <= 0) return;
    const int bytes = (int)p.k_bytes, steps = (bytes + 63) / 64, per = (steps + F::kWaves - 1) / F::kWaves;
    const int first = min(steps, wave * per), n = min(steps, first + per) - first;
    const char* a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const bool other = HALF && i >= MT / 2;  // (equal rows of both matrices, as an epilogue wants them)
        const long long r = (long long)at.m_tile * (HALF ? 8 * MT : 16 * MT) + 16 * (other ? i - MT / 2 : i) + at.l;
        a[i] = (other ? p.a.p2 : p.a.p) + min(r, p.a.rows - 1) * p.a.ld + 16 * at.g;
    }
    const char* const b = p.b.p + min((long long)at.l, (long long)at.live - 1) * p.b.ld + 16 * at.g;
    struct Batch {
        tok_u4 a[U][MT], b[U];
    };
    // (unconditional: what lies behind the end of k, or of the wave's part, is read from elsewhere)
    auto load = [&](Batch& v, int step) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (first + step + u) * 64;
            const bool is = step + u < n && k + 16 * at.g < bytes;
            const char* const zeros = reinterpret_cast<const char*>(&tok_zeros);
#pragma unroll
            for (int i = 0; i < MT; ++i) v.a[u][i] = *reinterpret_cast<const tok_u4*>(is ? a[i] + k : zeros);
            v.b[u] = *reinterpret_cast<const tok_u4*>(is ? b + k : zeros);
        }
    };
    sel_f4 acc[MT][1];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i][0] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](const Batch& v) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < (sizeof(T) == 2 ? 1 : 4); ++e)
#pragma unroll
                for (int i = 0; i < MT; ++i) tok_mma<T>(acc[i][0], v.a[u][i], v.b[u], e);
    };
    Batch even, odd;
    load(even, 0);
    for (int step = 0; step < n; step += 2 * U) {
        load(odd, step + U);
        multiply(even);
        load(even, step + 2 * U);
        multiply(odd);
    }
    tok_settle(acc);
#pragma unroll
    for (int i = 0; i < MT; ++i) s_sum[wave][i][lane] = acc[i][0];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int w = 1; w < F::kWaves; ++w) acc[i][0] += s_sum[w][i][lane];
    epilogue.template run<T, typename F::Shape>(at, acc);
}

// 17 to 64 columns (16 NI): B, which all waves of a work-group read, goes through the LDS, 256 bytes of k at a time; A still goes
// straight into registers.  Two waves share rows and have half of k each.  (48 rows, 2304 channels, 2 x 6144 features in
// float16: B from the L2 into every wave's registers took 24 us, as much again as A.)
template <int MT_, int NI_> struct TokSome {
    static constexpr int MT = MT_, NI = NI_, kWaves = 4, kRows = 32 * MT_;  // of A, to a work-group
    static constexpr int kChunk = 256, kSteps = kChunk / 64, kPart = 16 * NI * kChunk, kLds = 4 * kPart;
    using Shape = TokShape<16 * MT_, 16, 1, 1>;
};

template <class T, class F, int HALF, class Epilogue>
__global__ __launch_bounds__(F::kWaves * NHIP_WAVE, 2) void tok_some_kernel(TokProduct p, Epilogue epilogue) {
    constexpr int MT = F::MT, NI = F::NI;
    extern __shared__ __attribute__((aligned(16))) char tok_lds[];  // [2 in turn][2 halves of k][16 NI rows][256]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NHIP_WAVE), lane = threadIdx.x % NHIP_WAVE;
    const int mine = wave % 2, half = wave / 2;
    TokPlace at;
    at.m_tile = 2 * nhip_xcd_remap(blockIdx.x, gridDim.x) + mine;
    at.split = at.wave_m = at.wave_n = at.wave = 0;
    at.l = lane % 16;
    at.g = lane / 16;
    at.live = (int)(p.live ? min((long long)*p.live, p.b.rows) : p.b.rows);
    at.lds = nullptr;
    if (at.live <= 0) return;
    const int bytes = (int)p.k_bytes, chunks = (bytes + F::kChunk - 1) / F::kChunk, per = (chunks + 1) / 2;  // the same of both halves
    const int k0 = half * per * F::kChunk;
    const char* a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const bool other = HALF && i >= MT / 2;
        const long long r = (long long)at.m_tile * (HALF ? 8 * MT : 16 * MT) + 16 * (other ? i - MT / 2 : i) + at.l;
        a[i] = (other ? p.a.p2 : p.a.p) + min(r, p.a.rows - 1) * p.a.ld + 16 * at.g;
    }
    const char* const zeros = reinterpret_cast<const char*>(&tok_zeros);
    // Instruction i of the two waves of a half brings rows 4 i ... 4 i + 3; row r's 16 bytes c lie at c ^ (r % 8).
    constexpr int kLoads = 16 * NI / 8;
    auto send = [&](int chunk) {
        char* const to = tok_lds + ((chunk & 1) * 2 + half) * F::kPart;
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
            const int i = mine + 2 * q, row = 4 * i + lane / 16, k = k0 + chunk * F::kChunk + 16 * ((lane % 16) ^ (row & 7));
            const char* const from = p.b.p + (long long)min(row, at.live - 1) * p.b.ld + k;
            tok_load_lds(k < bytes ? from : zeros, to + i * 1024);
        }
    };
    tok_u4 even[F::kSteps][MT], odd[F::kSteps][MT];
    auto load = [&](tok_u4 (&v)[F::kSteps][MT], int chunk) {  // (unconditional: what lies behind the end is read from elsewhere)
#pragma unroll
        for (int s = 0; s < F::kSteps; ++s) {
            const int k = k0 + chunk * F::kChunk + 64 * s;
            const bool is = chunk < per && k + 16 * at.g < bytes;
#pragma unroll
            for (int i = 0; i < MT; ++i) v[s][i] = *reinterpret_cast<const tok_u4*>(is ? a[i] + k : zeros);
        }
    };
    sel_f4 acc[MT][NI];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
    // a chunk: the next one's rows are sent for and loaded first
    auto go = [&](int chunk, const tok_u4 (&v)[F::kSteps][MT], tok_u4 (&next)[F::kSteps][MT]) {
        tok_wait<F::kSteps * MT>();  // B's part has come, A's may still be under way; the part before it is read
        send(chunk + 1);             // (behind the last one: zeros)
        __builtin_amdgcn_sched_barrier(0);
        load(next, chunk + 1);
        __builtin_amdgcn_sched_barrier(0);
        const char* const from = tok_lds + ((chunk & 1) * 2 + half) * F::kPart + at.l * F::kChunk;
#pragma unroll
        for (int s = 0; s < F::kSteps; ++s) {
            tok_u4 b[NI];
#pragma unroll
            for (int j = 0; j < NI; ++j)
                b[j] = *reinterpret_cast<const tok_u4*>(from + j * 16 * F::kChunk + (((4 * s + at.g) ^ (at.l & 7)) << 4));
#pragma unroll
            for (int e = 0; e < (sizeof(T) == 2 ? 1 : 4); ++e)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j) tok_mma<T>(acc[i][j], v[s][i], b[j], e);
        }
    };
    send(0);
    __builtin_amdgcn_sched_barrier(0);
    load(even, 0);
    __builtin_amdgcn_sched_barrier(0);
    for (int chunk = 0; chunk < per; chunk += 2) {
        go(chunk, even, odd);
        if (chunk + 1 < per) go(chunk + 1, odd, even);
    }
    tok_settle(acc);
    tok_wait<0>();  // (all is read, and nothing comes any more)
    sel_f4* const s_sum = reinterpret_cast<sel_f4*>(tok_lds) + (mine * MT * NI) * NHIP_WAVE + lane;
    if (half) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) s_sum[(i * NI + j) * NHIP_WAVE] = acc[i][j];
    }
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        if (16 * j >= at.live) continue;
        sel_f4 sum[MT][1];
#pragma unroll
        for (int i = 0; i < MT; ++i) sum[i][0] = acc[i][j] + s_sum[(i * NI + j) * NHIP_WAVE];
        at.n_tile = j;
        epilogue.template run<T, typename F::Shape>(at, sum);
    }
}

#define TOK_FEW 64  // rows of B that the kernels for few columns take
// MT: tiles of 16 rows to a wave (of both matrices, where there are two)
template <class T, int MT, int HALF, class E>
static inline int tok_few(hipStream_t stream, TokProduct p, const E& epilogue) {
    const long long rows = HALF ? 8 * MT : 16 * MT, tiles = (p.a.rows + rows - 1) / rows;
    if (tiles == 0 || p.b.rows == 0) return 0;
    if (p.b.rows > TOK_FEW || tiles > 0xffffff || p.k_bytes > 0x3fffffff) return NHIP_E_BADARG;
    if (p.b.rows <= 16) {
        using F = TokFew<MT>;
        TOK_LAUNCH(p.last, (tok_few_kernel<T, F, HALF, E>), dim3((unsigned)tiles), dim3(F::kWaves * NHIP_WAVE), 0, stream, p, epilogue);
        NHIP_LAUNCH_CHECK();
        return 0;
    }
    auto go = [&](auto some) {
        using F = decltype(some);
        auto kernel = tok_some_kernel<T, F, HALF, E>;
        if (int e = sel_allow_lds(stream, kernel, F::kLds)) return e;
        TOK_LAUNCH(p.last, kernel, dim3((unsigned)((tiles + 1) / 2)), dim3(F::kWaves * NHIP_WAVE), F::kLds, stream, p, epilogue);
        return (int)hipGetLastError();
    };
    if (p.b.rows <= 32) return go(TokSome<MT, 2>());
    if (p.b.rows <= 48) return go(TokSome<MT, 3>());
    return go(TokSome<MT, 4>());
}

// 64 values along m of 16 columns, value(i, v) being a lane's four of tile i of four, to rows of `ld` elements of 16 bits at `to`
// (16-byte aligned): through the wave's part of the LDS, so that a lane stores 16 bytes and a row gets whole lines.
// (Stored as they lie, 8 bytes to a lane in rows of 32: the gradient of 8192 x 65536 logits, 20 % masked, 718 us to a half, 680 so.)
template <class T, class F>
__device__ __forceinline__ void tok_put(const TokPlace& at, T* to, long long ld, int rows, int cols, F&& value) {
    static_assert(sizeof(T) == 2, "");
    char* const lds = at.lds + at.wave * TOK_PUT;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[4];
        value(i, v);
        sel_store<T, 4>(reinterpret_cast<T*>(lds + at.l * 128 + ((2 * i + at.g / 2) ^ (at.l & 7)) * 16 + at.g % 2 * 8), v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int lane = at.l + 16 * at.g, c = lane % 8;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int row = 8 * q + lane / 8;
        const tok_u4 v = *reinterpret_cast<const tok_u4*>(lds + row * 128 + ((c ^ (row & 7)) * 16));
        if (row >= rows) continue;
        T* const p = to + row * ld + 8 * c;
        if (8 * c + 8 <= cols) {
            *reinterpret_cast<tok_u4*>(p) = v;
        } else {
            const SelPack<T, 8> e = __builtin_bit_cast(SelPack<T, 8>, v);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (8 * c + k < cols) p[k] = e.v[k];
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Four values of column n in rows m ... m + 3 (a lane's part of a tile), stored along m at g[n, m] and (unless it is NULL) along n
// at gt[m, n].
// 16 bits: the four lanes of neighbouring columns exchange theirs, so that each stores four neighbours along n, too.
template <class T>
__device__ __forceinline__ void tok_store_both(T* g, long long g_ld, T* gt, long long gt_ld, long long n, long long m,
                                               const float (&v)[4]) {
    T* const to = g + n * g_ld + m;
    if (!gt) {
        sel_store<T, 4>(to, v);
    } else if constexpr (sizeof(T) == 2) {
        typedef unsigned pair __attribute__((ext_vector_type(2)));
        SelPack<T, 4> q;
#pragma unroll
        for (int r = 0; r < 4; ++r) q.v[r] = (T)v[r];
        const pair p = __builtin_bit_cast(pair, q);
        *reinterpret_cast<pair*>(to) = p;
        const int lane = threadIdx.x & 3;
        auto from = [](unsigned x, auto order) {
            return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(order)::value, 0xf, 0xf, true);
        };
        // with the neighbour: rows 0 and 2 in even lanes, 1 and 3 in odd ones, of two columns
        const unsigned which = lane & 1 ? 0x03020706u : 0x05040100u;
        const unsigned a0 = __builtin_amdgcn_perm(from(p.x, std::integral_constant<int, 0xb1>()), p.x, which);
        const unsigned a1 = __builtin_amdgcn_perm(from(p.y, std::integral_constant<int, 0xb1>()), p.y, which);
        // with the lane two further: of four columns
        const unsigned other = from(lane & 2 ? a0 : a1, std::integral_constant<int, 0x4e>());
        pair t;
        t.x = lane & 2 ? other : a0;
        t.y = lane & 2 ? a1 : other;
        *reinterpret_cast<pair*>(gt + (m + lane) * gt_ld + n - lane) = t;
    } else {
        sel_store<T, 4>(to, v);
#pragma unroll
        for (int r = 0; r < 4; ++r) gt[(m + r) * gt_ld + n] = v[r];
    }
}

template <class T, class S, int HALF, int ACROSS = 0, class E>
static inline int tok_product(hipStream_t stream, const TokProduct& p, const E& epilogue) {
    const long long tiles = (long long)p.m_tiles * p.n_tiles * p.splits, groups = 256 * S::kAtOnce;
    if (tiles == 0) return 0;
    if (tiles > 0x3fffffff) return NHIP_E_BADARG;
    auto kernel = tok_product_kernel<T, S, HALF, ACROSS, E>;
    constexpr int kLds = S::kLds + (ACROSS ? 2 * 64 * (TOK_ACROSS - 1024) : 0);
    if (int e = sel_allow_lds(stream, kernel, kLds)) return e;
    // (as many to each die: with as many work-groups as tiles a die could have a tile more than it had work-groups, and take
    // two rounds; 474 tiles of 128 x 128, 2540 channels in float32: 505 us, 372 so)
    const long long even = (tiles + NHIP_NXCD - 1) / NHIP_NXCD * NHIP_NXCD;
    TOK_LAUNCH(p.last, kernel, dim3((unsigned)(even < groups ? even : groups)), dim3(S::kThreads), kLds, stream, p, epilogue);
    NHIP_LAUNCH_CHECK();
    return 0;
}

using TokLarge = TokShape<256, 256, 2, 4>;
#define TOK_LEAST_BM 32  // of the kernels for few columns (without HALF); other shapes' tiles have 128 rows at least
#define TOK_MOST_TILE 256

// The shape of a product of m x n in elements of `size` bytes: tiles of 256 x 256 where they are enough to go round, of fewer
// columns where there are few.  (8192 x 11008 x 2048 in bfloat16: 1320 TFLOP/s by tiles of 256, 800 by tiles of 128.  These are all
// under way at once up to 512, which are 128 large ones: 25000 x 250 x 2048 in 31 us, by large tiles 44; 19200 x 500 x 2048 in
// 54, by large tiles 47.  In 32 bits, where the matrix instructions take as long either way, the smaller ones share 256
// compute units more evenly.)
static inline bool tok_is_large(long long m, long long n, int size, int splits, int least = 129) {
    const long long large = ((m + 255) / 256) * ((n + 255) / 256) * splits;
    return n > 128 && m > 128 && large >= (size == 2 ? least : 512);
}
// (of more than TOK_FEW columns: fewer go to tok_few, or may be any)
template <class F> static inline int tok_with_many(long long m, long long n, int size, int splits, F&& f) {
    if (tok_is_large(m, n, size, splits)) return f(TokLarge());
    return f(TokShape<128, 128, 2, 2>());
}
template <class F> static inline int tok_with_shape(long long m, long long n, int size, int splits, F&& f) {
    if (n > 64) return tok_with_many(m, n, size, splits, f);
    if (n > 16) return f(TokShape<128, 64, 4, 1>());
    return f(TokShape<128, 16, 4, 1>());
}

// Into how many parts k (of k_bytes) is cut so that a product of m x n goes round 256 compute units, parts of eight stages at
// least; and the most parts that there may be.
static inline long long tok_most_splits(long long k_bytes) {
    const long long n = k_bytes / TOK_KB / 8;
    return n < 1 ? 1 : n < 64 ? n : 64;
}
static inline int tok_splits(long long m, long long n, int size, long long k_bytes) {
    if (m < 1 || n < 1) return 1;
    const long long most = tok_most_splits(k_bytes);
    long long s = 1;
    if (size == 2 && n > 128 && m > 128) s = 256 / (((m + 255) / 256) * ((n + 255) / 256));
    else s = 512 / (((m + 127) / 128) * ((n + 127) / 128));
    return (int)(s < 1 ? 1 : s < most ? s : most);
}
