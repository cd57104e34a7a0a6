// The matrix product behind the operators over tokens (gated projection, losses over a vocabulary):
//
//     D[m, n] = sum_k A[m, k] B[n, k],     rows of A and B along k, sums in 32 bits
//
// and what becomes of D is the caller's: an epilogue gets it in registers.  A work-group forms a tile of BM x BN; tiles of A
// and B of 128 bytes along k lie in the LDS in two stages, and the next stage is on its way, straight from memory into the
// LDS, while one is multiplied.
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

#define TOK_MOST_LD (1 << 23)  // 256 rows lie within 2^31 bytes
#define TOK_KB 128  // bytes of k in a stage: 64 elements of 16 bits, 32 of 32

// acc += a b over 64 bytes of k: lane group g = lane / 16 holds k = 8 g ... 8 g + 7 (16 bits), or four products of
// k = 4 g + e, which the hardware sums over g (32 bits; both operands agree on the order).
template <class T> __device__ __forceinline__ void tok_mma(sel_f4& acc, tok_u4 a, tok_u4 b) {
    if constexpr (std::is_same<T, __bf16>::value) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(tok_b8, a), __builtin_bit_cast(tok_b8, b), acc, 0, 0, 0);
    } else if constexpr (std::is_same<T, _Float16>::value) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(tok_h8, a), __builtin_bit_cast(tok_h8, b), acc, 0, 0, 0);
    } else {
        const sel_f4 x = __builtin_bit_cast(sel_f4, a), y = __builtin_bit_cast(sel_f4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
    }
}

// An operand: rows of `ld` bytes at p (multiples of 16 both; TOK_MOST_LD at most).  HALF != 0: two matrices side by side, the
// second at p2; of every 2 HALF rows of a tile the first half are the first one's, so that a wave holds equal rows of both.
struct TokRows {
    const char *p, *p2;
    long long ld;
    long long rows;  // that there are (of each): those beyond are read as the last one
};

struct TokProduct {
    TokRows a, b;
    const int* live;   // how many rows of B count (device), or NULL: b.rows
    const int* k_live; // how many elements of k count (device), or NULL
    long long k_bytes; // of a row
    int m_tiles, n_tiles;
    int splits;        // parts that k is cut into
};

template <int BM_, int BN_, int WM_, int WN_> struct TokShape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;     // tile, waves along m and n
    static constexpr int kWaves = WM * WN, kThreads = kWaves * NHIP_WAVE;
    static constexpr int kWaveM = BM / WM, kWaveN = BN / WN, MI = kWaveM / 16, NI = kWaveN / 16;
    static constexpr int kStage = (BM + BN) * TOK_KB;
    static constexpr int kEpilogue = 8 * WM * BN, kLds = 2 * kStage + kEpilogue;  // an epilogue has 8 bytes per column and wave of m
    // work-groups to a compute unit, by the LDS and the registers of eight waves
    static constexpr int kAtOnce = (160 << 10) / kLds < 8 / kWaves ? (160 << 10) / kLds : 8 / kWaves;
    static_assert(kWaveM % 16 == 0 && kWaveN % 16 == 0, "waves hold whole tiles");
};

// Where a work-group's wave is
struct TokPlace {
    int m_tile, n_tile, split;
    int wave_m, wave_n, l, g;   // lane % 16, lane / 16
    int live;                   // rows of B that count
    char* lds;                  // S::kEpilogue bytes, the epilogue's own
};

static __device__ const tok_u4 tok_zeros = {0, 0, 0, 0};  // what lies behind the end of a row

static __device__ __forceinline__ void tok_load_lds(const char* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// One operand's part of a stage: instruction i of a wave brings rows 8 i ... 8 i + 7.  Row r's 16 bytes c lie at c ^ (r % 8),
// so that 8 rows' same bytes lie in different banks.
template <int ROWS, int WAVES, int HALF> struct TokLoader {
    static constexpr int kAll = ROWS / 8, kMine = (kAll + WAVES - 1) / WAVES;
    const char* at[kMine];

    __device__ __forceinline__ void begin(const TokRows& t, long long row0, int wave, int lane, long long k0) {
        const long long first = HALF ? row0 / 2 : row0;
        const int last = (int)min((long long)ROWS, t.rows - first) - 1;
        const unsigned c = 16 * ((lane % 8) ^ (lane / 8));
#pragma unroll
        for (int q = 0; q < kMine; ++q) {
            int row = 8 * (wave + q * WAVES) + lane / 8;
            const char* p = t.p;
            if constexpr (HALF > 0) {
                p = row / HALF % 2 ? t.p2 : t.p;
                row = row / (2 * HALF) * HALF + row % HALF;
            }
            at[q] = p + first * t.ld + k0 + (unsigned)min(row, last) * (unsigned)t.ld + c;
        }
    }
    // `left`: bytes of k from here on
    __device__ __forceinline__ void load(char* to, int wave, int lane, int left) {
        const int c = 16 * ((lane % 8) ^ (lane / 8));
#pragma unroll
        for (int q = 0; q < kMine; ++q) {
            const int i = wave + q * WAVES;
            if (kAll % WAVES == 0 || i < kAll) {
                tok_load_lds(c < left ? at[q] : reinterpret_cast<const char*>(&tok_zeros), to + i * 1024);
                at[q] += TOK_KB;
            }
        }
    }
};

template <class T, class S>
__device__ __forceinline__ void tok_stage(sel_f4 (&acc)[S::MI][S::NI], const char* a, const char* b, int l, int g) {
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
        const int c = ((4 * sub + g) ^ (l & 7)) * 16 + l * TOK_KB;
        tok_u4 fa[S::MI], fb[S::NI];
#pragma unroll
        for (int i = 0; i < S::MI; ++i) fa[i] = *reinterpret_cast<const tok_u4*>(a + c + i * 16 * TOK_KB);
#pragma unroll
        for (int j = 0; j < S::NI; ++j) fb[j] = *reinterpret_cast<const tok_u4*>(b + c + j * 16 * TOK_KB);
#pragma unroll
        for (int i = 0; i < S::MI; ++i)
#pragma unroll
            for (int j = 0; j < S::NI; ++j) tok_mma<T>(acc[i][j], fa[i], fb[j]);
    }
}

// Tile `id` of m_tiles x n_tiles: bands of 8 tiles of m, so that the tiles under way at once on a die share rows in its L2
static __device__ __forceinline__ void tok_tile(int id, int m_tiles, int n_tiles, int& m, int& n) {
    constexpr int kBand = 8;
    const int band = id / (kBand * n_tiles), first = band * kBand;
    const int wide = min(kBand, m_tiles - first), at = id - band * kBand * n_tiles;
    m = first + at % wide;
    n = at / wide;
}

// As many work-groups as run at once go over the tiles, those of a die over neighbouring ones.  The first stage of the next
// tile is on its way during the last one of a tile and its epilogue.  Tiles of rows that do not count are no tiles.
template <class T, class S, int HALF, class Epilogue>
__global__ __launch_bounds__(S::kThreads) void tok_product_kernel(TokProduct p, Epilogue epilogue) {
    extern __shared__ __attribute__((aligned(16))) char tok_lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NHIP_WAVE), lane = threadIdx.x % NHIP_WAVE;
    TokPlace at;
    at.live = (int)(p.live ? min((long long)*p.live, p.b.rows) : p.b.rows);
    at.wave_m = wave % S::WM;
    at.wave_n = wave / S::WM;
    at.l = lane % 16;
    at.g = lane / 16;
    at.lds = tok_lds + 2 * S::kStage;
    const int n_tiles = (at.live + S::BN - 1) / S::BN, tiles = p.m_tiles * n_tiles, total = tiles * p.splits;
    const long long bytes = p.k_live ? (long long)*p.k_live * (int)sizeof(T) : p.k_bytes;
    const int all = (int)((bytes + TOK_KB - 1) / TOK_KB), per = (all + p.splits - 1) / p.splits;
    const int dies = min(NHIP_NXCD, (int)gridDim.x), die = blockIdx.x % dies, step = ((int)gridDim.x - die + dies - 1) / dies;
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
    TokLoader<S::BM, S::kWaves, HALF> la;
    TokLoader<S::BN, S::kWaves, 0> lb;
    long long left = 0;
    auto begin = [&](const Tile& t) {
        const long long k0 = (long long)t.k0 * TOK_KB;
        left = bytes - k0;
        la.begin(p.a, (long long)t.m * S::BM, wave, lane, k0);
        lb.begin(p.b, (long long)t.n * S::BN, wave, lane, k0);
    };
    auto fetch = [&](int stage) {
        char* const to = tok_lds + stage * S::kStage;
        const int some = (int)min(left, (long long)TOK_KB);
        la.load(to, wave, lane, some);
        lb.load(to + S::BM * TOK_KB, wave, lane, some);
        left -= TOK_KB;
    };

    int stage = 0;
    bool ready = false;  // the tile's first stage is on its way
    Tile next = tile(id);
    while (id < end) {
        const Tile now = next;
        at.m_tile = now.m;
        at.n_tile = now.n;
        at.split = now.split;
        id += step;
        next = tile(id);
        const bool more = id < end && next.stages > 0;
        sel_f4 acc[S::MI][S::NI];
#pragma unroll
        for (int i = 0; i < S::MI; ++i)
#pragma unroll
            for (int j = 0; j < S::NI; ++j) acc[i][j] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!ready && now.stages > 0) {
            __syncthreads();  // (both stages are read)
            begin(now);
            fetch(stage);
        }
        ready = now.stages > 0 && more;
        for (int k = 0; k < now.stages; ++k) {
            __syncthreads();  // this stage has come, the other one is read
            const bool last = k + 1 == now.stages;
            if (last && more) begin(next);
            if (!last || more) fetch(stage ^ 1);
            const char* const a = tok_lds + stage * S::kStage;
            tok_stage<T, S>(acc, a + at.wave_m * S::kWaveM * TOK_KB, a + (S::BM + at.wave_n * S::kWaveN) * TOK_KB, at.l, at.g);
            stage ^= 1;
        }
        // (a result that is read behind the loop's branch: see sel_settle)
#pragma unroll
        for (int i = 0; i < S::MI; ++i)
#pragma unroll
            for (int j = 0; j < S::NI; ++j) asm volatile("" : "+v"(acc[i][j]));
        asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");
#pragma unroll
        for (int i = 0; i < S::MI; ++i)
#pragma unroll
            for (int j = 0; j < S::NI; ++j) asm volatile("" : "+v"(acc[i][j]));
        epilogue.template run<T, S>(at, acc);
    }
}

// Four values of column n in rows m ... m + 3 (a lane's part of a tile), stored along m at g[n, m] and along n at gt[m, n].
// 16 bits: the four lanes of neighbouring columns exchange theirs, so that each stores four neighbours along n, too.
template <class T>
__device__ __forceinline__ void tok_store_both(T* g, long long g_ld, T* gt, long long gt_ld, long long n, long long m,
                                               const float (&v)[4]) {
    T* const to = g + n * g_ld + m;
    if constexpr (sizeof(T) == 2) {
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

template <class T, class S, int HALF, class E>
static inline int tok_product(hipStream_t stream, const TokProduct& p, const E& epilogue) {
    const long long tiles = (long long)p.m_tiles * p.n_tiles * p.splits, groups = 256 * S::kAtOnce;
    if (tiles == 0) return 0;
    if (tiles > 0x3fffffff) return NHIP_E_BADARG;
    auto kernel = tok_product_kernel<T, S, HALF, E>;
    if (int e = sel_allow_lds(stream, kernel, S::kLds)) return e;
    NHIP_LAUNCH(kernel, dim3((unsigned)(tiles < groups ? tiles : groups)), dim3(S::kThreads), S::kLds, stream, p, epilogue);
    NHIP_LAUNCH_CHECK();
    return 0;
}

// Calls f(tile shape) for a product of m x n
template <class F> static inline int tok_with_shape(long long m, long long n, F&& f) {
    const long long large = ((m + 255) / 256) * ((n + 255) / 256);
    if (n > 128 && large >= 128) return f(TokShape<256, 256, 2, 4>());
    if (n > 64) return f(TokShape<128, 128, 2, 2>());
    if (n > 16) return f(TokShape<128, 64, 4, 1>());
    return f(TokShape<128, 16, 4, 1>());
}
#define TOK_LEAST_BM 128  // of the shapes above
#define TOK_MOST_TILE 256
