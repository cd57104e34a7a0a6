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

// An operand: rows of `ld` bytes at p (multiples of 16 both).  `half` != 0: two matrices side by side, the second at p2; of
// every 2 `half` rows of a tile the first half are the first one's, so that a wave holds equal rows of both.
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
    int splits;        // parts that k is cut into (gridDim.y)
};

template <int BM_, int BN_, int WM_, int WN_> struct TokShape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;     // tile, waves along m and n
    static constexpr int kWaves = WM * WN, kThreads = kWaves * NHIP_WAVE;
    static constexpr int kWaveM = BM / WM, kWaveN = BN / WN, MI = kWaveM / 16, NI = kWaveN / 16;
    static constexpr int kStage = (BM + BN) * TOK_KB, kLds = 2 * kStage;
    static_assert(kWaveM % 16 == 0 && kWaveN % 16 == 0, "waves hold whole tiles");
};

// Where a work-group's wave is
struct TokPlace {
    int m_tile, n_tile, split;
    int wave_m, wave_n, l, g;   // lane % 16, lane / 16
    int live;                   // rows of B that count
    char* lds;                  // free for the epilogue after a barrier
};

static __device__ const tok_u4 tok_zeros = {0, 0, 0, 0};  // what lies behind the end of a row

static __device__ __forceinline__ void tok_load_lds(const char* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// One operand's part of a stage: instruction i of a wave brings rows 8 i ... 8 i + 7.  Row r's 16 bytes c lie at c ^ (r % 8),
// so that 8 rows' same bytes lie in different banks.
template <int ROWS, int WAVES> struct TokLoader {
    static constexpr int kAll = ROWS / 8, kMine = (kAll + WAVES - 1) / WAVES;
    const char* at[kMine];

    __device__ __forceinline__ void begin(const TokRows& t, long long row0, int half, int wave, int lane, long long k0) {
#pragma unroll
        for (int q = 0; q < kMine; ++q) {
            const int row = 8 * (wave + q * WAVES) + lane / 8;
            long long r = row0 + row;
            const char* p = t.p;
            if (half) {
                const int of = row % (2 * half);
                r = row0 / 2 + row / (2 * half) * half + of % half;
                p = of < half ? t.p : t.p2;
            }
            r = r < t.rows ? r : t.rows - 1;
            at[q] = p + r * t.ld + k0 + 16 * ((lane % 8) ^ (lane / 8));
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

template <class T, class S, int HALF, class Epilogue>
__global__ __launch_bounds__(S::kThreads) void tok_product_kernel(TokProduct p, Epilogue epilogue) {
    extern __shared__ __attribute__((aligned(16))) char tok_lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NHIP_WAVE), lane = threadIdx.x % NHIP_WAVE;
    TokPlace at;
    tok_tile(nhip_xcd_remap(blockIdx.x, gridDim.x), p.m_tiles, p.n_tiles, at.m_tile, at.n_tile);
    at.live = p.live ? min((long long)*p.live, p.b.rows) : (int)p.b.rows;
    at.split = blockIdx.y;
    if ((long long)at.n_tile * S::BN >= at.live) return;  // uniform over the work-group
    at.wave_m = wave % S::WM;
    at.wave_n = wave / S::WM;
    at.l = lane % 16;
    at.g = lane / 16;
    at.lds = tok_lds;

    long long bytes = p.k_live ? (long long)*p.k_live * (int)sizeof(T) : p.k_bytes;
    const int all = (int)((bytes + TOK_KB - 1) / TOK_KB), per = (all + p.splits - 1) / p.splits;
    const int k0 = min(all, at.split * per), n = min(all, k0 + per) - k0;
    long long left = bytes - (long long)k0 * TOK_KB;

    sel_f4 acc[S::MI][S::NI];
#pragma unroll
    for (int i = 0; i < S::MI; ++i)
#pragma unroll
        for (int j = 0; j < S::NI; ++j) acc[i][j] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
    TokLoader<S::BM, S::kWaves> la;
    TokLoader<S::BN, S::kWaves> lb;
    la.begin(p.a, (long long)at.m_tile * S::BM, HALF, wave, lane, (long long)k0 * TOK_KB);
    lb.begin(p.b, (long long)at.n_tile * S::BN, 0, wave, lane, (long long)k0 * TOK_KB);
    auto fetch = [&](int stage) {
        char* const to = tok_lds + stage * S::kStage;
        const int some = (int)min(left, (long long)TOK_KB);
        la.load(to, wave, lane, some);
        lb.load(to + S::BM * TOK_KB, wave, lane, some);
        left -= TOK_KB;
    };
    if (n > 0) fetch(0);
    for (int k = 0; k < n; ++k) {
        __syncthreads();  // this stage has come, the other one is read
        if (k + 1 < n) fetch((k + 1) & 1);
        const char* const a = tok_lds + (k & 1) * S::kStage;
        tok_stage<T, S>(acc, a + at.wave_m * S::kWaveM * TOK_KB, a + (S::BM + at.wave_n * S::kWaveN) * TOK_KB, at.l, at.g);
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

template <class T, class S, int HALF, class E>
static inline int tok_product(hipStream_t stream, const TokProduct& p, const E& epilogue) {
    const long long tiles = (long long)p.m_tiles * p.n_tiles;
    if (tiles == 0) return 0;
    if (tiles > 0x7fffff || p.splits < 1 || p.splits > SEL_MAX_GRID_Y) return NHIP_E_BADARG;
    auto kernel = tok_product_kernel<T, S, HALF, E>;
    if (int e = sel_allow_lds(stream, kernel, S::kLds)) return e;
    NHIP_LAUNCH(kernel, dim3((unsigned)tiles, (unsigned)p.splits), dim3(S::kThreads), S::kLds, stream, p, epilogue);
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
