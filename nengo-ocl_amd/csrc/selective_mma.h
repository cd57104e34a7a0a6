// Matrix products of the selective scan on the matrix cores: fragments of 16 x 32 elements, the
// same for 16-bit and 32-bit elements.
//
// A fragment holds, for the row (first operand) or column (second operand) `lane % 16`, the eight
// values of k at
//     k(e) = 16 (e / 4) + 4 (lane / 16) + e % 4,      e = 0 ... 7.
// The hardware sums over k in whatever order both operands agree on.  This order is that of the
// results: result tile D holds column `lane % 16`, rows 4 (lane / 16) + r in its four registers, so
// that two result tiles side by side are the fragment of a further product without passing
// through memory, and four neighbouring k lie together in memory (8-byte reads of rows).
#pragma once

#include "selective_common.h"

typedef __bf16 sel_b4 __attribute__((ext_vector_type(4)));
typedef __bf16 sel_b8 __attribute__((ext_vector_type(8)));

template <class Tc> struct SelFrag;

template <> struct SelFrag<__bf16> {
    sel_b8 v;
    __device__ __forceinline__ float get(int e) const { return (float)v[e]; }
    __device__ __forceinline__ void set(int e, float f) { v[e] = (__bf16)f; }
};
template <> struct SelFrag<float> {
    float v[8];
    __device__ __forceinline__ float get(int e) const { return v[e]; }
    __device__ __forceinline__ void set(int e, float f) { v[e] = f; }
};

// How many fragments stand for float32 values without loss: three bfloat16 hold 24 bits between
// them.  The other operand holds inputs, which are exact.
template <class Tc> struct SelSplit { static constexpr int n = 1; };
template <> struct SelSplit<__bf16> { static constexpr int n = 3; };

// acc += first second over 32 values of k.  32-bit elements: eight products of four k.
__device__ __forceinline__ void sel_mma(sel_f4& acc, const SelFrag<__bf16>& a, const SelFrag<__bf16>& b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, acc, 0, 0, 0);
}
__device__ __forceinline__ void sel_mma(sel_f4& acc, const SelFrag<float>& a, const SelFrag<float>& b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc, 0, 0, 0);
}

// Fragment of a matrix in LDS whose rows run along k: `row` is this lane's row, at the first k.
__device__ __forceinline__ SelFrag<__bf16> sel_rows(const __bf16* row, int g) {
    const sel_b4 lo = *reinterpret_cast<const sel_b4*>(row + 4 * g);
    const sel_b4 hi = *reinterpret_cast<const sel_b4*>(row + 16 + 4 * g);
    SelFrag<__bf16> f;
    f.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return f;
}
__device__ __forceinline__ SelFrag<float> sel_rows(const float* row, int g) {
    const sel_f4 lo = *reinterpret_cast<const sel_f4*>(row + 4 * g);
    const sel_f4 hi = *reinterpret_cast<const sel_f4*>(row + 16 + 4 * g);
    SelFrag<float> f;
#pragma unroll
    for (int e = 0; e < 4; ++e) { f.v[e] = lo[e]; f.v[4 + e] = hi[e]; }
    return f;
}

// Fragment of a matrix in LDS whose rows run across: `at` is its element (first k, first row or
// column of the tile), `stride` the length of its rows (a multiple of 4).  16-bit elements: the
// 16 lanes of a quarter of the wave name four rows of 16 elements, four to a lane, and each gets
// its column of them (ds_read_b64_tr_b16).
__device__ __forceinline__ SelFrag<__bf16> sel_cols(const __bf16* at, int stride, int l, int g) {
    typedef __attribute__((address_space(3))) sel_b4* lds;
    const __bf16* p = at + (4 * g + (l >> 2)) * stride + 4 * (l & 3);
    const sel_b4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds)(p));
    const sel_b4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds)(p + 16 * stride));
    SelFrag<__bf16> f;
    f.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return f;
}
__device__ __forceinline__ SelFrag<float> sel_cols(const float* at, int stride, int l, int g) {
    SelFrag<float> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = at[(16 * (e >> 2) + 4 * g + (e & 3)) * stride + l];
    return f;
}

// Eight float32 values as fragments that add up to them.  What is no number or infinite is so in
// the first alone.
template <class Tc>
__device__ __forceinline__ void sel_split(const float (&x)[8], SelFrag<Tc> (&f)[SelSplit<Tc>::n]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float rest = x[e];
#pragma unroll
        for (int s = 0; s < SelSplit<Tc>::n; ++s) {
            f[s].set(e, rest);
            if (s + 1 < SelSplit<Tc>::n) rest = fabsf(x[e]) < 3.0e38f ? rest - f[s].get(e) : 0.0f;
        }
    }
}

// Row length in LDS: `n` elements (a multiple of 8) and 16 bytes, so that the rows of a tile begin
// in different banks and at multiples of 16 bytes.
template <class Tc> __host__ __device__ constexpr int sel_stride(int n) { return n + 16 / (int)sizeof(Tc); }

// Rows of inputs into LDS, zero beyond their ends: ROWS x COLS from `src` (row stride `stride`), of which
// n_rows x n_cols are there.  vec: rows begin at multiples of 16 bytes.
template <class T, class Tc, int ROWS, int COLS>
__device__ __forceinline__ void sel_stage(Tc* dst, const T* src, long long stride, int n_rows, int n_cols,
                                          bool vec) {
    constexpr int V = 16 / (int)sizeof(T), kPer = COLS / V, kRow = sel_stride<Tc>(COLS);
#pragma unroll 4
    for (int q = threadIdx.x; q < ROWS * kPer; q += NHIP_WG) {
        const int r = q / kPer, c = (q % kPer) * V;
        SelPack<Tc, V> v;
        if (vec && r < n_rows && c + V <= n_cols) {
            const SelPack<T, V> in = *reinterpret_cast<const SelPack<T, V>*>(src + r * stride + c);
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = (Tc)in.v[i];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                v.v[i] = r < n_rows && c + i < n_cols ? (Tc)src[r * stride + c + i] : (Tc)0.0f;
        }
        // (packs of 16 bytes: rows in LDS begin at multiples of 16)
        Tc* out = dst + r * kRow + c;
        if constexpr (sizeof(Tc) * V == 16) {
            *reinterpret_cast<SelPack<Tc, V>*>(out) = v;
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 4)
                *reinterpret_cast<sel_f4*>(out + i) = sel_f4{v.v[i], v.v[i + 1], v.v[i + 2], v.v[i + 3]};
        }
    }
}

// ------------------------------------------------------------------------- steps of a chunk
// With step_t = f(dt_t + bias) and c_t = sum of step A over the tokens up to t of the chunk, in
// units of log 2: what decays from token j to token i is 2^(c_i - c_j).  c is summed in 64 bits
// and kept as a whole part and a rest, whose differences are exact to 2^-24: a large step
// (c of thousands) costs the tokens behind it nothing.
template <int Q> struct SelSteps {
    alignas(16) float step[Q];
    alignas(16) float whole[Q], rest[Q];
    alignas(16) float raw[Q];
};

constexpr double kSelLog2e = 1.4426950408889634;

__device__ __forceinline__ double sel_prefix(double v, int lane) {
#pragma unroll
    for (int d = 1; d < NHIP_WAVE; d *= 2) {
        const double other = __shfl_up(v, d);
        if (lane >= d) v += other;
    }
    return v;
}

// One wave; lane t: token t0 + t of the sequence.  Beyond its end step is zero and c goes on as it is.
template <int Q>
__device__ __forceinline__ void sel_steps(SelSteps<Q>& s, const nhip_scan_args& a, const SelSeq& seq,
                                          int t0, int head) {
    const int lane = threadIdx.x & (NHIP_WAVE - 1);
    float step = 0.0f, raw = 0.0f;
    double c = 0.0;
    if (lane < Q && t0 + lane < seq.n) {
        const long long at = a.tokens.starts ? (seq.row0 + t0 + lane) * a.dt.token
                                             : seq.seq * a.dt.seq + (t0 + lane) * a.dt.token;
        raw = sel_element(a.dt.p, a.dt_type, at + head * a.dt.head) + (a.dt_bias ? a.dt_bias[head] : 0.0f);
        step = a.softplus ? sel_softplus(raw) : raw;
        c = (double)step * (double)a.A[head] * kSelLog2e;
        // 2^-2000 is zero in 32 bits, as everything below it
        c = c < -2000.0 ? -2000.0 : (c > 2000.0 ? 2000.0 : c);
    }
    c = sel_prefix(c, lane);
    if (lane < Q) {
        const double whole = rint(c);
        s.step[lane] = step;
        s.raw[lane] = raw;
        s.whole[lane] = (float)whole;
        s.rest[lane] = (float)(c - whole);
    }
}

__device__ __forceinline__ float sel_exp2(float v) { return __builtin_amdgcn_exp2f(v); }

template <int Q>
__device__ __forceinline__ float sel_decay(const SelSteps<Q>& s, int from, int to) {
    return sel_exp2((s.whole[to] - s.whole[from]) + (s.rest[to] - s.rest[from]));
}
template <int Q> __device__ __forceinline__ float sel_decay_from_start(const SelSteps<Q>& s, int to) {
    return sel_exp2(s.whole[to] + s.rest[to]);
}
