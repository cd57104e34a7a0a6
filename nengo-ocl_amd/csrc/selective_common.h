// Shared parts of the operators for blocks that filter selectively (short causal convolution,
// selective scan, gated norm): element types, chunks of ragged sequences, small reductions.
#pragma once

#include <cstdint>

#include "nhip_common.h"

typedef float sel_f4 __attribute__((ext_vector_type(4)));

#define SEL_MAX_GRID_Y 65535
#define SEL_MAX_GROUPS ((1LL << 32) / NHIP_WG - 1)  // work-groups along x: an axis has fewer than 2^32 threads
#define SEL_MAX_TOKENS 0x7fff0000LL  // (room for a chunk behind the last token in 32 bits)

// ------------------------------------------------------------------------------ element types
// Sums, states and statistics are float32; a value is rounded to a 16-bit type once, when it
// is stored (to nearest, ties to even).  Operands of matrix products that are no inputs go in as
// several parts of 16 bits (SelSplit).
template <class T, int N> struct alignas(sizeof(T) * N) SelPack { T v[N]; };

template <class T, int N>
__device__ __forceinline__ void sel_load(const T* p, float (&out)[N]) {
    const SelPack<T, N> q = *reinterpret_cast<const SelPack<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = (float)q.v[i];
}

template <class T, int N>
__device__ __forceinline__ void sel_store(T* p, const float (&in)[N]) {
    SelPack<T, N> q;
#pragma unroll
    for (int i = 0; i < N; ++i) q.v[i] = (T)in[i];
    *reinterpret_cast<SelPack<T, N>*>(p) = q;
}

// The same past the caches: a launch ends when the L2s' written lines are in memory, and these are there already
// (the convolution of 8 x 2048 tokens, 2304 channels, bfloat16: 41.7 -> 30.9 us).  At any size: a small call takes what its
// launch takes either way.
template <class T, int N>
__device__ __forceinline__ void sel_store_past(T* p, const float (&in)[N]) {
    typedef unsigned words __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(T) * N == 16) {
        SelPack<T, N> q;
#pragma unroll
        for (int i = 0; i < N; ++i) q.v[i] = (T)in[i];
        __builtin_nontemporal_store(__builtin_bit_cast(words, q), reinterpret_cast<words*>(p));
    } else {
        sel_store<T, N>(p, in);
    }
}

// Calls f(element type) for the type code; false where there is no such type.
template <class F> static inline bool sel_with_type(int type, F&& f) {
    switch (type) {
        case NHIP_F32: f(float()); return true;
        case NHIP_BF16: f(__bf16()); return true;
        case NHIP_F16: f(_Float16()); return true;
    }
    return false;
}

static inline int sel_size(int type) { return type == NHIP_F32 ? 4 : 2; }

static inline bool sel_aligned(const void* p, int bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0;
}

// An element whose type is known at run time only (the steps of the scan: one per token and head)
__device__ __forceinline__ float sel_element(const void* p, int type, long long i) {
    if (type == NHIP_F32) return static_cast<const float*>(p)[i];
    if (type == NHIP_BF16) return (float)static_cast<const __bf16*>(p)[i];
    return (float)static_cast<const _Float16*>(p)[i];
}

__device__ __forceinline__ void sel_set_element(void* p, int type, long long i, float v) {
    if (type == NHIP_F32) static_cast<float*>(p)[i] = v;
    else if (type == NHIP_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
    else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// 1 / (1 + exp(-v)): one at +inf and zero at -inf; v_rcp_f32 is good to one unit in the last place.
__device__ __forceinline__ float sel_sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896341f));
}

// exp(v): 2^v' with the whole part of v' = v log2(e) set aside, so that its rounding costs nothing.  v is cut first, far
// beyond what 32 bits hold (what is no number stays none): the product of a larger one is rounded to more than
// the 128 that its rest may have, and that of an infinite one has no rest.
__device__ __forceinline__ float sel_exp(float v) {
    v = v < -200.0f ? -200.0f : (v > 200.0f ? 200.0f : v);
    const float whole = rintf(v * 1.44269504088896341f);
    const float rest = fmaf(v, 1.925963033500e-8f, fmaf(v, 1.44269502162933349609f, -whole));  // log2(e) in two parts
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(rest), (int)fmaxf(whole, -300.0f));  // (a number in any case)
}

// max(v, 0) + log(1 + exp(-|v|)), without loss for large negative v: with u = exp(-|v|) and w = 1 + u as
// rounded, log(1 + u) = log(w) u / (w - 1) to first order in the rounding (Kahan).
__device__ __forceinline__ float sel_softplus(float v) {
    const float u = sel_exp(-fabsf(v)), w = 1.0f + u, d = w - 1.0f;
    const float log_w = __builtin_amdgcn_logf(w) * 0.693147180559945309f;
    return fmaxf(v, 0.0f) + (d > 0.0f ? log_w * (u * __builtin_amdgcn_rcpf(d)) : u);
}

// ---------------------------------------------------------------------- chunks of sequences
// A sequence is worked on in chunks of `q` tokens that begin with its first one, so that no
// chunk holds tokens of two sequences; an empty sequence has one chunk (it still has a final
// state to hand on).
struct SelSeq {
    int seq;           // -1: there is no such chunk
    int n;             // tokens of the sequence
    int chunk;         // first chunk of the sequence (sel_seq_of_chunk: the chunk within the sequence)
    long long row0;    // where its first token lies among the rows of contiguous outputs
};

__host__ __device__ __forceinline__ int sel_chunks(int n, int q) { return n > 0 ? (n + q - 1) / q : 1; }

__device__ __forceinline__ int sel_bound(const nhip_tokens& t, int s) {
    const int v = t.starts[s];
    const int top = (int)t.n_tokens;
    return v < 0 ? 0 : (v > top ? top : v);
}

__device__ __forceinline__ int sel_length(const nhip_tokens& t, int s) {
    const int n = sel_bound(t, s + 1) - sel_bound(t, s);
    return n > 0 ? n : 0;
}

// The most chunks that these tokens can make: every sequence ends at most one chunk early.
static inline long long sel_max_chunks(const nhip_tokens& t, int q) {
    if (!t.starts) return (long long)t.n_seqs * sel_chunks(t.length, q);
    return t.n_tokens / q + t.n_seqs;
}

// Sequences that overlap (offsets that go back) can make more chunks than sel_max_chunks: those
// beyond it have no work-group, and whoever counts to them stays below 2^31.
__device__ __forceinline__ int sel_add_chunks(int a, int b) { return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu); }

// Which sequence chunk c belongs to.  Ragged: the 64 lanes of a wave take a sequence each and
// add up their chunks (uniform over the wave, no table, no launch of its own; 64 sequences
// cost about as much as a read of memory).
__device__ __forceinline__ SelSeq sel_seq_of_chunk(const nhip_tokens& t, int c, int q) {
    SelSeq r;
    if (!t.starts) {
        const int per = sel_chunks(t.length, q);
        r.seq = c / per;
        r.chunk = c - r.seq * per;
        r.n = t.length;
        r.row0 = (long long)r.seq * t.length;
        if (r.seq >= t.n_seqs) r.seq = -1;
        return r;
    }
    const int lane = threadIdx.x & (NHIP_WAVE - 1);
    int before = 0;
    r.seq = -1; r.n = 0; r.chunk = 0; r.row0 = 0;
    for (int s0 = 0; s0 < t.n_seqs; s0 += NHIP_WAVE) {
        const int s = s0 + lane;
        const int n = s < t.n_seqs ? sel_length(t, s) : 0;
        const int mine = s < t.n_seqs ? sel_chunks(n, q) : 0;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < NHIP_WAVE; d *= 2) {
            const int other = __shfl_up(sum, d);
            if (lane >= d) sum = sel_add_chunks(sum, other);
        }
        const int total = __builtin_amdgcn_readlane(sum, NHIP_WAVE - 1);
        if (c < sel_add_chunks(before, total)) {
            const unsigned long long past = __ballot(sel_add_chunks(before, sum) > c);
            const int at = __ffsll((long long)past) - 1;
            // (in scalar registers: they are the same in all lanes, which the compiler cannot see)
            const int lane_of = __builtin_amdgcn_readfirstlane(at);
            r.seq = s0 + lane_of;
            r.n = __builtin_amdgcn_readlane(n, lane_of);
            r.chunk = c - before - (__builtin_amdgcn_readlane(sum, lane_of) - __builtin_amdgcn_readlane(mine, lane_of));
            r.row0 = __builtin_amdgcn_readfirstlane(sel_bound(t, r.seq));
            return r;
        }
        before += total;
    }
    return r;
}

// Sequence s, and the number of chunks before its first one (uniform over the wave).
__device__ __forceinline__ SelSeq sel_seq(const nhip_tokens& t, int s, int q) {
    SelSeq r;
    r.seq = s;
    if (!t.starts) {
        r.n = t.length;
        r.chunk = s * sel_chunks(t.length, q);
        r.row0 = (long long)s * t.length;
        return r;
    }
    const int lane = threadIdx.x & (NHIP_WAVE - 1);
    int sum = 0;
    for (int i = lane; i < s; i += NHIP_WAVE) sum = sel_add_chunks(sum, sel_chunks(sel_length(t, i), q));
#pragma unroll
    for (int d = 1; d < NHIP_WAVE; d *= 2) sum = sel_add_chunks(sum, __shfl_xor(sum, d));
    r.chunk = __builtin_amdgcn_readfirstlane(sum);
    r.n = __builtin_amdgcn_readfirstlane(sel_length(t, s));
    r.row0 = __builtin_amdgcn_readfirstlane(sel_bound(t, s));
    return r;
}

// Element 0 of the row of token t of a sequence
template <class T>
__device__ __forceinline__ const T* sel_row(const nhip_rows& a, const nhip_tokens& k, const SelSeq& s,
                                            int t) {
    const long long at = k.starts ? (s.row0 + t) * a.token : s.seq * a.seq + t * a.token;
    return static_cast<const T*>(a.p) + at;
}

// ------------------------------------------------------------------------------- reductions
__device__ __forceinline__ float sel_wave_sum(float v) {
#pragma unroll
    for (int d = NHIP_WAVE / 2; d > 0; d /= 2) v += __shfl_xor(v, d);
    return v;
}

// Over the 16 lanes of a quarter of the wave, by rotations within it
template <int N> __device__ __forceinline__ float sel_rotated(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float sel_row_sum(float v) {
    v += sel_rotated<8>(v);
    v += sel_rotated<4>(v);
    v += sel_rotated<2>(v);
    return v + sel_rotated<1>(v);
}

// Column sums of parts[rows][n], always in the same order: 16 waves take a share of the rows each.
// The columns go to up to three results: those below `split` to out[(c % width) * stride + c / width]
// (a transposition where the rows hold another order than the result), those below `split2` to out2,
// the others to out3; NULL: not wanted.
struct SelReduce {
    const float* parts;
    long long n;
    int rows;
    long long split, split2;
    float* out;
    long long width, stride;
    float *out2, *out3;
};
#define SEL_REDUCE_WAVES 16
#define SEL_MAX_SUMS (((1LL << 32) / (SEL_REDUCE_WAVES * NHIP_WAVE) - 1) * NHIP_WAVE)  // columns: an axis has fewer than 2^32 threads

static __global__ __launch_bounds__(SEL_REDUCE_WAVES * NHIP_WAVE) void sel_reduce_kernel(SelReduce a) {
    __shared__ float s[SEL_REDUCE_WAVES][NHIP_WAVE];
    const int lane = threadIdx.x & (NHIP_WAVE - 1), wave = threadIdx.x / NHIP_WAVE;
    const long long c = (long long)blockIdx.x * NHIP_WAVE + lane;
    float sum = 0.0f;
    if (c < a.n) {
        const int per = (a.rows + SEL_REDUCE_WAVES - 1) / SEL_REDUCE_WAVES;
        const int r1 = min(a.rows, (wave + 1) * per);
#pragma unroll 8
        for (int r = wave * per; r < r1; ++r) sum += a.parts[r * a.n + c];
    }
    s[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && c < a.n) {
#pragma unroll
        for (int w = 1; w < SEL_REDUCE_WAVES; ++w) sum += s[w][lane];
        if (c < a.split) {
            if (a.out) a.out[(c % a.width) * a.stride + c / a.width] = sum;
        } else if (c < a.split2) {
            if (a.out2) a.out2[c - a.split] = sum;
        } else if (a.out3) {
            a.out3[c - a.split2] = sum;
        }
    }
}

static inline int sel_reduce(hipStream_t stream, const SelReduce& a) {
    const dim3 grid((unsigned)((a.n + NHIP_WAVE - 1) / NHIP_WAVE));
    NHIP_LAUNCH_LAST(sel_reduce_kernel, grid, dim3(SEL_REDUCE_WAVES * NHIP_WAVE), 0, stream, a);
    NHIP_LAUNCH_CHECK();
    return 0;
}

// The LDS of a launch above 64 KiB has to be asked for, once per kernel and device (again with each call, which changes
// nothing and costs less than to look it up): on the stream's device, which need not be the current one.
template <class K> static inline int sel_allow_lds(hipStream_t stream, K kernel, size_t bytes) {
    if (bytes <= 65536) return 0;
    int current = 0;
    hipDevice_t device = 0;
    if (int e = (int)hipGetDevice(&current)) return e;
    if (int e = (int)hipStreamGetDevice(stream, &device)) return e;
    if (device != current)
        if (int e = (int)hipSetDevice(device)) return e;
    int rc = (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)bytes);
    if (device != current) {
        const int back = (int)hipSetDevice(current);
        rc = rc ? rc : back;
    }
    return rc;
}

static inline bool sel_tokens_ok(const nhip_tokens& t) {
    if (t.n_seqs < 0 || t.n_tokens < 0 || t.n_tokens > SEL_MAX_TOKENS) return false;
    if (!t.starts) return t.length >= 0 && (long long)t.n_seqs * t.length == t.n_tokens;
    return true;
}
