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
// them.  The other operand holds inputs, which are exact.  What leads to a result of 16 bits and to nothing else goes in as
// `out` parts: two bfloat16 hold 16 bits, off by 2^-16 at most where the result's own rounding is 2^-8.
template <class Tc> struct SelSplit { static constexpr int n = 1, out = 1; };
template <> struct SelSplit<__bf16> { static constexpr int n = 3, out = 2; };

// acc += first second over 32 values of k.  32-bit elements: eight products of four k.
__device__ __forceinline__ void sel_mma(sel_f4& acc, const SelFrag<__bf16>& a, const SelFrag<__bf16>& b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, acc, 0, 0, 0);
}
__device__ __forceinline__ void sel_mma(sel_f4& acc, const SelFrag<float>& a, const SelFrag<float>& b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc, 0, 0, 0);
}

// Waits until the products before it are done and leaves their sums in vector registers.  A result that
// is read behind a branch needs this: the wait states between a matrix instruction and what
// reads its registers are the program's to keep, and this compiler counts them within a block
// (roc-7.2.0: a branch right behind the instruction led to reads one wait state after it, which
// returned the last of the four registers' old value).
template <int N> __device__ __forceinline__ void sel_settle(sel_f4 (&a)[N]) {
#pragma unroll
    for (int i = 0; i < N - 1; ++i) asm volatile("" : "+v"(a[i]));
    asm volatile("s_nop 15" : "+v"(a[N - 1]));
}
__device__ __forceinline__ void sel_settle(sel_f4& a) { asm volatile("s_nop 15" : "+v"(a)); }

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

// A matrix in LDS kept as tiles of 16 x 16, of which only some are held: where the four elements `four` of a row of a
// tile lie, and fragments over two tiles, along their rows and across.  16-bit elements: 512 bytes without gaps, fours of
// rows 4 apart in other places, so that 16 lanes meet no bank twice (rows of 32 bytes in their order do, four
// times).  32-bit elements: 16 bytes between the rows.
template <class Tc> struct SelTile {
    static constexpr bool kSwapped = sizeof(Tc) == 2;
    static constexpr int kRow = kSwapped ? 16 : 20, kSize = 16 * kRow;
    static __device__ __forceinline__ int at(int row, int four) {
        return kRow * row + 4 * (kSwapped ? four ^ (row >> 2) : four);
    }
    static __device__ __forceinline__ SelFrag<__bf16> rows(const __bf16* lo, const __bf16* hi, int l, int g) {
        const sel_b4 a = *reinterpret_cast<const sel_b4*>(lo + at(l, g)), b = *reinterpret_cast<const sel_b4*>(hi + at(l, g));
        SelFrag<__bf16> f;
        f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        return f;
    }
    static __device__ __forceinline__ SelFrag<float> rows(const float* lo, const float* hi, int l, int g) {
        const sel_f4 a = *reinterpret_cast<const sel_f4*>(lo + at(l, g)), b = *reinterpret_cast<const sel_f4*>(hi + at(l, g));
        SelFrag<float> f;
#pragma unroll
        for (int e = 0; e < 4; ++e) { f.v[e] = a[e]; f.v[4 + e] = b[e]; }
        return f;
    }
    static __device__ __forceinline__ SelFrag<__bf16> cols(const __bf16* lo, const __bf16* hi, int l, int g) {
        typedef __attribute__((address_space(3))) sel_b4* lds;
        const int mine = at(4 * g + (l >> 2), l & 3);
        const sel_b4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds)(lo + mine));
        const sel_b4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds)(hi + mine));
        SelFrag<__bf16> f;
        f.v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        return f;
    }
    static __device__ __forceinline__ SelFrag<float> cols(const float* lo, const float* hi, int l, int g) {
        SelFrag<float> f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f.v[e] = (e < 4 ? lo : hi)[kRow * (4 * g + (e & 3)) + l];
        return f;
    }
};

// Float32 values as parts that add up to them.  (bfloat16: two values at a time, which is one instruction to
// round them and one for each to widen it; element by element the compiler rounds each alone)
template <int N, int P> __device__ __forceinline__ void sel_parts(const float (&x)[N], unsigned (&out)[P][N / 2]) {
    typedef float two __attribute__((ext_vector_type(2)));
    typedef __bf16 two_b __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
        two rest = {x[2 * e], x[2 * e + 1]};
#pragma unroll
        for (int s = 0; s < P; ++s) {
            out[s][e] = __builtin_bit_cast(unsigned, __builtin_convertvector(rest, two_b));
            rest.x -= __uint_as_float(out[s][e] << 16);
            rest.y -= __uint_as_float(out[s][e] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ void sel_split(const float (&x)[8], SelFrag<float> (&f)[1]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[0].v[e] = x[e];
}
template <int P> __device__ __forceinline__ void sel_split(const float (&x)[8], SelFrag<__bf16> (&f)[P]) {
    unsigned out[P][4];
    sel_parts(x, out);
#pragma unroll
    for (int s = 0; s < P; ++s) f[s].v = __builtin_bit_cast(sel_b8, out[s]);
}
// Four of them to LDS, the parts of each at `to` and `rest`
__device__ __forceinline__ void sel_store_parts(float* to, float*, const float (&x)[4]) {
    *reinterpret_cast<sel_f4*>(to) = sel_f4{x[0], x[1], x[2], x[3]};
}
__device__ __forceinline__ void sel_store_parts(__bf16* to, __bf16* rest, const float (&x)[4]) {
    unsigned out[2][2];
    sel_parts(x, out);
    *reinterpret_cast<uint2*>(to) = uint2{out[0][0], out[0][1]};
    *reinterpret_cast<uint2*>(rest) = uint2{out[1][0], out[1][1]};
}

// Whether all elements are finite (magnitudes of 16 bits are compared as whole numbers, two at a time), and
// what is left with zeros in the place of those that are not; ones in their place
template <int H, int K> __device__ __forceinline__ bool sel_finite(const SelFrag<__bf16> (&f)[H][K]) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    us2 most = {0, 0};
#pragma unroll
    for (int q = 0; q < H * K; ++q) {
        const u4 m = __builtin_bit_cast(u4, f[q / K][q % K].v);
#pragma unroll
        for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(us2, m[e] & 0x7fff7fffu));
    }
    return most.x < 0x7f80 && most.y < 0x7f80;
}
template <int H, int K> __device__ __forceinline__ bool sel_finite(const SelFrag<float> (&f)[H][K]) {
    float m = 0.0f;
#pragma unroll
    for (int q = 0; q < H * K; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaf(f[q / K][q % K].v[e], 0.0f, m);
    return m == 0.0f;
}
template <class Tc> __device__ __forceinline__ SelFrag<Tc> sel_take_unfinite(SelFrag<Tc>& f) {
    SelFrag<Tc> ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool ok = fabsf(f.get(e)) < INFINITY;
        ones.set(e, ok ? 0.0f : 1.0f);
        if (!ok) f.set(e, 0.0f);
    }
    return ones;
}

// Row length in LDS of `n` elements (a multiple of 32).  Reads of rows (sel_rows) go by 16 lanes of 8 bytes,
// or 8 of 16, over 32 banks: they meet no bank twice with 8 bytes (16) more than the elements.  Reads across
// 16-bit rows (sel_cols) take four rows of 32 bytes at once: 32 bytes more.
template <class Tc> __host__ __device__ constexpr int sel_stride(int n) { return n + 4; }
template <class Tc> __host__ __device__ constexpr int sel_stride_cols(int n) {
    return n + (sizeof(Tc) == 2 ? 16 : 4);
}

// Rows of inputs on their way into LDS through registers, so that the next chunk's are fetched while
// one is worked on: ROWS x COLS elements, zero beyond the n_rows x n_cols (one at least) that are
// there.  VEC: rows begin at multiples of 16 bytes, hold whole packs and lie within 2^31 bytes.  The
// loads are unconditional, from places cut to those that exist, and what is too much is left out when
// it is stored; and VEC is a template's: a load under any condition, uniform or not, is waited for where
// its branch ends, and the packs of a chunk came one after the other (9,000 cycles, not 3,000).
template <class T, class Tc, int ROWS, int COLS, bool VEC> struct SelStage {
    static constexpr int V = 16 / (int)sizeof(T), kRow = COLS / V, kPacks = ROWS * kRow / NHIP_WG;
    static constexpr int kRowStep = NHIP_WG / kRow;  // rows between a thread's packs
    static_assert(ROWS * kRow % NHIP_WG == 0 && NHIP_WG % kRow == 0, "every thread holds as many packs, in one column");
    SelPack<T, V> held[kPacks];

    // (formed anew each time: kept over a loop, the places take the registers of what is worked on)
    static __device__ __forceinline__ unsigned thread() {
        unsigned tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        return tid;
    }

    __device__ __forceinline__ void load(const T* src, long long stride, int n_rows, int n_cols) {
        const unsigned tid = thread();
        const int row = tid / kRow, col = (tid % kRow) * V;
        if constexpr (VEC) {
            const unsigned st = (unsigned)stride * (unsigned)sizeof(T), last = (unsigned)(n_rows - 1) * st;
            const unsigned r0 = (unsigned)row * st, c = (unsigned)min(col, n_cols - V) * (unsigned)sizeof(T);
            unsigned at[kPacks];
            if (n_rows == ROWS) {
#pragma unroll
                for (int q = 0; q < kPacks; ++q) at[q] = r0 + c + (unsigned)(q * kRowStep) * st;
            } else {
#pragma unroll
                for (int q = 0; q < kPacks; ++q) at[q] = min(r0 + (unsigned)(q * kRowStep) * st, last) + c;
            }
#pragma unroll
            for (int q = 0; q < kPacks; ++q)
                held[q] = *reinterpret_cast<const SelPack<T, V>*>(reinterpret_cast<const char*>(src) + at[q]);
        } else {
#pragma unroll
            for (int q = 0; q < kPacks; ++q) {
                const T* p = src + min(row + q * kRowStep, n_rows - 1) * stride;
#pragma unroll
                for (int i = 0; i < V; ++i) held[q].v[i] = p[min(col + i, n_cols - 1)];
            }
        }
    }
    template <int STRIDE, bool WHOLE> __device__ __forceinline__ void put(Tc* dst, int n_rows, int n_cols) const {
        const unsigned tid = thread();
        const int row = tid / kRow, col = (tid % kRow) * V;
        Tc* const first = dst + __mul24(row, STRIDE) + col;
#pragma unroll
        for (int q = 0; q < kPacks; ++q) {
            const int r = row + q * kRowStep;
            Tc* const out = first + q * kRowStep * STRIDE;
            const int there = r < n_rows ? n_cols - col : 0;
            SelPack<Tc, V> v;
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = WHOLE || (VEC ? 0 : i) < there ? (Tc)held[q].v[i] : (Tc)0.0f;
            if constexpr (sizeof(Tc) * V == 16 && STRIDE * sizeof(Tc) % 16 == 0) {
                *reinterpret_cast<SelPack<Tc, V>*>(out) = v;
            } else if constexpr (sizeof(Tc) == 2) {
#pragma unroll
                for (int i = 0; i < V; i += 4)
                    *reinterpret_cast<SelPack<Tc, 4>*>(out + i) = SelPack<Tc, 4>{{v.v[i], v.v[i + 1], v.v[i + 2], v.v[i + 3]}};
            } else {
#pragma unroll
                for (int i = 0; i < V; i += 4)
                    *reinterpret_cast<sel_f4*>(out + i) = sel_f4{(float)v.v[i], (float)v.v[i + 1], (float)v.v[i + 2],
                                                                 (float)v.v[i + 3]};
            }
        }
    }
    template <int STRIDE> __device__ __forceinline__ void store(Tc* dst, int n_rows, int n_cols) const {
        if (n_rows == ROWS && n_cols == COLS) put<STRIDE, true>(dst, n_rows, n_cols);
        else put<STRIDE, false>(dst, n_rows, n_cols);
    }
};

// ------------------------------------------------------------------------- steps of a chunk
// With step_t = f(dt_t + bias) and c_t = sum of step A over the tokens up to t of the chunk, in
// units of log 2: what decays from token j to token i is 2^(c_i - c_j).  c is summed in 64 bits
// and kept as a whole part, whose differences are exact, and a rest of at most 1/2: a large step
// (c of thousands) costs the tokens behind it nothing, and no argument of an exponential is
// rounded to less than 2^-24.  The exponentials of all pairs of tokens are products of two of them.
template <int Q> struct SelSteps {
    alignas(16) float step[Q];
    alignas(16) int whole[Q];
    alignas(16) float to[Q];          // 2^rest_t, and 2^-rest_t step_t: e^{c_i - c_j} step_j is
    alignas(16) float from_step[Q];   //   to_i from_step_j 2^(whole_i - whole_j)
    alignas(16) float from_start[Q];  // 2^c_t
    alignas(16) float to_end[Q];      // 2^(c_Q - c_t)
    alignas(16) float to_end_step[Q];
};

constexpr double kSelLog2e = 1.4426950408889634;

template <int CTRL, int ROWS> __device__ __forceinline__ double sel_dpp(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double(((long long)hi << 32) | (unsigned)lo);
}

// Sum over the lanes up to this one: lanes 1, 2, 4, 8 back within each row of 16, then the last lane
// of the row or rows before.
__device__ __forceinline__ double sel_prefix(double v) {
    v += sel_dpp<0x111, 0xf>(v);
    v += sel_dpp<0x112, 0xf>(v);
    v += sel_dpp<0x114, 0xf>(v);
    v += sel_dpp<0x118, 0xf>(v);
    v += sel_dpp<0x142, 0xa>(v);
    v += sel_dpp<0x143, 0xc>(v);
    return v;
}

__device__ __forceinline__ float sel_exp2(int whole, float rest) {
    return __builtin_ldexpf(__builtin_amdgcn_exp2f(rest), whole);
}

// What lane t of a wave reads for token t0 + t of the sequence, on its way: two halves of an element of 32
// bits, or one of 16 twice, from a place cut to those that exist.  (No load is under a condition: one
// is waited for where its branch ends, here a chunk before it is used.)
struct SelDt {
    unsigned lo, hi;
    __device__ __forceinline__ float value(int type) const {
        const float f32 = __uint_as_float((hi << 16) | lo), bf16 = __uint_as_float(lo << 16);
        const float f16 = (float)__builtin_bit_cast(_Float16, (unsigned short)lo);
        return type == NHIP_F32 ? f32 : type == NHIP_BF16 ? bf16 : f16;
    }
};
struct SelDtRow {  // where a head's begin, and the bytes from token to token and from half to half
    const char* p;
    long long token;
    int half;
};
__device__ __forceinline__ SelDtRow sel_dt_row(const nhip_scan_args& a, const SelSeq& seq, int head) {
    const int size = a.dt_type == NHIP_F32 ? 4 : 2;
    const long long first = a.tokens.starts ? seq.row0 * a.dt.token : seq.seq * a.dt.seq;
    return {static_cast<const char*>(a.dt.p) + (head * a.dt.head + first) * size, a.dt.token * size, size - 2};
}
__device__ __forceinline__ SelDt sel_dt(const SelDtRow& row, int t0, int n) {
    int lane = threadIdx.x & (NHIP_WAVE - 1);
    asm volatile("" : "+v"(lane));  // (the address is formed anew each time: kept, it takes two registers)
    const char* p = row.p + max(0, min(t0 + lane, n - 1)) * row.token;
    SelDt d;
    d.lo = *reinterpret_cast<const unsigned short*>(p);
    d.hi = *reinterpret_cast<const unsigned short*>(p + row.half);
    return d;
}

// One wave; lane t: token t of the chunk, n of which there are, with dt as read.  Beyond them step is
// zero and c goes on as it is.  Returns dt + bias.
template <int Q>
__device__ __forceinline__ float sel_steps(SelSteps<Q>& s, float dt, int n, float A, float bias, bool softplus) {
    int lane = threadIdx.x & (NHIP_WAVE - 1);
    asm volatile("" : "+v"(lane));
    float step = 0.0f, raw = 0.0f;
    double c = 0.0;
    if (lane < Q && lane < n) {
        raw = dt + bias;
        step = softplus ? sel_softplus(raw) : raw;
        c = (double)step * (double)A * kSelLog2e;
        // 2^-2000 is zero in 32 bits, as everything below it
        c = c < -2000.0 ? -2000.0 : (c > 2000.0 ? 2000.0 : c);
    }
    c = sel_prefix(c);
    const double whole = rint(c);
    const int w = whole == whole ? (int)whole : 0;  // (what is no number is so in the rest)
    const float rest = (float)(c - whole);
    const int w_end = __builtin_amdgcn_readlane(w, Q - 1);
    const float rest_end = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(rest), Q - 1));
    if (lane < Q) {
        s.step[lane] = step;
        s.whole[lane] = w;
        s.to[lane] = __builtin_amdgcn_exp2f(rest);
        s.from_step[lane] = __builtin_amdgcn_exp2f(-rest) * step;
        s.from_start[lane] = sel_exp2(w, rest);
        const float to_end = sel_exp2(w_end - w, rest_end - rest);
        s.to_end[lane] = to_end;
        s.to_end_step[lane] = to_end * step;
    }
    return raw;
}
