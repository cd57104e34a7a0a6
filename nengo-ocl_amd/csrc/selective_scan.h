// The selective scan in chunks of Q tokens, shared by the operator and its gradient.
//
//     S[t] = e^{step_t A} S[t - 1] + step_t x_t (x) B_t,      y_t = S[t] C_t + D x_t
//
// Over a chunk that a state S enters, with c_i the sum of step A up to token i of the chunk:
//     y_i = sum_{j <= i} (C_i . B_j) e^{c_i - c_j} step_j x_j + e^{c_i} S C_i + D x_i
//     S  <- e^{c_Q} S + sum_j e^{c_Q - c_j} step_j x_j (x) B_j
// so that all but one pass over Q x Q weights are matrix products.
#pragma once

#include "selective_mma.h"

// What the walk over the chunks of a sequence does with each
enum SelWalk {
    kSelOutputs = 0,     // y, and the final state
    kSelStates = 1,      // stores the state that enters each chunk
    kSelStatesBack = 2,  // the gradient of the state: from the last chunk to the first, stores what
                         // leaves each chunk:  G <- e^{c_Q} G + sum_i e^{c_i} dy_i (x) C_i
};

struct SelWalkPlan {
    int n_tiles;          // of 64 of the head's dimension
    int vec;              // which operands lie at multiples of 16 bytes: bits below
    long long max_chunks;
    float* states;        // [chunk][head][dim][states]
};
enum { kSelVecX = 1, kSelVecB = 2, kSelVecC = 4, kSelVecY = 8, kSelVecState = 16, kSelVecDy = 32 };

// Tokens of a chunk: 64, or 32 where 256 states would not fit the LDS otherwise.
constexpr int sel_chunk_of(int np) { return np > 128 ? 32 : 64; }

// States are kept in multiples of 32; f(std::integral_constant) for the smallest that holds n.
template <class F> static inline bool sel_with_states(int n, F&& f) {
    using std::integral_constant;
    if (n <= 32) f(integral_constant<int, 32>());
    else if (n <= 64) f(integral_constant<int, 64>());
    else if (n <= 128) f(integral_constant<int, 128>());
    else if (n <= 256) f(integral_constant<int, 256>());
    else return false;
    return true;
}
static inline int sel_chunk_tokens(int n) { return sel_chunk_of(n > 128 ? 256 : 128); }

// Four neighbouring states of a row in memory
__device__ __forceinline__ sel_f4 sel_state_load(const float* p, int n, int states, bool vec) {
    if (vec && n + 4 <= states) return *reinterpret_cast<const sel_f4*>(p + n);
    sel_f4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = n + r < states ? p[n + r] : 0.0f;
    return v;
}
__device__ __forceinline__ void sel_state_store(float* p, int n, int states, bool vec, const sel_f4& v) {
    if (vec && n + 4 <= states) {
        *reinterpret_cast<sel_f4*>(p + n) = v;
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (n + r < states) p[n + r] = v[r];
}

// Four neighbouring elements of a row of an output
template <class T>
__device__ __forceinline__ void sel_store4(T* p, int c, int cols, bool vec, const sel_f4& v) {
    if (vec && c + 4 <= cols) {
        sel_store<T, 4>(p + c, {v[0], v[1], v[2], v[3]});
        return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (c + r < cols) p[c + r] = (T)v[r];
}

template <class Tc, int NP, bool OUTPUTS> struct SelWalkLds {
    static constexpr int Q = sel_chunk_of(NP);
    alignas(16) Tc x[Q * sel_stride<Tc>(64)];
    alignas(16) Tc B[Q * sel_stride<Tc>(NP)];
    alignas(16) Tc C[OUTPUTS ? Q * sel_stride<Tc>(NP) : 8];
    alignas(16) Tc weights[OUTPUTS ? Q * sel_stride<Tc>(Q) : 8];  // [i][j]: (C_i . B_j) e^{c_i - c_j} step_j
    SelSteps<Q> steps;
};

// One work-group walks over the chunks of a sequence for 64 of a head's dimension, 16 to a wave,
// whose part of the state stays in registers: lane l of a wave holds row p = l % 16 of it, the states
// 16 t + 4 (l / 16) + r in register r of tile t -- the order of a fragment over the states, so that
// the state is an operand of the next chunk's products as it is.
template <class T, class Tc, int NP, int WALK>
__global__ __launch_bounds__(NHIP_WG) void sel_walk_kernel(nhip_scan_args a, SelWalkPlan plan) {
    using Lds = SelWalkLds<Tc, NP, WALK == kSelOutputs>;
    constexpr int Q = Lds::Q, QT = Q / 16, NT = NP / 16;
    constexpr int SX = sel_stride<Tc>(64), SN = sel_stride<Tc>(NP), SW = sel_stride<Tc>(Q);
    constexpr int kSplits = SelSplit<Tc>::n;
    extern __shared__ __align__(16) char lds_bytes[];
    Lds& s = *reinterpret_cast<Lds*>(lds_bytes);

    // neighbouring heads read the same B and C: they go to one die, whose L2 holds them
    const int id = nhip_xcd_remap(blockIdx.x, gridDim.x);
    const int tile = id % plan.n_tiles, head = (id / plan.n_tiles) % a.n_heads;
    const SelSeq seq = sel_seq(a.tokens, id / (plan.n_tiles * a.n_heads), Q);
    const int group = head / (a.n_heads / a.n_groups);
    const int wave = threadIdx.x / NHIP_WAVE, l = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
    const int p_tile = tile * 64, p = p_tile + wave * 16 + l;
    const int cols = min(64, a.dim - p_tile);
    const bool vec_state = plan.vec & kSelVecState;
    const long long head_state = (long long)a.dim * a.states;

    sel_f4 state[NT];
    {
        const float* from = WALK == kSelStatesBack ? a.dfinal : a.initial;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            state[t] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (from && p < a.dim)
                state[t] = sel_state_load(from + ((long long)seq.seq * a.n_heads + head) * head_state + (long long)p * a.states,
                                          16 * t + 4 * g, a.states, vec_state);
        }
    }
    if constexpr (WALK == kSelOutputs)
        for (int q = threadIdx.x; q < Q * SW; q += NHIP_WG) s.weights[q] = (Tc)0.0f;  // (above the diagonal for good)
    const float D = WALK == kSelOutputs && a.D ? a.D[head] : 0.0f;

    const int n_chunks = (seq.n + Q - 1) / Q;
    for (int k = 0; k < n_chunks; ++k) {
        const int chunk = WALK == kSelStatesBack ? n_chunks - 1 - k : k;
        const int t0 = chunk * Q, n = min(Q, seq.n - t0);
        __syncthreads();
        const nhip_rows& x = WALK == kSelStatesBack ? a.dy : a.x;
        const nhip_rows& B = WALK == kSelStatesBack ? a.C : a.B;
        sel_stage<T, Tc, Q, 64>(s.x, sel_row<T>(x, a.tokens, seq, t0) + head * x.head + p_tile, x.token, n, cols,
                                plan.vec & (WALK == kSelStatesBack ? kSelVecDy : kSelVecX));
        sel_stage<T, Tc, Q, NP>(s.B, sel_row<T>(B, a.tokens, seq, t0) + group * B.head, B.token, n, a.states,
                                plan.vec & (WALK == kSelStatesBack ? kSelVecC : kSelVecB));
        if constexpr (WALK == kSelOutputs)
            sel_stage<T, Tc, Q, NP>(s.C, sel_row<T>(a.C, a.tokens, seq, t0) + group * a.C.head, a.C.token, n,
                                    a.states, plan.vec & kSelVecC);
        if (wave == 0) sel_steps<Q>(s.steps, a, seq, t0, head);
        __syncthreads();

        SelFrag<Tc> xf[QT / 2];  // row p of x transposed, over the tokens
#pragma unroll
        for (int ks = 0; ks < QT / 2; ++ks) xf[ks] = sel_cols(s.x + 32 * ks * SX + 16 * wave, SX, l, g);

        if constexpr (WALK == kSelOutputs) {
            for (int t = wave; t < QT * (QT + 1) / 2; t += 4) {
                int it = 0;
                while ((it + 1) * (it + 2) / 2 <= t) ++it;
                const int jt = t - it * (it + 1) / 2;
                sel_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < NP / 32; ++ks)
                    sel_mma(acc, sel_rows(s.B + (16 * jt + l) * SN + 32 * ks, g),
                            sel_rows(s.C + (16 * it + l) * SN + 32 * ks, g));
                const int i = 16 * it + l, j0 = 16 * jt + 4 * g;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    v[r] = j0 + r <= i ? acc[r] * sel_decay(s.steps, j0 + r, i) * s.steps.step[j0 + r] : 0.0f;
                sel_store<Tc, 4>(s.weights + i * SW + j0, v);
            }
            __syncthreads();
            SelFrag<Tc> sf[NP / 32];  // the state that enters, over the states
#pragma unroll
            for (int ks = 0; ks < NP / 32; ++ks)
#pragma unroll
                for (int e = 0; e < 8; ++e) sf[ks].set(e, state[2 * ks + (e >> 2)][e & 3]);
#pragma unroll
            for (int it = 0; it < QT; ++it) {
                const int i = 16 * it + l;
                sel_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < NP / 32; ++ks)
                    sel_mma(acc, sf[ks], sel_rows(s.C + i * SN + 32 * ks, g));
                acc *= sel_decay_from_start(s.steps, i);
#pragma unroll
                for (int ks = 0; ks <= it / 2; ++ks) sel_mma(acc, xf[ks], sel_rows(s.weights + i * SW + 32 * ks, g));
                if (i < n && p_tile + 16 * wave < a.dim) {
                    const int c = 16 * wave + 4 * g;
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[r] = fmaf(D, (float)s.x[i * SX + c + r], acc[r]);
                    T* row = static_cast<T*>(a.y) + ((seq.row0 + t0 + i) * a.n_heads + head) * a.dim + p_tile;
                    sel_store4(row, c, cols, plan.vec & kSelVecY, acc);
                }
            }
        } else if (p < a.dim && seq.chunk + chunk < plan.max_chunks) {
            float* out = plan.states + ((seq.chunk + chunk) * a.n_heads + head) * head_state + (long long)p * a.states;
#pragma unroll
            for (int t = 0; t < NT; ++t) sel_state_store(out, 16 * t + 4 * g, a.states, vec_state, state[t]);
        }

        const float all = sel_decay_from_start(s.steps, Q - 1);
#pragma unroll
        for (int t = 0; t < NT; ++t) state[t] *= all;
#pragma unroll
        for (int ks = 0; ks < QT / 2; ++ks) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = 32 * ks + 16 * (e >> 2) + 4 * g + (e & 3);
                const float w = WALK == kSelStatesBack ? sel_decay_from_start(s.steps, j)
                                                       : sel_decay(s.steps, j, Q - 1) * s.steps.step[j];
                v[e] = xf[ks].get(e) * w;
            }
            SelFrag<Tc> split[kSplits];
            sel_split<Tc>(v, split);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const SelFrag<Tc> bf = sel_cols(s.B + 32 * ks * SN + 16 * t, SN, l, g);
#pragma unroll
                for (int q = 0; q < kSplits; ++q) sel_mma(state[t], bf, split[q]);
            }
        }
    }
    float* end = WALK == kSelOutputs ? a.final : WALK == kSelStatesBack ? a.dinitial : nullptr;
    if (end && p < a.dim) {
        end += ((long long)seq.seq * a.n_heads + head) * head_state + (long long)p * a.states;
#pragma unroll
        for (int t = 0; t < NT; ++t) sel_state_store(end, 16 * t + 4 * g, a.states, vec_state, state[t]);
    }
}

// ------------------------------------------------------------------------------- host side
static inline bool sel_rows_aligned(const nhip_rows& r, int type) {
    const int v = 16 / sel_size(type);
    return sel_aligned(r.p, 16) && r.seq % v == 0 && r.token % v == 0 && r.head % v == 0;
}

static inline int sel_scan_check(const nhip_scan_args* a) {
    if (!a || !a->A || a->n_heads <= 0 || a->dim <= 0 || a->n_groups <= 0 || a->n_heads % a->n_groups) return NHIP_E_BADARG;
    if (a->states < 1 || a->states > 256 || !sel_tokens_ok(a->tokens)) return NHIP_E_BADARG;
    if (a->type < NHIP_F32 || a->type > NHIP_F16 || a->dt_type < NHIP_F32 || a->dt_type > NHIP_F16) return NHIP_E_BADARG;
    if (a->tokens.n_tokens && (!a->x.p || !a->dt.p || !a->B.p || !a->C.p)) return NHIP_E_BADARG;
    if (sel_max_chunks(a->tokens, 32) > 0x7fffffffLL) return NHIP_E_BADARG;
    const long long groups = (long long)a->tokens.n_seqs * a->n_heads * ((a->dim + 63) / 64);
    return groups > 0x7fffffffLL ? NHIP_E_BADARG : 0;
}

static inline SelWalkPlan sel_walk_plan(const nhip_scan_args& a, float* states) {
    SelWalkPlan p;
    p.n_tiles = (a.dim + 63) / 64;
    p.states = states;
    p.max_chunks = sel_max_chunks(a.tokens, sel_chunk_tokens(a.states));
    p.vec = 0;
    if (sel_rows_aligned(a.x, a.type)) p.vec |= kSelVecX;
    if (sel_rows_aligned(a.B, a.type)) p.vec |= kSelVecB;
    if (sel_rows_aligned(a.C, a.type)) p.vec |= kSelVecC;
    if (sel_rows_aligned(a.dy, a.type)) p.vec |= kSelVecDy;
    if (a.dim % 4 == 0 && sel_aligned(a.y, 16) && sel_aligned(a.dx, 16)) p.vec |= kSelVecY;
    if (a.states % 4 == 0 && sel_aligned(a.initial, 16) && sel_aligned(a.final, 16) && sel_aligned(a.dfinal, 16) &&
        sel_aligned(a.dinitial, 16) && sel_aligned(states, 16) && sel_aligned(a.dB, 16) && sel_aligned(a.dC, 16))
        p.vec |= kSelVecState;
    return p;
}

// The LDS of a launch above 64 KiB has to be asked for once per kernel and device.
template <class K> static inline int sel_allow_lds(K kernel, size_t bytes) {
    if (bytes <= 65536) return 0;
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)bytes);
}

// 16-bit floats have their own products on the matrix cores only in their own type; bfloat16's range does
// not hold their precision, so they take the 32-bit ones.
template <class T> struct SelCompute { using type = float; };
template <> struct SelCompute<__bf16> { using type = __bf16; };

template <int WALK> static inline int sel_walk(hipStream_t stream, const nhip_scan_args& a, const SelWalkPlan& plan) {
    const unsigned grid = (unsigned)((long long)a.tokens.n_seqs * a.n_heads * plan.n_tiles);
    if (!grid) return 0;
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        using Tc = typename SelCompute<T>::type;
        sel_with_states(a.states, [&](auto np) {
            constexpr int NP = decltype(np)::value;
            constexpr size_t lds = sizeof(SelWalkLds<Tc, NP, WALK == kSelOutputs>);
            auto kernel = sel_walk_kernel<T, Tc, NP, WALK>;
            rc = sel_allow_lds(kernel, lds);
            if (rc) return;
            if (WALK == kSelOutputs) NHIP_LAUNCH(kernel, dim3(grid), dim3(NHIP_WG), lds, stream, a, plan);
            else NHIP_LAUNCH_FIRST(kernel, dim3(grid), dim3(NHIP_WG), lds, stream, a, plan);
            rc = (int)hipGetLastError();
        });
    });
    return rc;
}
