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

// What a walk over the chunks of a sequence is for
enum SelWalk {
    kSelOutputs = 0,  // y, and the final state
    kSelStates = 1,   // the state that enters each chunk, and (second half of the grid, where asked for) the
                      // gradient of the state that leaves each, from the last chunk to the first:
                      //     G <- e^{c_Q} G + sum_i e^{c_i} dy_i (x) C_i
    kSelEnds = 2,     // only what a segment adds to the state by its end, and how much it keeps of it
};

// Sequences are cut into segments of `chunks` chunks, each a work-group's walk for 64 of a head's
// dimension.  A first launch (kSelEnds) leaves every segment's own contribution, the second begins
// each with the sum over those before it.
struct SelWalkPlan {
    int n_tiles;            // of 64 of the head's dimension
    int vec;                // which operands lie at multiples of 16 bytes: bits below
    int chunks;             // per segment
    int directions;         // 2: both halves
    long long n_segments, n_chunks;
    float* states;          // [direction][chunk][head][dim][states]
    float* ends;            // [direction][segment][head][dim][states], NULL: no sequence has two segments
    float* keeps;           // [direction][segment][head]: what a segment keeps of the state it begins with
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
    static constexpr int SX = sel_stride_cols<Tc>(64), SB = sel_stride_cols<Tc>(NP), SC = sel_stride<Tc>(NP),
                         SW = sel_stride<Tc>(Q);
    alignas(16) Tc x[Q * SX];
    alignas(16) Tc B[Q * SB];
    alignas(16) Tc C[OUTPUTS ? Q * SC : 8];
    alignas(16) Tc weights[OUTPUTS ? Q * SW : 8];  // [i][j]: (C_i . B_j) e^{c_i - c_j} step_j
    SelSteps<Q> steps[2];                          // of this chunk and the next
};

// Adds what elements of x that are no finite numbers contribute to rows that read them, one by one: in
// the products they would reach the tokens in front of them too, as zero times infinity.
template <class Tc, int Q, int SX, int SW>
__device__ void sel_add_unfinite(sel_f4& acc, const Tc* x, const Tc* weights, int c, int i) {
    for (int j = 0; j <= i; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = (float)x[j * SX + c + r];
            if (!(fabsf(v) < INFINITY)) acc[r] = fmaf((float)weights[i * SW + j], v, acc[r]);
        }
}

// One work-group walks over the chunks of a segment for 64 of a head's dimension, 16 to a wave, whose
// part of the state stays in registers: lane l of a wave holds row p = l % 16 of it, the states
// 16 t + 4 (l / 16) + r in register r of tile t -- the order of a fragment over the states, so that
// the state is an operand of the next chunk's products as it is.  The inputs of the next chunk are
// fetched, and its steps formed, while one is worked on.
template <class T, class Tc, int NP, int WALK>
__global__ __launch_bounds__(NHIP_WG) void sel_walk_kernel(nhip_scan_args a, SelWalkPlan plan) {
    constexpr bool kOut = WALK == kSelOutputs;
    using Lds = SelWalkLds<Tc, NP, kOut>;
    constexpr int Q = Lds::Q, QT = Q / 16, QK = Q / 32, NT = NP / 16, NK = NP / 32;
    constexpr int SX = Lds::SX, SB = Lds::SB, SC = Lds::SC, SW = Lds::SW;
    constexpr int kTiles = QT * (QT + 1) / 2, kMyTiles = (kTiles + 3) / 4;
    constexpr int kSplits = SelSplit<Tc>::n;
    extern __shared__ __align__(16) char lds_bytes[];
    Lds& s = *reinterpret_cast<Lds*>(lds_bytes);

    // neighbouring heads read the same B and C: they go to one die, whose L2 holds them
    const int groups = gridDim.x / plan.directions;
    const int back = blockIdx.x >= groups;
    const int id = nhip_xcd_remap(blockIdx.x - back * groups, groups);
    const int tile = id % plan.n_tiles, head = (id / plan.n_tiles) % a.n_heads;
    const int segment = id / (plan.n_tiles * a.n_heads);
    const SelSeq seq = sel_seq_of_chunk(a.tokens, segment, Q * plan.chunks);
    if (seq.seq < 0) return;
    const int n_segments = sel_chunks(seq.n, Q * plan.chunks);
    // (nobody begins with what the last one, or going back the first, adds)
    if (WALK == kSelEnds && seq.chunk == (back ? 0 : n_segments - 1)) return;
    const int group = head / (a.n_heads / a.n_groups);
    const int wave = threadIdx.x / NHIP_WAVE, l = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
    const int p_tile = tile * 64, p = p_tile + wave * 16 + l;
    const int cols = min(64, a.dim - p_tile);
    const bool vec_state = plan.vec & kSelVecState;
    const long long head_state = (long long)a.dim * a.states;
    const long long my_state = head * head_state + (long long)p * a.states, all_states = a.n_heads * head_state;
    float* const ends = plan.ends ? plan.ends + back * plan.n_segments * all_states : nullptr;

    sel_f4 state[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) state[t] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (WALK != kSelEnds && p < a.dim) {
        const float* from = back ? a.dfinal : a.initial;
        if (from)
#pragma unroll
            for (int t = 0; t < NT; ++t)
                state[t] = sel_state_load(from + seq.seq * all_states + my_state, 16 * t + 4 * g, a.states, vec_state);
        // the segments walked before this one, in their order
        const int first = segment - seq.chunk, before = back ? n_segments - 1 - seq.chunk : seq.chunk;
        for (int k = 0; k < before; ++k) {
            const int other = first + (back ? n_segments - 1 - k : k);
            const float keeps = plan.keeps[(back * plan.n_segments + other) * a.n_heads + head];
            const float* end = ends + other * all_states + my_state;
#pragma unroll
            for (int t = 0; t < NT; ++t)
                state[t] = state[t] * keeps + sel_state_load(end, 16 * t + 4 * g, a.states, vec_state);
        }
    }
    if constexpr (kOut)
        for (int q = threadIdx.x; q < Q * SW; q += NHIP_WG) s.weights[q] = (Tc)0.0f;  // (above the diagonal for good)

    const nhip_rows& x = back ? a.dy : a.x;
    const nhip_rows& B = back ? a.C : a.B;
    const bool vec_x = plan.vec & (back ? kSelVecDy : kSelVecX), vec_B = plan.vec & (back ? kSelVecC : kSelVecB);
    const float D = kOut && a.D ? a.D[head] : 0.0f, A = a.A[head], bias = a.dt_bias ? a.dt_bias[head] : 0.0f;
    // chunks of the sequence that this segment holds, and the token at which walk number k of them begins
    const int chunk0 = seq.chunk * plan.chunks;
    const int n_chunks = min(plan.chunks, (seq.n + Q - 1) / Q - chunk0);
    auto token = [&](int k) { return (chunk0 + (back ? n_chunks - 1 - k : k)) * Q; };
    const int first_chunk = WALK == kSelStates ? sel_seq(a.tokens, seq.seq, Q).chunk : 0;

    SelStage<T, Tc, Q, 64> stage_x;
    SelStage<T, Tc, Q, NP> stage_B, stage_C;
    auto fetch = [&](int k) {
        const int t0 = token(k), n = min(Q, seq.n - t0);
        stage_x.load(sel_row<T>(x, a.tokens, seq, t0) + head * x.head + p_tile, x.token, n, cols, vec_x);
        stage_B.load(sel_row<T>(B, a.tokens, seq, t0) + group * B.head, B.token, n, a.states, vec_B);
        if constexpr (kOut)
            stage_C.load(sel_row<T>(a.C, a.tokens, seq, t0) + group * a.C.head, a.C.token, n, a.states,
                         plan.vec & kSelVecC);
    };
    // the last wave, which has the fewest tiles, forms the steps
    constexpr int kStepWave = 3;
    float dt = 0.0f, keeps = 1.0f;
    if (n_chunks > 0) {
        fetch(0);
        if (wave == kStepWave) {
            dt = sel_dt<Q>(a, seq, token(0), head);
            sel_steps<Q>(s.steps[0], dt, seq.n - token(0), A, bias, a.softplus);
            dt = n_chunks > 1 ? sel_dt<Q>(a, seq, token(1), head) : 0.0f;
        }
    }
    for (int k = 0; k < n_chunks; ++k) {
        const int t0 = token(k), n = min(Q, seq.n - t0);
        __syncthreads();
        stage_x.template store<SX>(s.x);
        stage_B.template store<SB>(s.B);
        if constexpr (kOut) stage_C.template store<SC>(s.C);
        __syncthreads();
        if (k + 1 < n_chunks) fetch(k + 1);
        const SelSteps<Q>& steps = s.steps[k & 1];

        SelFrag<Tc> xf[QK];  // row p of x transposed, over the tokens
        float odd = 0.0f;
#pragma unroll
        for (int ks = 0; ks < QK; ++ks) {
            xf[ks] = sel_cols(s.x + 32 * ks * SX + 16 * wave, SX, l, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) odd = fmaf(xf[ks].get(e), 0.0f, odd);
        }
        const bool unfinite = kOut && __any(odd != 0.0f);
        if (unfinite)
#pragma unroll
            for (int ks = 0; ks < QK; ++ks)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(fabsf(xf[ks].get(e)) < INFINITY)) xf[ks].set(e, 0.0f);

        if constexpr (kOut) {
#pragma unroll
            for (int m = 0; m < kMyTiles; ++m) {
                const int t = wave + 4 * m;
                if (t >= kTiles) break;
                const int it = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0, jt = t - it * (it + 1) / 2;
                const int i = 16 * it + l, j0 = 16 * jt + 4 * g;
                sel_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < NK; ++ks)
                    sel_mma(acc, sel_rows(s.B + (16 * jt + l) * SB + 32 * ks, g), sel_rows(s.C + i * SC + 32 * ks, g));
                sel_settle(acc);
                const int whole = steps.whole[i];
                const float rest = steps.rest[i];
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float decay = sel_exp2(whole - steps.whole[j0 + r], rest - steps.rest[j0 + r]);
                    v[r] = j0 + r <= i ? acc[r] * (decay * steps.step[j0 + r]) : 0.0f;
                }
                sel_store<Tc, 4>(s.weights + i * SW + j0, v);
            }
        }
        if (wave == kStepWave && k + 1 < n_chunks) {
            sel_steps<Q>(s.steps[(k + 1) & 1], dt, seq.n - token(k + 1), A, bias, a.softplus);
            dt = k + 2 < n_chunks ? sel_dt<Q>(a, seq, token(k + 2), head) : 0.0f;
        }
        if constexpr (kOut) {
            __syncthreads();
            SelFrag<Tc> sf[NK];  // the state that enters, over the states
#pragma unroll
            for (int ks = 0; ks < NK; ++ks)
#pragma unroll
                for (int e = 0; e < 8; ++e) sf[ks].set(e, state[2 * ks + (e >> 2)][e & 3]);
#pragma unroll
            for (int it = 0; it < QT; ++it) {
                const int i = 16 * it + l, c = 16 * wave + 4 * g;
                sel_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) sel_mma(acc, sf[ks], sel_rows(s.C + i * SC + 32 * ks, g));
                acc *= steps.from_start[i];
#pragma unroll
                for (int ks = 0; ks <= it / 2; ++ks) sel_mma(acc, xf[ks], sel_rows(s.weights + i * SW + 32 * ks, g));
                sel_settle(acc);
                if (unfinite) sel_add_unfinite<Tc, Q, SX, SW>(acc, s.x, s.weights, c, i);
                if (i < n && 16 * wave < cols) {
                    float own[4];
                    sel_load<Tc, 4>(s.x + i * SX + c, own);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[r] = fmaf(D, own[r], acc[r]);
                    T* row = static_cast<T*>(a.y) + ((seq.row0 + t0 + i) * a.n_heads + head) * a.dim + p_tile;
                    sel_store4(row, c, cols, plan.vec & kSelVecY, acc);
                }
            }
        }
        if (WALK == kSelStates) {
            const long long chunk = first_chunk + t0 / Q;
            if (p < a.dim && chunk < plan.n_chunks) {
                float* out = plan.states + (back * plan.n_chunks + chunk) * all_states + my_state;
#pragma unroll
                for (int t = 0; t < NT; ++t) sel_state_store(out, 16 * t + 4 * g, a.states, vec_state, state[t]);
            }
        }

        const float all = steps.from_start[Q - 1];
        keeps *= all;
#pragma unroll
        for (int t = 0; t < NT; ++t) state[t] *= all;
#pragma unroll
        for (int ks = 0; ks < QK; ++ks) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = 32 * ks + 16 * (e >> 2) + 4 * g + (e & 3);
                v[e] = xf[ks].get(e) * (back ? steps.from_start[j] : steps.to_end[j] * steps.step[j]);
            }
            SelFrag<Tc> split[kSplits];
            sel_split<Tc>(v, split);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const SelFrag<Tc> bf = sel_cols(s.B + 32 * ks * SB + 16 * t, SB, l, g);
#pragma unroll
                for (int q = 0; q < kSplits; ++q) sel_mma(state[t], bf, split[q]);
            }
        }
        sel_settle(state);
        if (unfinite)
            for (int j = 0; j < n; ++j) {
                const float v = (float)s.x[j * SX + 16 * wave + l];
                if (!(fabsf(v) < INFINITY))
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            state[t][r] = fmaf(v * (steps.to_end[j] * steps.step[j]),
                                               (float)s.B[j * SB + 16 * t + 4 * g + r], state[t][r]);
            }
    }
    float* end = nullptr;
    if (WALK == kSelEnds) {
        end = ends + segment * all_states + my_state;
        if (tile == 0 && threadIdx.x == 0)
            plan.keeps[(back * plan.n_segments + segment) * a.n_heads + head] = keeps;
    } else if (seq.chunk == (back ? 0 : n_segments - 1)) {
        end = kOut ? a.final : back ? a.dinitial : nullptr;
        if (end) end += seq.seq * all_states + my_state;
    }
    if (end && p < a.dim)
#pragma unroll
        for (int t = 0; t < NT; ++t) sel_state_store(end, 16 * t + 4 * g, a.states, vec_state, state[t]);
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
    // (work-groups: at most one per chunk, head and tile of the dimension in each direction)
    const long long most = 0x7fffffffLL, chunks = sel_max_chunks(a->tokens, 32), tiles = (a->dim + 63) / 64;
    if (chunks > most || chunks * a->n_heads > most || 2 * chunks * a->n_heads * tiles > most) return NHIP_E_BADARG;
    return 0;
}

static inline long long sel_round4(long long floats) { return (floats + 3) & ~3LL; }

// How the sequences are cut, for a workspace that begins with the ends and the keeps.  A compute unit works best on
// two walks at once; where the sequences, heads and tiles do not give that many, sequences are cut into segments
// of at least four chunks.
static inline SelWalkPlan sel_walk_plan(const nhip_scan_args& a, int directions, float* states) {
    SelWalkPlan p;
    const int q = sel_chunk_tokens(a.states);
    p.n_tiles = (a.dim + 63) / 64;
    p.directions = directions;
    p.states = states;
    p.n_chunks = sel_max_chunks(a.tokens, q);
    const long long walks = (long long)directions * a.n_heads * p.n_tiles;
    const long long longest = a.tokens.starts ? (a.tokens.n_tokens + q - 1) / q : sel_chunks(a.tokens.length, q);
    const long long total = a.tokens.starts ? longest : longest * a.tokens.n_seqs;
    long long wanted = (512 + walks - 1) / walks;  // segments
    if (!a.tokens.starts && a.tokens.n_seqs) wanted = (wanted + a.tokens.n_seqs - 1) / a.tokens.n_seqs * a.tokens.n_seqs;
    long long chunks = (total + wanted - 1) / wanted;
    if (chunks < 4) chunks = 4;
    const bool cut = chunks < longest;
    p.chunks = (int)(cut ? chunks : longest > 0 ? longest : 1);
    p.n_segments = sel_max_chunks(a.tokens, q * p.chunks);
    p.ends = cut ? reinterpret_cast<float*>(16) : nullptr;  // (its place is the caller's to fill in)
    p.keeps = nullptr;
    p.vec = 0;
    if (sel_rows_aligned(a.x, a.type)) p.vec |= kSelVecX;
    if (sel_rows_aligned(a.B, a.type)) p.vec |= kSelVecB;
    if (sel_rows_aligned(a.C, a.type)) p.vec |= kSelVecC;
    if (sel_rows_aligned(a.dy, a.type)) p.vec |= kSelVecDy;
    if (a.dim % 4 == 0 && sel_aligned(a.y, 16) && sel_aligned(a.dx, 16)) p.vec |= kSelVecY;
    if (a.states % 4 == 0 && sel_aligned(a.initial, 16) && sel_aligned(a.final, 16) && sel_aligned(a.dfinal, 16) &&
        sel_aligned(a.dinitial, 16) && sel_aligned(a.dB, 16) && sel_aligned(a.dC, 16))
        p.vec |= kSelVecState;
    return p;
}

// Floats of workspace that the cut needs (a multiple of 4), and its place
static inline long long sel_walk_space(const nhip_scan_args& a, const SelWalkPlan& p) {
    if (!p.ends) return 0;
    const long long per = (long long)p.directions * p.n_segments * a.n_heads;
    return sel_round4(per * a.dim * a.states) + sel_round4(per);
}
static inline void sel_walk_place(const nhip_scan_args& a, SelWalkPlan& p, float* space) {
    if (!p.ends) return;
    p.ends = space;
    p.keeps = space + sel_round4((long long)p.directions * p.n_segments * a.n_heads * a.dim * a.states);
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

template <int WALK> static inline int sel_walk_launch(hipStream_t stream, const nhip_scan_args& a, const SelWalkPlan& plan,
                                                      bool first, bool last) {
    const unsigned grid = (unsigned)(plan.directions * plan.n_segments * a.n_heads * plan.n_tiles);
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
            if (first && last) NHIP_LAUNCH(kernel, dim3(grid), dim3(NHIP_WG), lds, stream, a, plan);
            else if (first) NHIP_LAUNCH_FIRST(kernel, dim3(grid), dim3(NHIP_WG), lds, stream, a, plan);
            else if (last) NHIP_LAUNCH_LAST(kernel, dim3(grid), dim3(NHIP_WG), lds, stream, a, plan);
            else hipLaunchKernelGGL(kernel, dim3(grid), dim3(NHIP_WG), lds, stream, a, plan);
            rc = (int)hipGetLastError();
        });
    });
    return rc;
}

// WALK over all sequences, after a launch for the segments' ends where they are cut; `last`: nothing
// follows in this entry point.
template <int WALK> static inline int sel_walk(hipStream_t stream, const nhip_scan_args& a, const SelWalkPlan& plan, bool last) {
    if (plan.n_segments == 0) return 0;
    if (plan.ends)
        if (int e = sel_walk_launch<kSelEnds>(stream, a, plan, true, false)) return e;
    return sel_walk_launch<WALK>(stream, a, plan, !plan.ends, last);
}
