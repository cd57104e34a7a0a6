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

// Sequences are cut into segments of `chunks` chunks.  A work-group walks over one for two units of its heads'
// group, a unit being 64 of a head's dimension.  A first launch (kSelEnds) leaves what every segment adds on its
// own, a second turns that into the states that the segments begin with, for the walk itself.
struct SelWalkPlan {
    int n_tiles;            // units of a head
    int pairs;              // of units in a group
    bool vec;               // everything can be read and written 16 bytes at a time
    int chunks;             // per segment
    int directions;         // 2: both halves
    long long n_segments, n_chunks;
    float* states;          // [direction][chunk][head][dim][states]
    bool few;               // segments in a sequence: a walk adds up those before it itself
    float* ends;            // [direction][segment][head][dim][states], NULL: no sequence has two segments
    float* keeps;           // [direction][segment][head]: what a segment keeps of the state it begins with
};

// Tokens of a chunk: 64, or 32 where 256 states would not fit the LDS otherwise.
constexpr int sel_chunk_of(int np) { return np > 128 ? 32 : 64; }

// States are worked on as 32, 64, 128 or 256; f(std::integral_constant) for the smallest of these that holds n.
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

// Four neighbouring elements of a row of `cols`; VEC: rows hold whole fours, at multiples of 16 bytes (states) or
// of their size (outputs)
template <bool VEC>
__device__ __forceinline__ sel_f4 sel_state_load(const float* p, int n, int states) {  // (no load under a condition)
    sel_f4 v;
    if constexpr (VEC) {
        v = *reinterpret_cast<const sel_f4*>(p + min(n, states - 4));
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = p[min(n + r, states - 1)];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = n + r < states ? v[r] : 0.0f;
    return v;
}
template <bool VEC>
__device__ __forceinline__ void sel_state_store(float* p, int n, int states, const sel_f4& v) {
    if constexpr (VEC) {
        if (n < states) *reinterpret_cast<sel_f4*>(p + n) = v;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < states) p[n + r] = v[r];
    }
}
template <bool VEC, class T>
__device__ __forceinline__ void sel_store4(T* p, int c, int cols, const sel_f4& v) {
    if constexpr (VEC) {
        if (c < cols) sel_store<T, 4>(p + c, {v[0], v[1], v[2], v[3]});
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (c + r < cols) p[c + r] = (T)v[r];
    }
}

// The scheduler moves nothing across: left to itself it reads all operands of a chunk from the LDS at
// once, and spills.
__device__ __forceinline__ void sel_phase() { __builtin_amdgcn_sched_barrier(0); }

template <class Tc, int NP, bool OUTPUTS> struct SelWalkLds {
    static constexpr int Q = sel_chunk_of(NP);
    static constexpr int SX = sel_stride_cols<Tc>(64), SB = sel_stride_cols<Tc>(NP), SC = sel_stride<Tc>(NP),
                         SW = sel_stride<Tc>(Q);
    alignas(16) Tc x[2][Q * SX];
    alignas(16) Tc B[Q * SB];
    // weights [i][j]: (C_i . B_j) e^{c_i - c_j} step_j of each unit; their second parts (bfloat16) take the place of C
    static constexpr int kParts = SelSplit<Tc>::out, kRest = (kParts - 1) * 2 * Q * SW;
    alignas(16) Tc C[OUTPUTS ? (Q * SC > kRest ? Q * SC : kRest) : 8];
    alignas(16) Tc weights[OUTPUTS ? 2 : 1][OUTPUTS ? Q * SW : 8];
    __device__ __forceinline__ Tc* rest(int unit) { return C + unit * Q * SW; }
    SelSteps<Q> steps[2][2];                                        // [unit][chunk % 2]
};

// One work-group walks over the chunks of a segment for two units, two waves to each, a wave to 32 of the
// dimension, whose part of the state stays in registers: lane l holds rows p = 16 h + l % 16 of it, the
// states 16 t + 4 (l / 16) + r in register r of tile t -- the order of a fragment over the states, so that
// the state is an operand of the next chunk's products as it is.  Two units share B, C and their
// products, and 32 rows share what a wave reads of them: with one unit and 16 rows the LDS, which all
// operands but the state come from, was busy for as long as a chunk took.  The inputs of the next chunk
// are fetched while one is worked on, the steps of two chunks formed at once, by a wave each.  A
// work-group of the bfloat16 kernel with 128 states takes half of a compute unit's LDS and registers.
// 8 x 2048 tokens, 32 heads of 64, 128 states, bfloat16: 103 us for 175 MB and 40 GFLOP, 39 for the ends (53 MB in, 25
// out), 93 and 36 behind a hundred calls.  Bound by issue: the matrix cores work for 24 % of the time, the LDS for 36 %,
// and a chunk takes a wave about 1,300 vector instructions beside 196 matrix ones (half of these for the three parts of
// what the state gains).  Chunks of 32 tokens, at which four work-groups fit a unit, took 96 us when these took 95.  The
// state that enters and the weights go in as two parts: as one, the walk took 88 us and y was off by 2^-8 of the terms'
// magnitudes, not of itself.
template <class T, class Tc, int NP, int WALK, bool VEC>
__global__ __launch_bounds__(NHIP_WG, sizeof(Tc) == 2 && NP <= 128 ? 2 : 1)
void sel_walk_kernel(nhip_scan_args a, SelWalkPlan plan) {
    constexpr bool kOut = WALK == kSelOutputs;
    using Lds = SelWalkLds<Tc, NP, kOut>;
    constexpr int Q = Lds::Q, QT = Q / 16, QK = Q / 32, NT = NP / 16, NK = NP / 32;
    constexpr int SX = Lds::SX, SB = Lds::SB, SC = Lds::SC, SW = Lds::SW;
    constexpr int kSplits = SelSplit<Tc>::n, kParts = Lds::kParts;
    extern __shared__ __align__(16) char lds_bytes[];
    Lds& s = *reinterpret_cast<Lds*>(lds_bytes);

    // neighbouring heads read the same B and C: they go to one die, whose L2 holds them
    const int groups = gridDim.x / plan.directions;
    const int back = kOut ? 0 : blockIdx.x >= groups;
    const int id = nhip_xcd_remap(blockIdx.x - back * groups, groups);
    const int pair = id % plan.pairs, group = (id / plan.pairs) % a.n_groups;
    const int segment = id / (plan.pairs * a.n_groups);
    const SelSeq seq = sel_seq_of_chunk(a.tokens, segment, Q * plan.chunks);
    if (seq.seq < 0) return;
    const int n_segments = sel_chunks(seq.n, Q * plan.chunks);
    // (nobody begins with what the last one, or going back the first, adds)
    if (WALK == kSelEnds && seq.chunk == (back ? 0 : n_segments - 1)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NHIP_WAVE);
    const int lane_l = threadIdx.x & 15, lane_g = (threadIdx.x & 63) >> 4;
    // the units; a second one that is not there is the first again, and writes nothing
    const int per_group = a.n_heads / a.n_groups, units = per_group * plan.n_tiles;
    auto head_of = [&](int unit) { return group * per_group + min(2 * pair + unit, units - 1) / plan.n_tiles; };
    auto tile_of = [&](int unit) { return 64 * (min(2 * pair + unit, units - 1) % plan.n_tiles); };
    const int mine = wave >> 1, head = head_of(mine), p_tile = tile_of(mine);
    const int p_wave = 32 * (wave & 1);  // within the unit
    const bool writes = 2 * pair + mine < units;
    const int cols = min(64, a.dim - p_tile);
    const long long head_state = (long long)a.dim * a.states, all_states = a.n_heads * head_state;
    const long long my_state = head * head_state + (long long)(p_tile + p_wave + lane_l) * a.states;
    const long long next_rows = 16LL * a.states;
    const bool there[2] = {p_wave + lane_l < cols, p_wave + 16 + lane_l < cols};
    float* const ends = plan.ends ? plan.ends + back * plan.n_segments * all_states : nullptr;

    sel_f4 state[2][NT];
    {
        const bool begun = plan.ends && !plan.few;
        const float* from = WALK == kSelEnds ? nullptr
                            : begun          ? ends + segment * all_states
                            : back           ? (a.dfinal ? a.dfinal + seq.seq * all_states : nullptr)
                                             : (a.initial ? a.initial + seq.seq * all_states : nullptr);
        // (rows that are not there: the last one again, for which nothing is written)
        const int p = min(p_tile + p_wave + lane_l, a.dim - 1), q = min(p_tile + p_wave + 16 + lane_l, a.dim - 1);
        const long long at[2] = {head * head_state + (long long)p * a.states, head * head_state + (long long)q * a.states};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int t = 0; t < NT; ++t)
                if (from) state[h][t] = sel_state_load<VEC>(from + at[h], 16 * t + 4 * lane_g, a.states);
                else state[h][t] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (WALK != kSelEnds && plan.ends && !begun) {
            const int first = segment - seq.chunk, before = back ? n_segments - 1 - seq.chunk : seq.chunk;
            for (int k = 0; k < before; ++k) {
                const long long other = min((long long)first + (back ? n_segments - 1 - k : k), plan.n_segments - 1);
                const float keeps = plan.keeps[(back * plan.n_segments + other) * a.n_heads + head];
                const float* const end = ends + other * all_states;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        state[h][t] = state[h][t] * keeps + sel_state_load<VEC>(end + at[h], 16 * t + 4 * lane_g, a.states);
            }
        }
    }
    const nhip_rows& x = back ? a.dy : a.x;
    const nhip_rows& B = back ? a.C : a.B;
    const float D = kOut && a.D ? a.D[head] : 0.0f, A = a.A[head], bias = a.dt_bias ? a.dt_bias[head] : 0.0f;
    // chunks of the sequence that this segment holds, and the token at which walk number k of them begins
    const int chunk0 = seq.chunk * plan.chunks;
    const int n_chunks = min(plan.chunks, (seq.n + Q - 1) / Q - chunk0);
    auto token = [&](int k) { return (chunk0 + (back ? n_chunks - 1 - k : k)) * Q; };
    const long long first_chunk = WALK == kSelStates ? sel_seq(a.tokens, seq.seq, Q).chunk : 0;

    SelStage<T, Tc, Q, 64, VEC> stage_x[2];
    SelStage<T, Tc, Q, NP, VEC> stage_B, stage_C;
    // where the next chunk's rows begin
    const int way = back ? -Q : Q, t_first = token(0);
    const T* x_at = sel_row<T>(x, a.tokens, seq, t_first);
    const T* B_at = sel_row<T>(B, a.tokens, seq, t_first) + group * B.head;
    const T* C_at = kOut ? sel_row<T>(a.C, a.tokens, seq, t_first) + group * a.C.head : nullptr;
    const long long x_way = way * x.token, B_way = way * B.token, C_way = kOut ? way * a.C.token : 0;
    const long long unit_at[2] = {head_of(0) * x.head + tile_of(0), head_of(1) * x.head + tile_of(1)};
    const int unit_cols[2] = {min(64, a.dim - tile_of(0)), min(64, a.dim - tile_of(1))};
    auto fetch = [&](int n) {
#pragma unroll
        for (int u = 0; u < 2; ++u) stage_x[u].load(x_at + unit_at[u], x.token, n, unit_cols[u]);
        stage_B.load(B_at, B.token, n, a.states);
        if constexpr (kOut) stage_C.load(C_at, a.C.token, n, a.states);
    };
    float keeps = 1.0f;
    SelDt dt = {0, 0};
    const SelDtRow dt_row = sel_dt_row(a, seq, head);
    const int ahead = wave & 1;  // which of two chunks this wave forms the steps of
    if (n_chunks > 0) {
        fetch(min(Q, seq.n - t_first));
        dt = sel_dt(dt_row, token(min(ahead, n_chunks - 1)), seq.n);
    }
    for (int k = 0; k < n_chunks; ++k) {
        const int t0 = token(k), n = min(Q, seq.n - t0);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; ++u) stage_x[u].template store<SX>(s.x[u], n, unit_cols[u]);
        stage_B.template store<SB>(s.B, n, a.states);
        if constexpr (kOut) stage_C.template store<SC>(s.C, n, a.states);
        if ((k & 1) == 0) {
            if (k + ahead < n_chunks)
                sel_steps<Q>(s.steps[mine][ahead], dt.value(a.dt_type), seq.n - token(k + ahead), A, bias, a.softplus);
            dt = sel_dt(dt_row, token(min(k + 2 + ahead, n_chunks - 1)), seq.n);
        }
        __syncthreads();
        // (unconditional, as the loads are: the last chunk is fetched twice)
        const bool more = k + 1 < n_chunks;
        x_at += more ? x_way : 0;
        B_at += more ? B_way : 0;
        if constexpr (kOut) C_at += more ? C_way : 0;
        fetch(min(Q, seq.n - (more ? t0 + way : t0)));
        const SelSteps<Q>& steps = s.steps[mine][k & 1];
        const Tc* const xs = s.x[mine];
        // (addresses are formed anew in each chunk: kept, they take the registers of the state)
        int l = lane_l, g = lane_g;
        asm volatile("" : "+v"(l), "+v"(g));
        // (24 bits: products of 32 take four times as long)
        const int l_X = __mul24(l, SX), l_B = __mul24(l, SB), l_C = __mul24(l, SC), l_W = __mul24(l, SW);

        SelFrag<Tc> xf[2][QK];  // rows p of x transposed, over the tokens
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int ks = 0; ks < QK; ++ks) xf[h][ks] = sel_cols(xs + 32 * ks * SX + p_wave + 16 * h, SX, l, g);
        // elements of x that are no finite numbers would reach, as zero times infinity, the tokens in front of them
        // too: they are left out of the products, and what reads them is made no number
        bool finite = true;
        auto odd = [&](int h, int ks) {  // (from LDS again: kept, they take registers though there are none)
            SelFrag<Tc> f = sel_cols(xs + 32 * ks * SX + p_wave + 16 * h, SX, l, g);
            return sel_take_unfinite(f);
        };
        if constexpr (kOut) finite = __all(sel_finite(xf));
        if (!finite)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int ks = 0; ks < QK; ++ks) (void)sel_take_unfinite(xf[h][ks]);

        if constexpr (kOut) {
            // Weights: tiles of the lower triangle of C . B, for both units, and those above it that a read of 32 tokens
            // takes along.  A wave's tiles are in rows (3: 0, 1, 2), (2: 0, 1, 2), (1: 0, 1; 3: 3), (0: 0, 1; 2: 3): the
            // first two share the rows of C.
            constexpr int kMine = QT == 4 ? 3 : 1;
            const int row_a = QT == 4 ? 3 - wave : (wave == 1 || wave == 2);
            const int row_b = QT == 4 && wave >= 2 ? 5 - wave : row_a;
            auto col_of = [&](int m) { return QT == 4 ? (wave >= 2 && m == 2 ? 3 : m) : (wave > 1); };
            sel_f4 acc[kMine];
#pragma unroll
            for (int m = 0; m < kMine; ++m) acc[m] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) {
                const SelFrag<Tc> c = sel_rows(s.C + 16 * row_a * SC + l_C + 32 * ks, g);
#pragma unroll
                for (int m = 0; m < kMine; ++m)
                    sel_mma(acc[m], sel_rows(s.B + 16 * col_of(m) * SB + l_B + 32 * ks, g),
                            m < 2 ? c : sel_rows(s.C + 16 * row_b * SC + l_C + 32 * ks, g));
            }

            sel_f4 out[2][QT];
            auto read_state = [&] {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int it = 0; it < QT; ++it) out[h][it] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) {
                    if (ks % 2 == 0) sel_phase();
                    SelFrag<Tc> sf[2][kParts];  // the state that enters, over the states
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = state[h][2 * ks + (e >> 2)][e & 3];
                        sel_split(v, sf[h]);
                    }
#pragma unroll
                    for (int it = 0; it < QT; ++it) {
                        const SelFrag<Tc> c = sel_rows(s.C + 16 * it * SC + l_C + 32 * ks, g);
#pragma unroll
                        for (int q = 0; q < kParts; ++q)
#pragma unroll
                            for (int h = 0; h < 2; ++h) sel_mma(out[h][it], sf[h][q], c);
                    }
                }
                sel_phase();
#pragma unroll
                for (int it = 0; it < QT; ++it) {
                    const float e = steps.from_start[16 * it + l];
                    out[0][it] *= e;
                    out[1][it] *= e;
                }
            };
            if constexpr (kParts > 1) {  // (nobody reads C any more when the second parts are stored)
                read_state();
                __syncthreads();
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                sel_phase();
                const SelSteps<Q>& st = s.steps[u][k & 1];
#pragma unroll
                for (int m = 0; m < kMine; ++m) {
                    const int row = 16 * (m < 2 ? row_a : row_b), i = row + l, j0 = 16 * col_of(m) + 4 * g;
                    const int whole = st.whole[i], at = row * SW + l_W + j0;
                    const float to = st.to[i];
                    float v[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float w = __builtin_ldexpf(acc[m][r] * (to * st.from_step[j0 + r]), whole - st.whole[j0 + r]);
                        v[r] = j0 + r <= i ? w : 0.0f;
                    }
                    sel_store_parts(s.weights[u] + at, s.rest(u) + at, v);
                }
            }
            __syncthreads();
            if constexpr (kParts == 1) read_state();
#pragma unroll
            for (int ks = 0; ks < QK; ++ks)
#pragma unroll
                for (int it = 2 * ks; it < QT; ++it)
#pragma unroll
                    for (int q = 0; q < kParts; ++q) {
                        const SelFrag<Tc> w = sel_rows((q ? s.rest(mine) : s.weights[mine]) + 16 * it * SW + l_W + 32 * ks, g);
                        sel_mma(out[0][it], xf[0][ks], w);
                        sel_mma(out[1][it], xf[1][ks], w);
                    }
            sel_settle(out[0]);
            sel_settle(out[1]);
            if (!finite)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    sel_f4 count[QT];  // how many of them each token reads
#pragma unroll
                    for (int it = 0; it < QT; ++it) count[it] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int ks = 0; ks < QK; ++ks) {
                        const SelFrag<Tc> ones = odd(h, ks);
#pragma unroll
                        for (int it = 2 * ks; it < QT; ++it) {
                            SelFrag<Tc> up_to;
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                up_to.set(e, 32 * ks + 16 * (e >> 2) + 4 * g + (e & 3) <= 16 * it + l ? 1.0f : 0.0f);
                            sel_mma(count[it], ones, up_to);
                        }
                    }
                    sel_settle(count);
#pragma unroll
                    for (int it = 0; it < QT; ++it)
#pragma unroll
                        for (int r = 0; r < 4; ++r) out[h][it][r] = count[it][r] > 0.0f ? NAN : out[h][it][r];
                }
            sel_phase();
            T* const y = static_cast<T*>(a.y) + ((seq.row0 + t0) * a.n_heads + head) * a.dim + p_tile;
            const unsigned row = (unsigned)(a.n_heads * a.dim);
#pragma unroll
            for (int it = 0; it < QT; ++it)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float own[4];
                    sel_load<Tc, 4>(xs + 16 * it * SX + l_X + p_wave + 16 * h + 4 * g, own);
#pragma unroll
                    for (int r = 0; r < 4; ++r) out[h][it][r] = fmaf(D, own[r], out[h][it][r]);
                }
            const unsigned at = l * row + 4 * g;
            if (VEC && writes && n == Q && cols == 64) {
                char* const to = reinterpret_cast<char*>(y + p_wave);  // (one place for the wave, and 32 bits from it)
#pragma unroll
                for (int it = 0; it < QT; ++it)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        sel_store<T, 4>(reinterpret_cast<T*>(to + (at + 16 * it * row) * (unsigned)sizeof(T)) + 16 * h,
                                        {out[h][it][0], out[h][it][1], out[h][it][2], out[h][it][3]});
            } else if (writes) {
#pragma unroll
                for (int it = 0; it < QT; ++it)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (16 * it + l < n)
                            sel_store4<VEC>(y + (unsigned)(16 * it + l) * row, p_wave + 16 * h + 4 * g, cols, out[h][it]);
            }
        }
        if (WALK == kSelStates) {
            const long long chunk = first_chunk + t0 / Q;
            if (writes && chunk < plan.n_chunks) {
                float* out = plan.states + (back * plan.n_chunks + chunk) * all_states + my_state;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (there[h])
#pragma unroll
                        for (int t = 0; t < NT; ++t)
                            sel_state_store<VEC>(out + h * next_rows, 16 * t + 4 * g, a.states, state[h][t]);
            }
        }

        const float* const weight = back ? steps.from_start : steps.to_end_step;
        const float all = steps.from_start[Q - 1];
        keeps *= all;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float keep = all;
            if (!finite) {  // (lane l of each quarter of the wave holds other tokens of row p)
                float bad = 0.0f;
#pragma unroll
                for (int ks = 0; ks < QK; ++ks) {
                    const SelFrag<Tc> ones = odd(h, ks);
#pragma unroll
                    for (int e = 0; e < 8; ++e) bad += ones.get(e);
                }
                bad += __shfl_xor(bad, 16);
                bad += __shfl_xor(bad, 32);
                keep = bad > 0.0f ? NAN : all;
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) state[h][t] *= keep;
        }
#pragma unroll
        for (int ks = 0; ks < QK; ++ks) {
            sel_phase();
            SelFrag<Tc> split[2][kSplits];
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = weight[32 * ks + 16 * (e >> 2) + 4 * g + (e & 3)];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = xf[h][ks].get(e) * w[e];
                sel_split(v, split[h]);
            }
            constexpr int kSide = 2;  // tiles side by side
#pragma unroll
            for (int t0 = 0; t0 < NT; t0 += kSide) {
                SelFrag<Tc> bf[kSide];
#pragma unroll
                for (int t = 0; t < kSide; ++t) bf[t] = sel_cols(s.B + 32 * ks * SB + 16 * (t0 + t), SB, l, g);
#pragma unroll
                for (int q = 0; q < kSplits; ++q)
#pragma unroll
                    for (int t = 0; t < kSide; ++t)
#pragma unroll
                        for (int h = 0; h < 2; ++h) sel_mma(state[h][t0 + t], bf[t], split[h][q]);
            }
        }
    }
    sel_settle(state[0]);
    sel_settle(state[1]);
    float* end = nullptr;
    if (WALK == kSelEnds) {
        end = ends + segment * all_states + my_state;
        if (writes && p_tile == 0 && (threadIdx.x & 127) == 0)
            plan.keeps[(back * plan.n_segments + segment) * a.n_heads + head] = keeps;
    } else if (seq.chunk == (back ? 0 : n_segments - 1)) {
        end = kOut ? a.final : back ? a.dinitial : nullptr;
        if (end) end += seq.seq * all_states + my_state;
    }
    if (end && writes)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (there[h])
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    sel_state_store<VEC>(end + h * next_rows, 16 * t + 4 * lane_g, a.states, state[h][t]);
}

// From what each segment of a sequence adds to the state to the state that it begins with, in place: a lane takes
// V elements of a head's state through the segments.
template <int V>
static __global__ __launch_bounds__(NHIP_WG) void sel_begin_kernel(nhip_scan_args a, SelWalkPlan plan, int q) {
    const int head_state = a.dim * a.states, blocks = (head_state + NHIP_WG * V - 1) / (NHIP_WG * V);
    const int block = blockIdx.x % blocks, head = (blockIdx.x / blocks) % a.n_heads;
    const int which = blockIdx.x / (blocks * a.n_heads), s = which % a.tokens.n_seqs, back = which / a.tokens.n_seqs;
    const SelSeq seq = sel_seq(a.tokens, s, q * plan.chunks);
    const int at = (block * NHIP_WG + threadIdx.x) * V;
    const int n = (int)min((long long)sel_chunks(seq.n, q * plan.chunks), plan.n_segments - seq.chunk);
    if (at >= head_state || n <= 0) return;
    const long long all_states = (long long)a.n_heads * head_state, mine = (long long)head * head_state + at;
    float state[V];
    const float* from = back ? a.dfinal : a.initial;
#pragma unroll
    for (int i = 0; i < V; ++i) state[i] = from ? from[s * all_states + mine + i] : 0.0f;
    float* const ends = plan.ends + (back * plan.n_segments + seq.chunk) * all_states + mine;
    const float* const keeps = plan.keeps + (back * plan.n_segments + seq.chunk) * a.n_heads + head;
    constexpr int kAhead = 8;
    for (int k0 = 0; k0 < n; k0 += kAhead) {
        float adds[kAhead][V], keep[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {  // (the last one's was not formed: nobody begins with it)
            const int w = min(k0 + k, n - 1), segment = back ? n - 1 - w : w;
            sel_load<float, V>(ends + segment * all_states, adds[k]);
            keep[k] = keeps[(long long)segment * a.n_heads];
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (k0 + k >= n) break;
            const int segment = back ? n - 1 - k0 - k : k0 + k;
            sel_store<float, V>(ends + segment * all_states, state);
#pragma unroll
            for (int i = 0; i < V; ++i) state[i] = fmaf(state[i], keep[k], adds[k][i]);
        }
    }
}

// ------------------------------------------------------------------------------- host side
// Whether rows can be read 16 bytes at a time, with offsets of 32 bits within a chunk
static inline bool sel_rows_wide(const nhip_rows& r, int type, int cols) {
    const int v = 16 / sel_size(type);
    return sel_aligned(r.p, 16) && cols % v == 0 && r.seq % v == 0 && r.token % v == 0 && r.head % v == 0 &&
           r.token >= 0 && r.token < (1 << 23);
}

static inline int sel_scan_check(const nhip_scan_args* a) {
    if (!a || !a->A || a->n_heads <= 0 || a->dim <= 0 || a->n_groups <= 0 || a->n_heads % a->n_groups) return NHIP_E_BADARG;
    if (a->states < 1 || a->states > 256 || !sel_tokens_ok(a->tokens)) return NHIP_E_BADARG;
    if (a->type < NHIP_F32 || a->type > NHIP_F16 || a->dt_type < NHIP_F32 || a->dt_type > NHIP_F16) return NHIP_E_BADARG;
    if (a->tokens.n_tokens && (!a->x.p || !a->dt.p || !a->B.p || !a->C.p)) return NHIP_E_BADARG;
    // (work-groups: at most one per chunk, head and tile of the dimension in each direction)
    const long long most = 0x7fffffffLL, chunks = sel_max_chunks(a->tokens, 32), tiles = (a->dim + 63) / 64;
    if (chunks > most || chunks * a->n_heads > most || 2 * chunks * a->n_heads * tiles > most) return NHIP_E_BADARG;
    // (offsets of 32 bits within a chunk)
    if ((long long)a->n_heads * a->dim >= (1 << 23) || (long long)a->dim * a->states > (1 << 28)) return NHIP_E_BADARG;
    return 0;
}

static inline long long sel_round4(long long floats) { return (floats + 3) & ~3LL; }

// How the sequences are cut, for a workspace that begins with the ends and the keeps.  A compute unit holds two walks
// of the bfloat16 kernel for up to 128 states, one of the others.  Sequences that give every unit a walk stay whole
// (gradient of 8 x 2048 tokens, 32 heads of 64, 128 states, both directions: 482 us, cut in two 489); fewer are cut
// into as many segments as walks fit (8 x 2048 tokens forward: 121 us with 512 walks, 157 with 256), down to a chunk
// each (4001 tokens in nine ragged sequences, 12 heads, 32 bits: 64 us, with four chunks 104).  Up to four segments are
// added up by the walks themselves (the same 8 x 2048 tokens: 114 us, by a launch of its own 133), more by that launch
// (32768 tokens in 32 segments: 222 us, by the walks 301; all of these with the weights of pairs as one part).
static inline SelWalkPlan sel_walk_plan(const nhip_scan_args& a, int directions, float* states) {
    SelWalkPlan p;
    const int q = sel_chunk_tokens(a.states);
    p.n_tiles = (a.dim + 63) / 64;
    p.directions = directions;
    p.states = states;
    p.n_chunks = sel_max_chunks(a.tokens, q);
    p.pairs = (a.n_heads / a.n_groups * p.n_tiles + 1) / 2;
    const long long walks = (long long)directions * a.n_groups * p.pairs;
    const long long longest = a.tokens.starts ? (a.tokens.n_tokens + q - 1) / q : sel_chunks(a.tokens.length, q);
    const long long total = a.tokens.starts ? longest : longest * a.tokens.n_seqs;
    const long long target = a.type == NHIP_BF16 && a.states <= 128 ? 512 : 256;
    long long wanted = (target + walks - 1) / walks;  // segments
    if (!a.tokens.starts && a.tokens.n_seqs) {
        if (a.tokens.n_seqs * walks >= 256) wanted = a.tokens.n_seqs;
        wanted = (wanted + a.tokens.n_seqs - 1) / a.tokens.n_seqs * a.tokens.n_seqs;
    }
    long long chunks = (total + wanted - 1) / wanted;
    const bool cut = chunks < longest;
    p.chunks = (int)(cut ? chunks : longest > 0 ? longest : 1);
    p.n_segments = sel_max_chunks(a.tokens, q * p.chunks);
    p.few = (longest + p.chunks - 1) / p.chunks <= 4;
    p.ends = cut ? reinterpret_cast<float*>(16) : nullptr;  // (its place is the caller's to fill in)
    p.keeps = nullptr;
    p.vec = sel_rows_wide(a.x, a.type, a.dim) && sel_rows_wide(a.B, a.type, a.states) &&
            sel_rows_wide(a.C, a.type, a.states) && (!a.dy.p || sel_rows_wide(a.dy, a.type, a.dim));
    for (const void* q : {(const void*)a.y, (const void*)a.dx, (const void*)a.dB, (const void*)a.dC, (const void*)a.initial,
                          (const void*)a.final, (const void*)a.dfinal, (const void*)a.dinitial})
        p.vec = p.vec && sel_aligned(q, 16);
    return p;
}

// Work-groups, for V elements of a state to a lane, of the launch that turns segments' ends into beginnings
static inline long long sel_begin_groups(const nhip_scan_args& a, const SelWalkPlan& p, int v) {
    const long long per = NHIP_WG * v, blocks = ((long long)a.dim * a.states + per - 1) / per;
    return blocks * a.n_heads * a.tokens.n_seqs * p.directions;
}
static inline long long sel_walk_groups(const nhip_scan_args& a, const SelWalkPlan& p) {
    return (long long)p.directions * p.n_segments * a.n_groups * p.pairs;
}
// Whether the launches of a walk are ones
static inline bool sel_walk_fits(const nhip_scan_args& a, const SelWalkPlan& p) {
    return sel_walk_groups(a, p) <= SEL_MAX_GROUPS &&
           (!p.ends || p.few || sel_begin_groups(a, p, p.vec ? 4 : 1) <= SEL_MAX_GROUPS);
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

// 16-bit floats have their own products on the matrix cores only in their own type; bfloat16's range does
// not hold their precision, so they take the 32-bit ones.
template <class T> struct SelCompute { using type = float; };
template <> struct SelCompute<__bf16> { using type = __bf16; };

template <int WALK> static inline int sel_walk_launch(hipStream_t stream, const nhip_scan_args& a, const SelWalkPlan& plan,
                                                      bool first, bool last) {
    const unsigned grid = (unsigned)sel_walk_groups(a, plan);
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        using Tc = typename SelCompute<T>::type;
        sel_with_states(a.states, [&](auto np) {
            constexpr int NP = decltype(np)::value;
            constexpr size_t lds = sizeof(SelWalkLds<Tc, NP, WALK == kSelOutputs>);
            auto kernel = plan.vec ? sel_walk_kernel<T, Tc, NP, WALK, true> : sel_walk_kernel<T, Tc, NP, WALK, false>;
            rc = sel_allow_lds(stream, kernel, lds);
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
    if (plan.n_segments == 0 || a.tokens.n_seqs == 0) return 0;  // (tokens of no sequence have segments, too)
    if (plan.ends) {
        if (int e = sel_walk_launch<kSelEnds>(stream, a, plan, true, false)) return e;
    }
    if (plan.ends && !plan.few) {
        const int q = sel_chunk_tokens(a.states);
        const dim3 grid((unsigned)sel_begin_groups(a, plan, plan.vec ? 4 : 1));
        if (plan.vec) hipLaunchKernelGGL(sel_begin_kernel<4>, grid, dim3(NHIP_WG), 0, stream, a, plan, q);
        else hipLaunchKernelGGL(sel_begin_kernel<1>, grid, dim3(NHIP_WG), 0, stream, a, plan, q);
        NHIP_LAUNCH_CHECK();
    }
    return sel_walk_launch<WALK>(stream, a, plan, !plan.ends, last);
}
