// The gradient of the selective scan.
//
// Two walks over the chunks leave the state S that enters each chunk and the gradient G of the state
// that leaves it; then every chunk stands for itself.  With L_ij = e^{c_i - c_j} for j <= i (else
// 0), sums over the heads of a group for B and C, and X_ij = dy_i . x_j, K_ij = C_i . B_j:
//     dx_j = step_j (sum_i K_ij L_ij dy_i + e^{c_Q - c_j} G B_j) + D dy_j
//     dB_j = step_j (sum_i X_ij L_ij C_i  + e^{c_Q - c_j} G^T x_j)
//     dC_i = sum_j X_ij L_ij step_j B_j   + e^{c_i} S^T dy_i
// and the gradient of a_t = step_t A, through every decay that spans token t:
//     da_t = sum_{i >= t > j} K_ij X_ij L_ij step_j + sum_{i >= t} q_i + sum_{j < t} r_j step_j + e^{c_Q} <G, S>
//     q_i = e^{c_i} C_i . S^T dy_i,     r_j = e^{c_Q - c_j} B_j . G^T x_j
//     dstep_t = A da_t + sum_{i >= t} K_it X_it L_it + r_t
// No sum of these is the difference of larger ones: the errors of da, which add up in dA over all the
// tokens, stay those of its own terms.
#include <type_traits>

#include "selective_scan.h"

namespace {

struct GradPlan {
    int n_tiles;
    int heads_per_group;   // heads that a work-group goes through
    int blocks;            // work-groups for the heads of one group
    long long n_chunks;
    const float *S, *G;    // [chunk][head][dim][states]
    float* parts;          // [chunk][3][head]: dA, dD, ddt_bias
    float* shared;         // blocks > 1: [block][dB, dC][token][group][states]
};

template <class Tc, int NP> struct GradLds {
    static constexpr int Q = sel_chunk_of(NP);
    static constexpr int SX = sel_stride<Tc>(64), SN = sel_stride<Tc>(NP);
    alignas(16) Tc x[Q * sel_stride<Tc>(64)];
    alignas(16) Tc dy[Q * sel_stride<Tc>(64)];
    alignas(16) Tc B[Q * sel_stride<Tc>(NP)];
    alignas(16) Tc C[Q * sel_stride<Tc>(NP)];
    // The parts of X_ij L_ij step_j, then those of K_ij L_ij step_j: tiles [16 of j][16 of i] of the lower triangle, and one
    // of zeros in the place of all others.  (Whole rows of the tables would leave no room for two parts beside another
    // work-group.)
    static constexpr int kParts = SelSplit<Tc>::out, kTiles = Q / 16 * (Q / 16 + 1) / 2, kZeros = 2 * kParts * kTiles;
    alignas(16) Tc pairs[kZeros + 1][SelTile<Tc>::kSize];
    static constexpr int X(int part, int it, int jt) {
        return it < jt ? kZeros : part * kTiles + it * (it + 1) / 2 + jt;
    }
    static constexpr int K(int part, int it, int jt) { return it < jt ? kZeros : kParts * kTiles + X(part, it, jt); }
    SelSteps<Q> steps;
    // Sums of a head.  over[jt][t]: of K X L step over i >= t in t's own tile of 16 and j < t in tile jt;
    // col[it][j]: of K X L over the i > j of tile it;  q, r, z: by wave
    float over[Q / 16][Q], col[Q / 16][Q], diag[Q], dot[Q], q[4][Q], r[4][Q], z[4];
};

// Eight elements of a state across its rows: k over 32 rows from p0, column n.  Loads are unconditional (one
// under a condition is waited for where its branch ends), from places cut to those that exist: what is too
// much meets zeros of the other operand.  WHOLE: all 32 rows exist; their places are then one offset from
// places that the whole wave shares.
template <bool WHOLE>
__device__ __forceinline__ void state_cols(const float* s, int p0, int n, int dim, int states, int g, float (&v)[8]) {
    const unsigned c = (unsigned)min(n, states - 1);
    const unsigned mine = 4 * (4 * g * (unsigned)states + c);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int k = 16 * (e >> 2) + (e & 3);
        if constexpr (WHOLE) {
            v[e] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(s + (p0 + k) * states) + mine);
        } else {
            v[e] = s[(unsigned)min(p0 + k + 4 * g, dim - 1) * (unsigned)states + c];
        }
    }
}
// Eight elements of row p, as a fragment over the states from n0
template <bool VEC>
__device__ __forceinline__ void state_row(const float* s, int p, int n0, int dim, int states, int g, float (&v)[8]) {
    const float* row = s + (unsigned)min(p, dim - 1) * (unsigned)states;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int n = n0 + 16 * h + 4 * g;
        if constexpr (VEC) {
            const sel_f4 four = *reinterpret_cast<const sel_f4*>(row + min(n, states - 4));
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * h + r] = four[r];
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) v[4 * h + r] = row[min(n + r, states - 1)];
        }
    }
}

// A work-group takes a chunk through a block of its group's heads, 64 of the dimension at a time: the sums for dB
// and dC of 16 states per wave (twice over for 128) stay in registers over all of them, B and C in the LDS.  WHOLE: the
// dimension is a multiple of 64.  4 x 2048 tokens, 32 heads of 64, 128 states, bfloat16: 187 us, 170 behind a
// hundred calls, of which the walks' states, 269 MB once and one half of them again as rows, would take 70 by themselves;
// the matrix cores work for 13 % of the time, the LDS for 26 %, and half of it the two waves of a unit both wait.  The
// walks before it take 41 (ends) and 90 (269 MB written).  With one part of the pairs' weights and of G it took 169,
// and dx, dB and dC were off by 2^-8 of their terms' magnitudes.
template <class T, class Tc, int NP, bool VEC, bool WHOLE>
__global__ __launch_bounds__(NHIP_WG, sizeof(Tc) == 2 && NP <= 128 ? 2 : 1) void grad_kernel(nhip_scan_args a, GradPlan plan) {
    using Lds = GradLds<Tc, NP>;
    constexpr int Q = Lds::Q, QT = Q / 16, QK = Q / 32, NT = NP / 16, NK = NP / 32;
    constexpr int kTiles = Lds::kTiles, kMyTiles = (kTiles + 3) / 4, kMyNT = (NT + 3) / 4;
    constexpr int SX = Lds::SX, SN = Lds::SN;
    using Tile = SelTile<Tc>;
    constexpr int kSplits = SelSplit<Tc>::n, kParts = Lds::kParts;
    extern __shared__ __align__(16) char lds_bytes[];
    Lds& s = *reinterpret_cast<Lds*>(lds_bytes);

    const int id = nhip_xcd_remap(blockIdx.x, gridDim.x);
    const int block = id % plan.blocks, group = (id / plan.blocks) % a.n_groups;
    const int chunk = id / (plan.blocks * a.n_groups);
    const int per_group = a.n_heads / a.n_groups;
    const int head0 = group * per_group + block * plan.heads_per_group;
    const int head1 = min(head0 + plan.heads_per_group, (group + 1) * per_group);
    const SelSeq seq = sel_seq_of_chunk(a.tokens, chunk, Q);
    const int t0 = seq.chunk * Q, n = seq.seq < 0 ? 0 : min(Q, seq.n - t0);
    float* const parts = plan.parts + (long long)chunk * 3 * a.n_heads;
    if (n <= 0) {  // no such chunk, or an empty sequence's
        for (int h = head0 + threadIdx.x; h < head1; h += NHIP_WG)
            parts[h] = parts[a.n_heads + h] = parts[2 * a.n_heads + h] = 0.0f;
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, lane_l = tid & 15, lane_g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid / NHIP_WAVE);
    const long long head_state = (long long)a.dim * a.states;

    {
        SelStage<T, Tc, Q, NP, VEC> stage_B, stage_C;
        stage_B.load(sel_row<T>(a.B, a.tokens, seq, t0) + group * a.B.head, a.B.token, n, a.states);
        stage_C.load(sel_row<T>(a.C, a.tokens, seq, t0) + group * a.C.head, a.C.token, n, a.states);
        stage_B.template store<SN>(s.B, n, a.states);
        stage_C.template store<SN>(s.C, n, a.states);
    }
    for (int q = tid; q < Tile::kSize; q += NHIP_WG) s.pairs[Lds::kZeros][q] = (Tc)0.0f;
    __syncthreads();

    int tile_i[kMyTiles], tile_j[kMyTiles];  // this wave's tiles of the lower triangle
    sel_f4 K[kMyTiles];                      // column j = 16 tile_j + l, rows i = 16 tile_i + 4 g + r
#pragma unroll
    for (int m = 0; m < kMyTiles; ++m) {
        const int t = wave + 4 * m;
        int it = 0;
        while ((it + 1) * (it + 2) / 2 <= t) ++it;
        tile_i[m] = t < kTiles ? it : -1;
        tile_j[m] = t - it * (it + 1) / 2;
        K[m] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (t < kTiles)
#pragma unroll
            for (int ks = 0; ks < NK; ++ks)
                sel_mma(K[m], sel_rows(s.C + (16 * it + lane_l) * SN + 32 * ks, lane_g),
                        sel_rows(s.B + (16 * tile_j[m] + lane_l) * SN + 32 * ks, lane_g));
        sel_settle(K[m]);
    }

    sel_f4 dB[kMyNT][QT], dC[kMyNT][QT];  // states 16 (wave + 4 m) + 4 g + r of token 16 t + l
#pragma unroll
    for (int m = 0; m < kMyNT; ++m)
#pragma unroll
        for (int t = 0; t < QT; ++t) dB[m][t] = dC[m][t] = sel_f4{0.0f, 0.0f, 0.0f, 0.0f};

    float raw = 0.0f;  // dt + dt_bias of token `lane` (the first wave)
    SelStage<T, Tc, Q, 64, VEC> stage_x, stage_dy;
    SelDt dt;
    // (the next tile's inputs are on their way while one is worked on)
    auto fetch = [&](int head, int p_tile) {
        const int cols = min(64, a.dim - p_tile);
        dt = sel_dt(sel_dt_row(a, seq, head), t0, seq.n);
        stage_x.load(sel_row<T>(a.x, a.tokens, seq, t0) + head * a.x.head + p_tile, a.x.token, n, cols);
        stage_dy.load(sel_row<T>(a.dy, a.tokens, seq, t0) + head * a.dy.head + p_tile, a.dy.token, n, cols);
    };
    fetch(head0, 0);
    for (int head = head0; head < head1; ++head) {
        const float D = a.D ? a.D[head] : 0.0f;
        const float* const S = plan.S + ((long long)chunk * a.n_heads + head) * head_state;
        const float* const G = plan.G + ((long long)chunk * a.n_heads + head) * head_state;
        for (int tile = 0; tile < plan.n_tiles; ++tile) {
            const int p_tile = tile * 64, cols = min(64, a.dim - p_tile);
            // (addresses are formed anew in each tile: kept, they take the registers of the sums)
            int l = lane_l, g = lane_g;
            asm volatile("" : "+v"(l), "+v"(g));
            float Sv[kMyNT][2][8], Gv[kMyNT][2][8];  // columns 16 (wave + 4 m) + l of both states
#pragma unroll
            for (int m = 0; m < kMyNT; ++m)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const int nt = min(wave + 4 * m, NT - 1);
                    state_cols<WHOLE>(S, p_tile + 32 * ks, 16 * nt + l, a.dim, a.states, g, Sv[m][ks]);
                    state_cols<WHOLE>(G, p_tile + 32 * ks, 16 * nt + l, a.dim, a.states, g, Gv[m][ks]);
                }
            __syncthreads();  // the tile before has been read
            stage_x.template store<SX>(s.x, n, cols);
            stage_dy.template store<SX>(s.dy, n, cols);
            if (tile == 0) {
                if (wave == 0)
                    raw = sel_steps<Q>(s.steps, dt.value(a.dt_type), n, a.A[head], a.dt_bias ? a.dt_bias[head] : 0.0f,
                                 a.softplus);
                for (int q = tid; q < QT * Q; q += NHIP_WG) s.over[q / Q][q % Q] = s.col[q / Q][q % Q] = 0.0f;
                for (int q = tid; q < 4 * Q; q += NHIP_WG) s.q[q / Q][q % Q] = s.r[q / Q][q % Q] = 0.0f;
                if (tid < Q) s.diag[tid] = s.dot[tid] = 0.0f;
                if (tid < 4) s.z[tid] = 0.0f;
            }
            __syncthreads();
            {
                const bool more = tile + 1 < plan.n_tiles;
                fetch(more ? head : min(head + 1, head1 - 1), more ? p_tile + 64 : 0);
            }
            float Gr[NK][8];  // row p of G
            const int p = p_tile + 16 * wave + l;
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) state_row<VEC>(G, p, 32 * ks, a.dim, a.states, g, Gr[ks]);

#pragma unroll
            for (int m = 0; m < kMyTiles; ++m) {
                if (tile_i[m] < 0) continue;
                sel_phase();
                const int it = tile_i[m], jt = tile_j[m], j = 16 * jt + l, i0 = 16 * it + 4 * g;
                sel_f4 X = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
                    sel_mma(X, sel_rows(s.dy + (16 * it + l) * SX + 32 * ks, g), sel_rows(s.x + j * SX + 32 * ks, g));
                sel_settle(X);
                const float step = s.steps.step[j];
                const int whole = s.steps.whole[j];
                const float from = 1.0f / s.steps.to[j];
                float kl[4], xl[4], ml[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = i0 + r;
                    const bool in = i >= j;
                    const float L = __builtin_ldexpf(s.steps.to[i] * from, s.steps.whole[i] - whole);
                    const float both = X[r] * L, xl_r = both * step, kl_r = K[m][r] * (L * step), ml_r = K[m][r] * both;
                    xl[r] = in ? xl_r : 0.0f;
                    kl[r] = in ? kl_r : 0.0f;
                    ml[r] = i > j ? ml_r : 0.0f;
                }
                if (it == jt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (i0 + r == j) {
                            s.diag[j] += K[m][r] * X[r];  // (L is one there)
                            s.dot[j] += X[r];
                        }
                // sums over the rows from each on: this lane's four, and those of the quarters behind
#pragma unroll
                for (int r = 2; r >= 0; --r) ml[r] += ml[r + 1];
                float tail = ml[0], other = __shfl_down(tail, 16);
                tail += g < 3 ? other : 0.0f;
                other = __shfl_down(tail, 32);
                tail += g < 2 ? other : 0.0f;
                if (g == 0) s.col[it][j] += tail;
                other = __shfl_down(tail, 16);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = i0 + r;
                    const float over = sel_row_sum(i > j ? (ml[r] + (g < 3 ? other : 0.0f)) * step : 0.0f);
                    if (l == 0) s.over[jt][i] += over;
                }
                Tc* const to = s.pairs[wave + 4 * m] + Tile::at(l, g);
                constexpr int kTable = kTiles * Tile::kSize;
                sel_store_parts(to, to + kTable, xl);
                sel_store_parts(to + kParts * kTable, to + (kParts + 1) * kTable, kl);
            }
            __syncthreads();

            // dx: 16 of the dimension to a wave
            if (16 * wave < cols) {
                SelFrag<Tc> gf[NK][kParts];
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) sel_split(Gr[ks], gf[ks]);
                SelFrag<Tc> df[QK];
#pragma unroll
                for (int ks = 0; ks < QK; ++ks) df[ks] = sel_cols(s.dy + 32 * ks * SX + 16 * wave, SX, l, g);
#pragma unroll
                for (int j2 = 0; j2 < QT; j2 += 2) {
                    sel_phase();
                    sel_f4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                    for (int ks = 0; ks < NK; ++ks) {
                        SelFrag<Tc> b[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) b[u] = sel_rows(s.B + (16 * (j2 + u) + l) * SN + 32 * ks, g);
#pragma unroll
                        for (int q = 0; q < kParts; ++q)
#pragma unroll
                            for (int u = 0; u < 2; ++u) sel_mma(acc[u], gf[ks][q], b[u]);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) acc[u] *= s.steps.to_end_step[16 * (j2 + u) + l];
#pragma unroll
                    for (int ks = j2 / 2; ks < QK; ++ks)
#pragma unroll
                        for (int q = 0; q < kParts; ++q)
#pragma unroll
                            for (int u = 0; u < 2; ++u)
                                sel_mma(acc[u], df[ks], Tile::rows(s.pairs[Lds::K(q, 2 * ks, j2 + u)],
                                                                   s.pairs[Lds::K(q, 2 * ks + 1, j2 + u)], l, g));
                    sel_settle(acc);
                    const int c = 16 * wave + 4 * g;
                    T* const row = static_cast<T*>(a.dx) + ((seq.row0 + t0) * a.n_heads + head) * a.dim + p_tile;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int j = 16 * (j2 + u) + l;
                        float own[4];
                        sel_load<Tc, 4>(s.dy + j * SX + c, own);
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[u][r] = fmaf(D, own[r], acc[u][r]);
                        if (j < n) sel_store4<VEC>(row + (unsigned)j * (unsigned)(a.n_heads * a.dim), c, cols, acc[u]);
                    }
                }
            }

            // dB, dC: every fourth tile of the states to a wave
            float z = 0.0f, qs[QT], rs[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) qs[t] = rs[t] = 0.0f;
#pragma unroll
            for (int m = 0; m < kMyNT; ++m) {
                const int nt = wave + 4 * m;
                if (nt >= NT) continue;
                sel_phase();
                float both = 0.0f;
#pragma unroll
                for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float more = fmaf(Sv[m][ks][e], Gv[m][ks][e], both);
                        both = WHOLE || p_tile + 32 * ks + 16 * (e >> 2) + 4 * g + (e & 3) < a.dim ? more : both;
                    }
                z += 16 * nt + l < a.states ? both : 0.0f;
                SelFrag<Tc> f[2][kSplits];
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) sel_split(Sv[m][ks], f[ks]);
                // (two tiles of tokens at once: the products of one wait for each other)
#pragma unroll
                for (int i2 = 0; i2 < QT; i2 += 2) {
                    sel_phase();
                    sel_f4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        SelFrag<Tc> d[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) d[u] = sel_rows(s.dy + (16 * (i2 + u) + l) * SX + 32 * ks, g);
#pragma unroll
                        for (int q = 0; q < kSplits; ++q)
#pragma unroll
                            for (int u = 0; u < 2; ++u) sel_mma(acc[u], f[ks][q], d[u]);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int i = 16 * (i2 + u) + l;
                        acc[u] *= s.steps.from_start[i];
                        float c[4];
                        sel_load<Tc, 4>(s.C + i * SN + 16 * nt + 4 * g, c);
#pragma unroll
                        for (int r = 0; r < 4; ++r) qs[i2 + u] = fmaf(acc[u][r], c[r], qs[i2 + u]);
                        dC[m][i2 + u] += acc[u];
                    }
#pragma unroll
                    for (int ks = 0; ks <= i2 / 2; ++ks) {
                        const SelFrag<Tc> b = sel_cols(s.B + 32 * ks * SN + 16 * nt, SN, l, g);
#pragma unroll
                        for (int q = 0; q < kParts; ++q)
#pragma unroll
                            for (int u = 0; u < 2; ++u)
                                sel_mma(dC[m][i2 + u], b, Tile::cols(s.pairs[Lds::X(q, i2 + u, 2 * ks)],
                                                                     s.pairs[Lds::X(q, i2 + u, 2 * ks + 1)], l, g));
                    }
                }
                sel_settle(dC[m]);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) sel_split(Gv[m][ks], f[ks]);
#pragma unroll
                for (int j2 = 0; j2 < QT; j2 += 2) {
                    sel_phase();
                    sel_f4 acc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        SelFrag<Tc> d[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) d[u] = sel_rows(s.x + (16 * (j2 + u) + l) * SX + 32 * ks, g);
#pragma unroll
                        for (int q = 0; q < kSplits; ++q)
#pragma unroll
                            for (int u = 0; u < 2; ++u) sel_mma(acc[u], f[ks][q], d[u]);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int j = 16 * (j2 + u) + l;
                        acc[u] *= s.steps.to_end[j];
                        float b[4];
                        sel_load<Tc, 4>(s.B + j * SN + 16 * nt + 4 * g, b);
#pragma unroll
                        for (int r = 0; r < 4; ++r) rs[j2 + u] = fmaf(acc[u][r], b[r], rs[j2 + u]);
                        dB[m][j2 + u] += acc[u] * s.steps.step[j];
                    }
#pragma unroll
                    for (int ks = j2 / 2; ks < QK; ++ks) {
                        const SelFrag<Tc> c = sel_cols(s.C + 32 * ks * SN + 16 * nt, SN, l, g);
#pragma unroll
                        for (int q = 0; q < kParts; ++q)
#pragma unroll
                            for (int u = 0; u < 2; ++u)
                                sel_mma(dB[m][j2 + u], c, Tile::rows(s.pairs[Lds::X(q, 2 * ks, j2 + u)],
                                                                     s.pairs[Lds::X(q, 2 * ks + 1, j2 + u)], l, g));
                    }
                }
                sel_settle(dB[m]);
            }
            z = sel_wave_sum(z);
            if (lane == 0) s.z[wave] += z;
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                qs[t] += __shfl_xor(qs[t], 16);
                qs[t] += __shfl_xor(qs[t], 32);
                rs[t] += __shfl_xor(rs[t], 16);
                rs[t] += __shfl_xor(rs[t], 32);
                if (g == 0) {
                    s.q[wave][16 * t + l] += qs[t];
                    s.r[wave][16 * t + l] += rs[t];
                }
            }
        }
        __syncthreads();
        if (wave == 0) {
            float step = 0.0f, own = 0.0f, r = 0.0f, dot = 0.0f;
            double behind = 0.0, passed = 0.0;  // what counts for the tokens up to this one / behind it
            double across = 0.0;                // the first sum of da
            const bool live = lane < Q && lane < n;
            if (live) {
                step = s.steps.step[lane];
                r = (s.r[0][lane] + s.r[1][lane]) + (s.r[2][lane] + s.r[3][lane]);
                behind = (double)((s.q[0][lane] + s.q[1][lane]) + (s.q[2][lane] + s.q[3][lane]));
                passed = (double)r * (double)step;
                own = s.diag[lane] + r;
                dot = s.dot[lane];
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    across += (double)s.over[t][lane];
                    own += s.col[t][lane];
                }
            }
#pragma unroll
            for (int t = 1; t < QT; ++t) {  // rows of the tiles behind this token's, columns in front of it
                const double v = live ? (double)s.col[t][lane] * (double)step : 0.0;
                const double in_front = sel_prefix(v) - v;
                across += lane < 16 * t ? in_front : 0.0;
            }
            const double sum = sel_prefix(behind), before = sel_prefix(passed) - passed;
            const double all = __shfl(sum, NHIP_WAVE - 1);
            const float z = ((s.z[0] + s.z[1]) + (s.z[2] + s.z[3])) * s.steps.from_start[Q - 1];
            float da = 0.0f, draw = 0.0f;
            if (live) {
                da = (float)(across + (all - sum + behind) + before + (double)z);
                draw = fmaf(a.A[head], da, own);
                if (a.softplus) draw *= 1.0f / (1.0f + expf(-raw));
                sel_set_element(a.ddt, a.dt_type, (seq.row0 + t0 + lane) * a.n_heads + head, draw);
            }
            const float dA = sel_wave_sum(da * step), dD = sel_wave_sum(dot), dbias = sel_wave_sum(draw);
            if (lane == 0) {
                parts[head] = dA;
                parts[a.n_heads + head] = dD;
                parts[2 * a.n_heads + head] = dbias;
            }
        }
    }

    const long long row = (long long)a.n_groups * a.states;
#pragma unroll
    for (int m = 0; m < kMyNT; ++m) {
        const int c = 16 * (wave + 4 * m) + 4 * lane_g;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int i = 16 * t + lane_l;
            if (i >= n || c >= a.states) continue;
            const long long at = (seq.row0 + t0 + i) * row + (long long)group * a.states;
            if (plan.blocks == 1) {
                sel_store4<VEC>(static_cast<T*>(a.dB) + at, c, a.states, dB[m][t]);
                sel_store4<VEC>(static_cast<T*>(a.dC) + at, c, a.states, dC[m][t]);
            } else {
                float* out = plan.shared + (long long)block * 2 * a.tokens.n_tokens * row;
                sel_state_store<VEC>(out + at, c, a.states, dB[m][t]);
                sel_state_store<VEC>(out + a.tokens.n_tokens * row + at, c, a.states, dC[m][t]);
            }
        }
    }
}

// dB and dC from the blocks of heads, in their order: a chunk's rows by `pieces` work-groups, V elements to a lane.  (By
// chunk, so that tokens of no sequence are left as they are: no block has anything of them.)
template <class T, int V>
__global__ __launch_bounds__(NHIP_WG) void add_blocks_kernel(nhip_scan_args a, const float* shared, int blocks, int pieces,
                                                             int q) {
    const int piece = blockIdx.x % pieces;
    const SelSeq seq = sel_seq_of_chunk(a.tokens, blockIdx.x / pieces, q);
    const int t0 = seq.chunk * q, n = seq.seq < 0 ? 0 : min(q, seq.n - t0);
    const long long row = (long long)a.n_groups * a.states, all = a.tokens.n_tokens * row;
    const long long first = (seq.row0 + t0) * row, count = n * row;
    const long long e = ((long long)piece * NHIP_WG + threadIdx.x) * V;
    if (e >= 2 * count) return;
    const bool of_C = e >= count;
    const long long i = first + (of_C ? e - count : e);
    const float* const from = shared + (of_C ? all : 0) + i;
    float sum[V];
    sel_load<float, V>(from, sum);
#pragma unroll 4
    for (int b = 1; b < blocks; ++b) {
        float more[V];
        sel_load<float, V>(from + (long long)b * 2 * all, more);
#pragma unroll
        for (int k = 0; k < V; ++k) sum[k] += more[k];
    }
    sel_store<T, V>(static_cast<T*>(of_C ? a.dC : a.dB) + i, sum);
}

struct Layout {
    SelWalkPlan walk;
    long long n_chunks, states, walk_space, parts, shared;  // floats
    int heads_per_group, blocks;
};

Layout layout(const nhip_scan_args& a) {
    Layout m;
    m.walk = sel_walk_plan(a, 2, nullptr);
    m.walk_space = sel_walk_space(a, m.walk);
    m.n_chunks = m.walk.n_chunks;
    m.states = m.n_chunks * a.n_heads * a.dim * a.states;
    m.parts = m.n_chunks * 3 * a.n_heads;
    // Heads share a work-group, and with it B, C and the sums for their gradients, as long as there are
    // work-groups for every compute unit twice over.
    const int per_group = a.n_heads / a.n_groups;
    long long blocks = m.n_chunks * a.n_groups > 0 ? (512 + m.n_chunks * a.n_groups - 1) / (m.n_chunks * a.n_groups) : 1;
    if (blocks > per_group) blocks = per_group;
    m.heads_per_group = (int)((per_group + blocks - 1) / blocks);
    m.blocks = (per_group + m.heads_per_group - 1) / m.heads_per_group;
    m.shared = m.blocks > 1 ? (long long)m.blocks * 2 * a.tokens.n_tokens * a.n_groups * a.states : 0;
    return m;
}

}  // namespace

extern "C" int nhip_selective_scan_grad_workspace(const nhip_scan_args* args, long long* bytes_out) {
    if (int e = sel_scan_check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    const Layout m = layout(*args);
    if (!sel_walk_fits(*args, m.walk) || m.n_chunks * args->n_groups * m.blocks > SEL_MAX_GROUPS) return NHIP_E_BADARG;
    *bytes_out = 4 * (sel_round4(2 * m.states) + m.walk_space + sel_round4(m.parts) + m.shared);
    return 0;
}

extern "C" int nhip_selective_scan_grad(void* stream, const nhip_scan_args* args) {
    long long need = 0;
    if (int e = nhip_selective_scan_grad_workspace(args, &need)) return e;
    const nhip_scan_args& a = *args;
    if (!a.dA || !a.dD || !a.ddt_bias) return NHIP_E_BADARG;
    if (a.tokens.n_tokens && (!a.dy.p || !a.dx || !a.ddt || !a.dB || !a.dC)) return NHIP_E_BADARG;
    if (need > a.workspace_bytes) return NHIP_E_TOOBIG;
    if (need && (!a.workspace || !sel_aligned(a.workspace, 16))) return NHIP_E_BADARG;
    Layout m = layout(a);
    const long long groups = m.n_chunks * a.n_groups * m.blocks;
    hipStream_t st = static_cast<hipStream_t>(stream);
    m.walk.states = static_cast<float*>(a.workspace);
    float* space = m.walk.states + sel_round4(2 * m.states);
    sel_walk_place(a, m.walk, space);
    float* parts = space + m.walk_space;
    float* shared = parts + sel_round4(m.parts);
    if (int e = sel_walk<kSelStates>(st, a, m.walk, false)) return e;
    int rc = 0;
    if (groups) {
        const GradPlan plan{m.walk.n_tiles, m.heads_per_group, m.blocks, m.n_chunks,
                            m.walk.states, m.walk.states + m.states, parts, shared};
        sel_with_type(a.type, [&](auto t) {
            using T = decltype(t);
            using Tc = typename SelCompute<T>::type;
            sel_with_states(a.states, [&](auto np) {
                constexpr int NP = decltype(np)::value;
                constexpr size_t lds = sizeof(GradLds<Tc, NP>);
                auto kernel = !m.walk.vec       ? grad_kernel<T, Tc, NP, false, false>
                              : a.dim % 64 == 0 ? grad_kernel<T, Tc, NP, true, true>
                                                : grad_kernel<T, Tc, NP, true, false>;
                rc = sel_allow_lds(st, kernel, lds);
                if (rc) return;
                hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(NHIP_WG), lds, st, a, plan);
                rc = (int)hipGetLastError();
            });
            if (!rc && m.blocks > 1) {
                // (there are fewer than 512 chunks and groups, so this is a small grid)
                const int q = sel_chunk_tokens(a.states), per = NHIP_WG * (m.walk.vec ? 4 : 1);
                const int pieces = (int)((2LL * q * a.n_groups * a.states + per - 1) / per);
                auto add = m.walk.vec ? add_blocks_kernel<T, 4> : add_blocks_kernel<T, 1>;
                hipLaunchKernelGGL(add, dim3((unsigned)(m.n_chunks * pieces)), dim3(NHIP_WG), 0, st, a, shared, m.blocks,
                                   pieces, q);
                rc = (int)hipGetLastError();
            }
        });
    }
    if (rc) return rc;
    const long long h = a.n_heads;
    return sel_reduce(st, SelReduce{parts, 3 * h, (int)m.n_chunks, h, 2 * h, a.dA, h, 1, a.dD, a.ddt_bias});
}
