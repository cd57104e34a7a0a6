// The selective scan over prompts, and its step for single tokens.
#include <type_traits>

#include "selective_scan.h"

namespace {

// One token: S <- e^{step A} S + step x (x) B, y = S C + D x.  The state is read and written, 8 bytes
// per element for 5 operations: memory bound.  Lanes of a wave share the rows of a head's state: LPR
// (a power of two) to a row, V neighbouring states NS times over; each takes ROWS rows, whose loads are all
// under way before the first is used, and B and C stay in registers for all of them.  128 requests, 64 heads of 64,
// 128 states: 537 MB in 96 us, 5.6 TB/s; one request, 24 heads of 64, 64 states: 4.0 us.
template <class T, int V, int NS, int ROWS>
__global__ __launch_bounds__(NHIP_WG) void step_kernel(nhip_scan_step_args a, int lpr) {
    const int side_by_side = NHIP_WG / lpr, per_group = side_by_side * ROWS;
    const int blocks = (a.dim + per_group - 1) / per_group;
    const int block = blockIdx.x % blocks;
    const int head = (blockIdx.x / blocks) % a.n_heads;
    const int r = blockIdx.x / (blocks * a.n_heads);
    const int slot = a.slots ? a.slots[r] : r;
    const int group = head / (a.n_heads / a.n_groups);
    const int c = threadIdx.x % lpr, p0 = block * per_group + threadIdx.x / lpr;
    T* const y = static_cast<T*>(a.y) + ((long long)r * a.n_heads + head) * a.dim;
    if (slot < 0 || slot >= a.n_slots) {
        for (int q = 0; q < ROWS; ++q) {
            const int p = p0 + q * side_by_side;
            if (c == 0 && p < a.dim) y[p] = (T)0.0f;
        }
        return;
    }
    float* const state = a.state + slot * a.state_stride + (long long)head * a.dim * a.states;
    float v[ROWS][NS][V];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
        const float* row = state + (unsigned)min(p0 + q * side_by_side, a.dim - 1) * (unsigned)a.states;
#pragma unroll
        for (int s = 0; s < NS; ++s) sel_load<float, V>(row + min((c + s * lpr) * V, a.states - V), v[q][s]);
    }
    const T* const x = static_cast<const T*>(a.x.p) + r * a.x.token + head * a.x.head;
    const T* const B = static_cast<const T*>(a.B.p) + r * a.B.token + group * a.B.head;
    const T* const C = static_cast<const T*>(a.C.p) + r * a.C.token + group * a.C.head;
    float b[NS][V], k[NS][V], in[ROWS];
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int n = (c + s * lpr) * V + i;
            b[s][i] = (float)B[min(n, a.states - 1)];
            k[s][i] = n < a.states ? (float)C[min(n, a.states - 1)] : 0.0f;
        }
#pragma unroll
    for (int q = 0; q < ROWS; ++q) in[q] = (float)x[min(p0 + q * side_by_side, a.dim - 1)];
    const float raw = sel_element(a.dt.p, a.dt_type, r * a.dt.token + head * a.dt.head) +
                      (a.dt_bias ? a.dt_bias[head] : 0.0f);
    const float step = a.softplus ? sel_softplus(raw) : raw;
    const float decay = sel_exp(step * a.A[head]);
    const float D = a.D ? a.D[head] : 0.0f;
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
        const int p = p0 + q * side_by_side;
        const float gain = step * in[q];
        float* const row = state + (unsigned)p * (unsigned)a.states;
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int n = (c + s * lpr) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[q][s][i] = fmaf(decay, v[q][s][i], gain * b[s][i]);
                sum = fmaf(n < a.states ? v[q][s][i] : 0.0f, k[s][i], sum);
            }
            if (p < a.dim && n < a.states) sel_store_past<float, V>(row + n, v[q][s]);
        }
        for (int d = lpr / 2; d > 0; d /= 2) sum += __shfl_xor(sum, d);
        if (c == 0 && p < a.dim) y[p] = (T)fmaf(D, in[q], sum);
    }
}

}  // namespace

extern "C" int nhip_selective_scan_workspace(const nhip_scan_args* args, long long* bytes_out) {
    if (int e = sel_scan_check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    const SelWalkPlan plan = sel_walk_plan(*args, 1, nullptr);
    if (!sel_walk_fits(*args, plan)) return NHIP_E_BADARG;
    *bytes_out = 4 * sel_walk_space(*args, plan);
    return 0;
}

extern "C" int nhip_selective_scan(void* stream, const nhip_scan_args* args) {
    if (int e = sel_scan_check(args)) return e;
    const nhip_scan_args& a = *args;
    if (a.tokens.n_tokens && !a.y) return NHIP_E_BADARG;
    SelWalkPlan plan = sel_walk_plan(a, 1, nullptr);
    if (!sel_walk_fits(a, plan)) return NHIP_E_BADARG;
    const long long need = 4 * sel_walk_space(a, plan);
    if (need > a.workspace_bytes) return NHIP_E_TOOBIG;
    if (need && (!a.workspace || !sel_aligned(a.workspace, 16))) return NHIP_E_BADARG;
    sel_walk_place(a, plan, static_cast<float*>(a.workspace));
    return sel_walk<kSelOutputs>(static_cast<hipStream_t>(stream), a, plan, true);
}

extern "C" int nhip_selective_step(void* stream, const nhip_scan_step_args* args) {
    if (!args || !args->A || args->n_heads <= 0 || args->dim <= 0 || args->n_groups <= 0 ||
        args->n_heads % args->n_groups || args->states < 1 || args->states > 256 || args->n < 0 || args->n_slots < 0)
        return NHIP_E_BADARG;
    const nhip_scan_step_args& a = *args;
    if (a.type < NHIP_F32 || a.type > NHIP_F16 || a.dt_type < NHIP_F32 || a.dt_type > NHIP_F16) return NHIP_E_BADARG;
    if (a.n == 0) return 0;
    if (!a.x.p || !a.dt.p || !a.B.p || !a.C.p || !a.state || !a.y) return NHIP_E_BADARG;
    const bool vec = a.states % 4 == 0 && sel_aligned(a.state, 16) && a.state_stride % 4 == 0;
    const int v = vec ? 4 : 1;
    int lpr = 1;
    while (lpr < NHIP_WAVE && lpr * v < a.states) lpr *= 2;
    // Eight rows to a lane where that leaves four work-groups to every compute unit, otherwise one.
    const int side_by_side = NHIP_WG / lpr;
    const bool many = (long long)a.n * a.n_heads * ((a.dim + 8 * side_by_side - 1) / (8 * side_by_side)) >= 1024;
    const int rows = side_by_side * (many ? 8 : 1);
    const long long groups = (long long)a.n * a.n_heads * ((a.dim + rows - 1) / rows);
    if (groups > SEL_MAX_GROUPS || (long long)a.dim * a.states > 0x7fffffffLL) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        const dim3 g((unsigned)groups);
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (vec && many) NHIP_LAUNCH((step_kernel<T, 4, 1, 8>), g, dim3(NHIP_WG), 0, st, a, lpr);
        else if (vec) NHIP_LAUNCH((step_kernel<T, 4, 1, 1>), g, dim3(NHIP_WG), 0, st, a, lpr);
        else if (many) NHIP_LAUNCH((step_kernel<T, 1, 4, 8>), g, dim3(NHIP_WG), 0, st, a, lpr);
        else NHIP_LAUNCH((step_kernel<T, 1, 4, 1>), g, dim3(NHIP_WG), 0, st, a, lpr);
        rc = (int)hipGetLastError();
    });
    return rc;
}
