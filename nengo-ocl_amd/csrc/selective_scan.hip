// The selective scan over prompts, and its step for single tokens.
#include <type_traits>

#include "selective_scan.h"

namespace {

// One token: S <- e^{step A} S + step x (x) B, y = S C + D x.  The state is read and written, 8 bytes
// per element for 5 operations: memory bound.  Lanes of a wave share the rows of a head's state: LPR
// (a power of two) to a row, V neighbouring states at a time.
template <class T, int V>
__global__ __launch_bounds__(NHIP_WG) void step_kernel(nhip_scan_step_args a, int lpr, int rows_per_group) {
    const int blocks = (a.dim + rows_per_group - 1) / rows_per_group;
    const int block = blockIdx.x % blocks;
    const int head = (blockIdx.x / blocks) % a.n_heads;
    const int r = blockIdx.x / (blocks * a.n_heads);
    const int slot = a.slots ? a.slots[r] : r;
    const int group = head / (a.n_heads / a.n_groups);
    const int c = threadIdx.x % lpr, side_by_side = NHIP_WG / lpr;
    const bool live = slot >= 0 && slot < a.n_slots;
    T* const y = static_cast<T*>(a.y) + ((long long)r * a.n_heads + head) * a.dim;
    const T* const x = static_cast<const T*>(a.x.p) + r * a.x.token + head * a.x.head;
    const T* const B = static_cast<const T*>(a.B.p) + r * a.B.token + group * a.B.head;
    const T* const C = static_cast<const T*>(a.C.p) + r * a.C.token + group * a.C.head;
    const float raw = sel_element(a.dt.p, a.dt_type, r * a.dt.token + head * a.dt.head) +
                      (a.dt_bias ? a.dt_bias[head] : 0.0f);
    const float step = a.softplus ? sel_softplus(raw) : raw;
    const float decay = expf(step * a.A[head]);
    const float D = a.D ? a.D[head] : 0.0f;
    const int p1 = min(a.dim, (block + 1) * rows_per_group);
    for (int p0 = block * rows_per_group; p0 < p1; p0 += side_by_side) {
        const int p = p0 + threadIdx.x / lpr;
        float sum = 0.0f;
        if (p < p1 && live) {
            const float in = step * (float)x[p];
            float* const row = a.state + slot * a.state_stride + ((long long)head * a.dim + p) * a.states;
            for (int n = c * V; n < a.states; n += lpr * V) {
                float v[V], b[V], k[V];
                sel_load<float, V>(row + n, v);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    b[i] = (float)B[n + i];
                    k[i] = (float)C[n + i];
                    v[i] = fmaf(decay, v[i], in * b[i]);
                    sum = fmaf(v[i], k[i], sum);
                }
                sel_store<float, V>(row + n, v);
            }
        }
        for (int d = lpr / 2; d > 0; d /= 2) sum += __shfl_xor(sum, d);
        if (c == 0 && p < p1) y[p] = (T)(live ? fmaf(D, (float)x[p], sum) : 0.0f);
    }
}

}  // namespace

extern "C" int nhip_selective_scan_workspace(const nhip_scan_args* args, long long* bytes_out) {
    if (int e = sel_scan_check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    *bytes_out = 4 * sel_walk_space(*args, sel_walk_plan(*args, 1, nullptr));
    return 0;
}

extern "C" int nhip_selective_scan(void* stream, const nhip_scan_args* args) {
    if (int e = sel_scan_check(args)) return e;
    const nhip_scan_args& a = *args;
    if (a.tokens.n_tokens && !a.y) return NHIP_E_BADARG;
    SelWalkPlan plan = sel_walk_plan(a, 1, nullptr);
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
    const int side_by_side = NHIP_WG / lpr;
    const int rows = side_by_side * 2;
    const long long groups = (long long)a.n * a.n_heads * ((a.dim + rows - 1) / rows);
    if (groups > 0x7fffffffLL) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        if (vec)
            NHIP_LAUNCH((step_kernel<T, 4>), dim3((unsigned)groups), dim3(NHIP_WG), 0, static_cast<hipStream_t>(stream), a, lpr, rows);
        else
            NHIP_LAUNCH((step_kernel<T, 1>), dim3((unsigned)groups), dim3(NHIP_WG), 0, static_cast<hipStream_t>(stream), a, lpr, rows);
        rc = (int)hipGetLastError();
    });
    return rc;
}
