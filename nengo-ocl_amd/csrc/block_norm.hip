// The norm in front of or behind a block, with the block's gate and its residual:
//
//     u = x  or  x gate sigmoid(gate)
//     before a block:  v = residual + scale u,  out = v / sqrt(mean(v^2) + eps) weight
//     after a block:   out = residual + scale (u / sqrt(mean(u^2) + eps) weight)
//
// (means over each of `groups` equal parts of a row) and its gradient.  All of it moves memory:
// every array is read or written once, a part of a row stays in registers between the sum of
// its squares and its use.
#include <type_traits>

#include "selective_common.h"

namespace {

// A part of a row is held by L lanes, V neighbouring channels at a time, R times over; R == 0: a part
// that registers do not hold, read again from the caches.
template <class T, int V>
struct Operands {
    const nhip_norm_args& a;
    long long row;
    int base;  // first channel of the part
    bool before;

    __device__ __forceinline__ void read(const void* p, long long stride, int c, float (&v)[V]) const {
        sel_load<T, V>(static_cast<const T*>(p) + row * stride + base + c, v);
    }
    __device__ __forceinline__ void param(const float* p, int c, float (&v)[V]) const {
        sel_load<float, V>(p + base + c, v);
    }
    // what the norm is taken of
    __device__ __forceinline__ void normed(int c, float (&v)[V]) const {
        read(a.x, a.x_stride, c, v);
        if (a.gate) {
            float g[V];
            read(a.gate, a.gate_stride, c, g);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] *= g[i] * sel_sigmoid(g[i]);
        }
        if (before) {
            float r[V], s[V];
            read(a.residual, a.residual_stride, c, r);
            if (a.scale) param(a.scale, c, s);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = a.scale ? fmaf(s[i], v[i], r[i]) : r[i] + v[i];
        }
    }
};

template <int L>
__device__ __forceinline__ float sum_over(float v, float* s) {
    v = sel_wave_sum(v);
    if constexpr (L > NHIP_WAVE) {
        const int wave = threadIdx.x / NHIP_WAVE;
        __syncthreads();
        if ((threadIdx.x & (NHIP_WAVE - 1)) == 0) s[wave] = v;
        __syncthreads();
        v = (s[0] + s[1]) + (s[2] + s[3]);
    }
    return v;
}

template <class T, int V, int L, int R>
__global__ __launch_bounds__(NHIP_WG) void norm_kernel(nhip_norm_args a) {
    __shared__ float s[8];
    const int lane = threadIdx.x % L, width = a.channels / a.groups;
    const long long part = (long long)blockIdx.x * (NHIP_WG / L) + threadIdx.x / L;
    if (part >= a.rows * a.groups) return;  // uniform over the lanes that share a part
    const Operands<T, V> op{a, part / a.groups, (int)(part % a.groups) * width, a.residual && !a.after};
    constexpr int kHeld = R ? R : 1;
    float v[kHeld][V];
    float sum = 0.0f;
    T* const v_out = op.before ? static_cast<T*>(a.v_out) + op.row * a.channels + op.base : nullptr;
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * L + lane) * V;
            if (c < width) {
                op.normed(c, v[r]);
#pragma unroll
                for (int i = 0; i < V; ++i) sum = fmaf(v[r][i], v[r][i], sum);
                if (v_out) sel_store<T, V>(v_out + c, v[r]);
            }
        }
    } else {
        for (int c = lane * V; c < width; c += L * V) {
            op.normed(c, v[0]);
#pragma unroll
            for (int i = 0; i < V; ++i) sum = fmaf(v[0][i], v[0][i], sum);
            if (v_out) sel_store<T, V>(v_out + c, v[0]);
        }
    }
    sum = sum_over<L>(sum, s);
    const float inv = 1.0f / sqrtf(sum / (float)width + a.eps);
    T* const out = static_cast<T*>(a.out) + op.row * a.channels + op.base;
    auto finish = [&](int c, float(&u)[V]) {
        float w[V];
        op.param(a.weight, c, w);
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = u[i] * inv * w[i];
        if (a.after && a.residual) {
            float r[V];
            op.read(a.residual, a.residual_stride, c, r);
            if (a.scale) op.param(a.scale, c, w);
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] = a.scale ? fmaf(w[i], u[i], r[i]) : r[i] + u[i];
        }
        sel_store<T, V>(out + c, u);
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * L + lane) * V;
            if (c < width) finish(c, v[r]);
        }
    } else {
        for (int c = lane * V; c < width; c += L * V) {
            op.normed(c, v[0]);
            finish(c, v[0]);
        }
    }
}

// With n = v inv (inv = 1 / sqrt(mean(v^2) + eps)) and e the gradient of n weight (dout, times
// scale behind a block): dweight = sum over rows of e n;  dv = inv (e weight - n mean(e weight n)).
// Each group of lanes keeps its channels over its rows (every gridDim.x-th) and the sums for
// weight and scale with them; a second launch adds the groups' sums up in their order.
template <class T, int V, int L, int R>
__global__ __launch_bounds__(NHIP_WG) void norm_grad_kernel(nhip_norm_args a, float* parts) {
    __shared__ float s[8];
    __shared__ float both[R > 0 && L == NHIP_WAVE ? 4 * NHIP_WAVE * V : 1];
    constexpr int kWaves = NHIP_WG / L;  // rows side by side
    const int lane = threadIdx.x % L, mine = threadIdx.x / L, width = a.channels / a.groups;
    const int base = blockIdx.y * width;
    const bool before = a.residual && !a.after, behind = a.residual && a.after;
    constexpr int kHeld = R ? R : 1;
    float dw[kHeld][V], ds[kHeld][V];
    float* const row_w = parts + (long long)blockIdx.x * 2 * a.channels + base;
    float* const row_s = row_w + a.channels;
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[r][i] = ds[r][i] = 0.0f;
    if constexpr (R == 0) {
        for (int c = lane * V; c < width; c += L * V)
#pragma unroll
            for (int i = 0; i < V; ++i) row_w[c + i] = row_s[c + i] = 0.0f;
    }
    for (long long row = (long long)blockIdx.x * kWaves + mine; row < a.rows;
         row += (long long)gridDim.x * kWaves) {
        const Operands<T, V> op{a, row, base, before};
        float v[kHeld][V], e[kHeld][V];
        float sum = 0.0f, dot = 0.0f;
        auto first = [&](int c, float(&u)[V], float(&g)[V]) {
            float w[V];
            op.normed(c, u);
            op.read(a.dout, a.dout_stride, c, g);
            op.param(a.weight, c, w);
            if (behind && a.scale) {
                float k[V];
                op.param(a.scale, c, k);
#pragma unroll
                for (int i = 0; i < V; ++i) w[i] *= k[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                sum = fmaf(u[i], u[i], sum);
                dot = fmaf(g[i] * w[i], u[i], dot);
            }
        };
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int c = (r * L + lane) * V;
                if (c < width) first(c, v[r], e[r]);
            }
        } else {
            for (int c = lane * V; c < width; c += L * V) first(c, v[0], e[0]);
        }
        sum = sum_over<L>(sum, s);
        dot = sum_over<L>(dot, s + 4);
        const float inv = 1.0f / sqrtf(sum / (float)width + a.eps);
        const float mean = dot * inv / (float)width;
        const long long at = row * a.channels + base;
        auto second = [&](int c, float(&u)[V], float(&g)[V], float(&w_sum)[V], float(&s_sum)[V]) {
            float w[V], k[V], d[V];
            op.param(a.weight, c, w);
#pragma unroll
            for (int i = 0; i < V; ++i) k[i] = 1.0f;
            if (a.scale) op.param(a.scale, c, k);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float n = u[i] * inv;
                const float to_w = behind ? g[i] * k[i] : g[i];  // gradient of n weight
                w_sum[i] = fmaf(to_w, n, w_sum[i]);
                if (behind) s_sum[i] = fmaf(g[i], n * w[i], s_sum[i]);
                d[i] = inv * fmaf(-n, mean, to_w * w[i]);
            }
            float x[V], gate[V], f[V];
            if (before || a.gate) op.read(a.x, a.x_stride, c, x);
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = 1.0f;
            if (a.gate) {
                op.read(a.gate, a.gate_stride, c, gate);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = sel_sigmoid(gate[i]);
            }
            if (before) {
                if (a.dv) {
                    float more[V];
                    op.read(a.dv, a.dv_stride, c, more);
#pragma unroll
                    for (int i = 0; i < V; ++i) d[i] += more[i];
                }
                if (a.dresidual) sel_store<T, V>(static_cast<T*>(a.dresidual) + at + c, d);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s_sum[i] = fmaf(d[i], a.gate ? x[i] * (gate[i] * f[i]) : x[i], s_sum[i]);
                    d[i] *= k[i];
                }
            }
            if (a.gate) {
                float dg[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    dg[i] = d[i] * x[i] * (f[i] * fmaf(gate[i], 1.0f - f[i], 1.0f));
                    d[i] *= gate[i] * f[i];
                }
                sel_store<T, V>(static_cast<T*>(a.dgate) + at + c, dg);
            }
            sel_store<T, V>(static_cast<T*>(a.dx) + at + c, d);
        };
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int c = (r * L + lane) * V;
                if (c < width) second(c, v[r], e[r], dw[r], ds[r]);
            }
        } else {
            for (int c = lane * V; c < width; c += L * V) {
                op.normed(c, v[0]);
                op.read(a.dout, a.dout_stride, c, e[0]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    dw[0][i] = row_w[c + i];
                    ds[0][i] = row_s[c + i];
                }
                second(c, v[0], e[0], dw[0], ds[0]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    row_w[c + i] = dw[0][i];
                    row_s[c + i] = ds[0][i];
                }
            }
        }
    }
    if constexpr (R > 0) {
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float m[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    m[i] = which ? ds[0][i] : dw[0][i];
#pragma unroll
                    for (int q = 1; q < R; ++q) m[i] = r == q ? (which ? ds[q][i] : dw[q][i]) : m[i];
                }
                float* const out = which ? row_s : row_w;
                const int c = (r * L + lane) * V;
                if constexpr (L == NHIP_WAVE) {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < V; ++i) both[(mine * NHIP_WAVE + lane) * V + i] = m[i];
                    __syncthreads();
                    if (mine == 0 && c < width)
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const int q = lane * V + i;
                            out[c + i] = (both[q] + both[NHIP_WAVE * V + q]) +
                                         (both[2 * NHIP_WAVE * V + q] + both[3 * NHIP_WAVE * V + q]);
                        }
                } else if (c < width) {
#pragma unroll
                    for (int i = 0; i < V; ++i) out[c + i] = m[i];
                }
            }
        }
    }
}

// How a part of `width` channels is held: a wave up to 1024 16-bit channels (512 of 32 bits),
// a group of four waves up to four times as many, and longer ones are read twice.
template <class F> void with_shape(bool vec, int per16, int width, F&& f) {
    const int v = vec ? per16 : 1;
    auto go = [&](auto lanes, auto held) {
        if (vec) f(std::true_type(), lanes, held);
        else f(std::false_type(), lanes, held);
    };
    using std::integral_constant;
    if (width <= 64 * v) go(integral_constant<int, 64>(), integral_constant<int, 1>());
    else if (width <= 128 * v) go(integral_constant<int, 64>(), integral_constant<int, 2>());
    else if (width <= 256 * v) go(integral_constant<int, 256>(), integral_constant<int, 1>());
    else if (width <= 512 * v) go(integral_constant<int, 256>(), integral_constant<int, 2>());
    else if (width <= 1024 * v) go(integral_constant<int, 256>(), integral_constant<int, 4>());
    else go(integral_constant<int, 256>(), integral_constant<int, 0>());
}

bool wide(const nhip_norm_args& a) {
    const int v = 16 / sel_size(a.type);
    if ((a.channels / a.groups) % v) return false;
    for (const void* p : {a.x, a.gate, a.residual, (const void*)a.weight, (const void*)a.scale,
                          (const void*)a.out, (const void*)a.v_out, a.dout, a.dv, (const void*)a.dx,
                          (const void*)a.dgate, (const void*)a.dresidual})
        if (!sel_aligned(p, 16)) return false;
    for (long long s : {a.x_stride, a.gate ? a.gate_stride : 0, a.residual ? a.residual_stride : 0,
                        a.dout ? a.dout_stride : 0, a.dv ? a.dv_stride : 0})
        if (s % v) return false;
    return true;
}

int check(const nhip_norm_args* a) {
    if (!a || a->channels <= 0 || a->groups <= 0 || a->channels % a->groups || a->rows < 0) return NHIP_E_BADARG;
    if (a->type < NHIP_F32 || a->type > NHIP_F16 || !a->weight) return NHIP_E_BADARG;
    // (arrays without elements may be null)
    if (a->rows && (!a->x || (a->scale && !a->residual))) return NHIP_E_BADARG;
    if (a->rows * a->groups > 0x7fffffffLL || a->groups > SEL_MAX_GRID_Y) return NHIP_E_BADARG;
    return 0;
}

// Rows of the table of sums: one per group of waves along the rows.  2048 groups over all parts
// give each of the 256 compute units eight; a few rows each, or the table costs more than the rows.
int sum_rows(const nhip_norm_args& a) {
    long long n = a.rows / 8;
    const long long most = 2048 / a.groups > 1 ? 2048 / a.groups : 1;
    if (n > most) n = most;
    return n < 1 ? 1 : (int)n;
}

}  // namespace

extern "C" int nhip_block_norm(void* stream, const nhip_norm_args* args) {
    if (int e = check(args)) return e;
    const nhip_norm_args& a = *args;
    if (a.rows == 0) return 0;
    if (!a.out) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    const int width = a.channels / a.groups;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        constexpr int V16 = 16 / sizeof(T);
        with_shape(wide(a), V16, width, [&](auto vec, auto lanes, auto held) {
            constexpr int V = decltype(vec)::value ? V16 : 1, L = decltype(lanes)::value, R = decltype(held)::value;
            const long long parts = a.rows * a.groups;
            constexpr int per = NHIP_WG / L;
            NHIP_LAUNCH((norm_kernel<T, V, L, R>), dim3((unsigned)((parts + per - 1) / per)), dim3(NHIP_WG), 0,
                        static_cast<hipStream_t>(stream), a);
            rc = (int)hipGetLastError();
        });
    });
    return rc;
}

extern "C" int nhip_block_norm_grad_workspace(const nhip_norm_args* args, long long* bytes_out) {
    if (int e = check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    *bytes_out = (long long)sum_rows(*args) * 2 * args->channels * 4;
    return 0;
}

extern "C" int nhip_block_norm_grad(void* stream, const nhip_norm_args* args) {
    long long need = 0;
    if (int e = nhip_block_norm_grad_workspace(args, &need)) return e;
    const nhip_norm_args& a = *args;
    if (!a.dweight || (a.scale && !a.dscale)) return NHIP_E_BADARG;
    if (a.rows && (!a.dout || !a.dx || (a.gate && !a.dgate))) return NHIP_E_BADARG;
    if (need > a.workspace_bytes) return NHIP_E_TOOBIG;
    if (!a.workspace) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    const int width = a.channels / a.groups, rows = sum_rows(a);
    float* parts = static_cast<float*>(a.workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        constexpr int V16 = 4;  // (8 bytes of 16-bit types: what a lane holds of eight channels leaves too few waves)
        with_shape(wide(a), V16, width, [&](auto vec, auto lanes, auto held) {
            constexpr int V = decltype(vec)::value ? V16 : 1, L = decltype(lanes)::value, R = decltype(held)::value;
            NHIP_LAUNCH_FIRST((norm_grad_kernel<T, V, L, R>), dim3((unsigned)rows, (unsigned)a.groups),
                              dim3(NHIP_WG), 0, st, a, parts);
            rc = (int)hipGetLastError();
        });
    });
    if (rc) return rc;
    return sel_reduce(st, SelReduce{parts, 2LL * a.channels, rows, a.channels, 2LL * a.channels, a.dweight,
                                    a.channels, 1, a.dscale, nullptr});
}
