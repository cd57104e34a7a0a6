// The norm in front of or behind a block, with the block's gate and its residual:
//
//     u = x  or  x gate sigmoid(gate)
//     before a block:  v = residual + scale u,  out = v / sqrt(mean(v^2) + eps) weight
//     after a block:   out = residual + scale (u / sqrt(mean(u^2) + eps) weight)
//
// (means over each of `groups` equal parts of a row) and its gradient.  All of it moves memory:
// every array is read or written once, a part of a row stays in registers between the sum of
// its squares and its use.  16384 rows of 2048 in four groups with a gate, bfloat16: 201 MB in 37 us, 5.4 TB/s.
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
    const long long part = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * (NHIP_WG / L) + threadIdx.x / L;
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
// weight and scale with them; a second launch adds the groups' sums up in their order.  The next row is on its
// way while one is worked on (8192 rows of 2048, bfloat16, residual: 37 us for 201 MB, 53 without).
template <class T, int V, int L, int R>
__global__ __launch_bounds__(NHIP_WG, 2) void norm_grad_kernel(nhip_norm_args a, float* parts) {
    __shared__ float s[8];
    __shared__ float both[R > 0 && L == NHIP_WAVE ? 4 * NHIP_WAVE * V : 1];
    constexpr int kWaves = NHIP_WG / L;  // rows side by side
    const int lane = threadIdx.x % L, mine = threadIdx.x / L, width = a.channels / a.groups;
    const int base = blockIdx.y * width;
    const bool before = a.residual && !a.after, behind = a.residual && a.after;
    float* const row_w = parts + (long long)blockIdx.x * 2 * a.channels + base;
    float* const row_s = row_w + a.channels;
    const long long step = (long long)gridDim.x * kWaves;

    // What a lane needs of V channels of a row
    struct Raw {
        SelPack<T, V> x, gate, residual, dout, dv;
    };
    // loads are unconditional, from channels and rows cut to those that exist: one under a condition is waited
    // for where its branch ends
    auto fetch = [&](Raw& raw, long long row, int c) {
        const long long r = min(row, a.rows - 1);
        const int at = base + min(c, width - V);
        auto get = [&](const void* p, long long stride) {
            return *reinterpret_cast<const SelPack<T, V>*>(static_cast<const T*>(p) + r * stride + at);
        };
        raw.x = get(a.x, a.x_stride);
        raw.dout = get(a.dout, a.dout_stride);
        if (a.gate) raw.gate = get(a.gate, a.gate_stride);
        if (before) raw.residual = get(a.residual, a.residual_stride);
        if (a.dv) raw.dv = get(a.dv, a.dv_stride);
    };
    struct Values {
        float v[V], e[V], x[V], f[V], slope[V], more[V];  // normed, dout, x, gate sigmoid(gate), its derivative, dv
    };
    auto params = [&](int c, float(&w)[V], float(&k)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = a.weight[base + min(c, width - V) + i];
            k[i] = a.scale ? a.scale[base + min(c, width - V) + i] : 1.0f;
        }
    };
    auto open = [&](const Raw& raw, const float(&k)[V], Values& u) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            u.x[i] = (float)raw.x.v[i];
            u.e[i] = (float)raw.dout.v[i];
            u.f[i] = 1.0f;
            u.slope[i] = 0.0f;
            if (a.gate) {
                const float g = (float)raw.gate.v[i], sg = sel_sigmoid(g);
                u.f[i] = g * sg;
                u.slope[i] = sg * fmaf(g, 1.0f - sg, 1.0f);
            }
            u.v[i] = u.x[i] * u.f[i];
            if (before) u.v[i] = fmaf(k[i], u.v[i], (float)raw.residual.v[i]);
            u.more[i] = a.dv ? (float)raw.dv.v[i] : 0.0f;
        }
    };
    auto sums = [&](int c, const Values& u, const float(&w)[V], const float(&k)[V], float& sum, float& dot) {
        if (c >= width) return;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sum = fmaf(u.v[i], u.v[i], sum);
            dot = fmaf(u.e[i] * (behind ? w[i] * k[i] : w[i]), u.v[i], dot);
        }
    };
    auto close = [&](long long row, int c, const Values& u, const float(&w)[V], const float(&k)[V], float inv, float mean,
                     float(&dw)[V], float(&ds)[V]) {
        if (c >= width) return;
        const long long at = row * a.channels + base + c;
        float d[V], dg[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float n = u.v[i] * inv;
            const float to_w = behind ? u.e[i] * k[i] : u.e[i];  // gradient of n weight
            dw[i] = fmaf(to_w, n, dw[i]);
            d[i] = fmaf(inv, fmaf(-n, mean, to_w * w[i]), u.more[i]);
            if (behind) ds[i] = fmaf(u.e[i], n * w[i], ds[i]);
        }
        if (before) {
            if (a.dresidual) sel_store<T, V>(static_cast<T*>(a.dresidual) + at, d);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                ds[i] = fmaf(d[i], u.x[i] * u.f[i], ds[i]);
                d[i] *= k[i];
            }
        }
        if (a.gate) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dg[i] = d[i] * u.x[i] * u.slope[i];
                d[i] *= u.f[i];
            }
            sel_store<T, V>(static_cast<T*>(a.dgate) + at, dg);
        }
        sel_store<T, V>(static_cast<T*>(a.dx) + at, d);
    };
    auto channel = [&](int r) { return (r * L + lane) * V; };
    const long long row0 = (long long)blockIdx.x * kWaves + mine;

    if constexpr (R > 0) {
        // (more channels to a lane leave no registers for the next row: 4096 rows of 4096, 32 bits, 169 us with it, 59.5 without)
        constexpr bool kAhead = R * V * sizeof(T) <= 32;
        float w[R][V], k[R][V], dw[R][V], ds[R][V];
        Raw raw[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            params(channel(r), w[r], k[r]);
            if (kAhead && a.rows) fetch(raw[r], row0, channel(r));
#pragma unroll
            for (int i = 0; i < V; ++i) dw[r][i] = ds[r][i] = 0.0f;
        }
        for (long long row = row0; row < a.rows; row += step) {
            Values u[R];
            float sum = 0.0f, dot = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (!kAhead) fetch(raw[r], row, channel(r));
#pragma unroll
            for (int r = 0; r < R; ++r) open(raw[r], k[r], u[r]);
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (kAhead) fetch(raw[r], row + step, channel(r));
#pragma unroll
            for (int r = 0; r < R; ++r) sums(channel(r), u[r], w[r], k[r], sum, dot);
            sum = sum_over<L>(sum, s);
            dot = sum_over<L>(dot, s + 4);
            const float inv = 1.0f / sqrtf(sum / (float)width + a.eps);
            const float mean = dot * inv / (float)width;
#pragma unroll
            for (int r = 0; r < R; ++r) close(row, channel(r), u[r], w[r], k[r], inv, mean, dw[r], ds[r]);
        }
        // the waves' sums, or the group's own
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float* const out = which ? row_s : row_w;
                const int c = channel(r);
                if constexpr (L == NHIP_WAVE) {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < V; ++i) both[(mine * NHIP_WAVE + lane) * V + i] = which ? ds[r][i] : dw[r][i];
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
                    for (int i = 0; i < V; ++i) out[c + i] = which ? ds[r][i] : dw[r][i];
                }
            }
    } else {
        for (int c = lane * V; c < width; c += L * V)
#pragma unroll
            for (int i = 0; i < V; ++i) row_w[c + i] = row_s[c + i] = 0.0f;
        for (long long row = row0; row < a.rows; row += step) {
            float sum = 0.0f, dot = 0.0f, w[V], k[V], dw[V], ds[V];
            Raw raw;
            Values u;
            for (int c = lane * V; c < width; c += L * V) {
                params(c, w, k);
                fetch(raw, row, c);
                open(raw, k, u);
                sums(c, u, w, k, sum, dot);
            }
            sum = sum_over<L>(sum, s);
            dot = sum_over<L>(dot, s + 4);
            const float inv = 1.0f / sqrtf(sum / (float)width + a.eps);
            const float mean = dot * inv / (float)width;
            for (int c = lane * V; c < width; c += L * V) {
                params(c, w, k);
                fetch(raw, row, c);
                open(raw, k, u);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    dw[i] = row_w[c + i];
                    ds[i] = row_s[c + i];
                }
                close(row, c, u, w, k, inv, mean, dw, ds);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    row_w[c + i] = dw[i];
                    row_s[c + i] = ds[i];
                }
            }
        }
    }
}

// How a part of `width` channels is held, `per16` of them side by side in a lane (one where rows do not allow
// wide reads): by a wave up to 128 times as many, by a group of four waves up to 1024 times; longer ones are read twice.
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

// Whether every part of a row begins at a multiple of 16 bytes and holds whole packs of 16.  (The gradient's lanes, which
// take 8 bytes of 16-bit types, go by the same rule.)
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

// Rows of the table of sums: one per group of waves along the rows.  `groups` over all parts; eight rows each
// at least, or the table costs more than the rows.
int sum_rows(const nhip_norm_args& a, int groups) {
    const long long n = a.rows / 8, most = groups / a.groups > 1 ? groups / a.groups : 1;
    return (int)(n > most ? most : n < 1 ? 1 : n);
}
constexpr int kMostGroups = 2048;
// As many groups as run at once, by the registers that a lane takes, where it takes many (8192 rows of 2048 with a
// residual: bfloat16, three to a compute unit, 56.7 us with 1024 groups, 48.9 with 768, 48.4 with 512, 60.3 with
// 256; 32 bits, two to a unit, 44.9 us with 1024, 49.9 with 768, 41.3 with 512), otherwise twice as many, which
// share the rows more evenly (parts of 256, bfloat16, with a gate: 42.2 us with 1024, 39.4 with 2048).
template <class T, int V, int R> constexpr int groups_at_once() {
    return 256 * (V == 1 || R < 2 ? 8 : R == 2 && sizeof(T) == 2 ? 3 : 2);
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
            // (an axis of a grid has fewer than 2^32 threads)
            const long long n = (parts + per - 1) / per, across = n < 65536 ? n : 65536;
            NHIP_LAUNCH((norm_kernel<T, V, L, R>), dim3((unsigned)across, (unsigned)((n + across - 1) / across)),
                        dim3(NHIP_WG), 0, static_cast<hipStream_t>(stream), a);
            rc = (int)hipGetLastError();
        });
    });
    return rc;
}

extern "C" int nhip_block_norm_grad_workspace(const nhip_norm_args* args, long long* bytes_out) {
    if (int e = check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    *bytes_out = (long long)sum_rows(*args, kMostGroups) * 2 * args->channels * 4;
    return 0;
}

extern "C" int nhip_block_norm_grad(void* stream, const nhip_norm_args* args) {
    long long need = 0;
    if (int e = nhip_block_norm_grad_workspace(args, &need)) return e;
    const nhip_norm_args& a = *args;
    if (!a.dweight || (a.scale && !a.dscale)) return NHIP_E_BADARG;
    if (a.channels >= 1 << 27) return NHIP_E_BADARG;  // (columns of the sums' launch: 16 threads each, two to a channel)
    if (a.rows && (!a.dout || !a.dx || (a.gate && !a.dgate))) return NHIP_E_BADARG;
    if (need > a.workspace_bytes) return NHIP_E_TOOBIG;
    if (!a.workspace) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    const int width = a.channels / a.groups;
    int rows = 0;
    float* parts = static_cast<float*>(a.workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        constexpr int V16 = 4;  // (8 bytes of 16-bit types: what a lane holds of eight channels leaves too few waves)
        with_shape(wide(a), V16, width, [&](auto vec, auto lanes, auto held) {
            constexpr int V = decltype(vec)::value ? V16 : 1, L = decltype(lanes)::value, R = decltype(held)::value;
            rows = sum_rows(a, groups_at_once<T, V, R>());
            NHIP_LAUNCH_FIRST((norm_grad_kernel<T, V, L, R>), dim3((unsigned)rows, (unsigned)a.groups),
                              dim3(NHIP_WG), 0, st, a, parts);
            rc = (int)hipGetLastError();
        });
    });
    if (rc) return rc;
    return sel_reduce(st, SelReduce{parts, 2LL * a.channels, rows, a.channels, 2LL * a.channels, a.dweight,
                                    a.channels, 1, a.dscale, nullptr});
}
