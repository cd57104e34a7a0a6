// The layer norm and its gradient, with the residual in front of it:
//
//     v = x  or  residual + x,   m = mean(v),   u = (v - m) / sqrt(mean((v - m)^2) + eps),   out = u weight + bias
//     with e = dout weight:   dv += (e - mean(e) - u mean(e u)) / sqrt(...),   dweight = sum dout u,   dbias = sum dout
//
// All of it moves memory: every array is read or written once, a row stays in registers between its sums and their
// use.  The mean is taken away before squares are summed, so that a mean far from zero costs no digits.
//
// Rows that registers do not hold are read three times: forward above 1024 packs of 16 bytes (8192 channels of 16 bits; 1024 where rows
// are no whole packs), backward above 4096 channels (1024), where the sums for weight and bias go through memory for each
// row, too.  bfloat16 with a residual, 8192 rows: forward 1504 channels 17 us, 1500 48, 8192 111; gradient 1504 channels 52 us,
// 1500 111, 4096 125, 8192 495 (134 for its bytes).
#include "norm_rows.h"

namespace {

template <class T, int V, int L, int R>
__global__ __launch_bounds__(NHIP_WG) void layer_norm_kernel(nhip_layer_norm_args a) {
    __shared__ float s[8];
    const int lane = threadIdx.x % L, width = a.channels;
    const long long row = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * (NHIP_WG / L) + threadIdx.x / L;
    if (row >= a.rows) return;  // uniform over the lanes that share a row
    constexpr int kHeld = R ? R : 1;
    T* const out = static_cast<T*>(a.out) + row * width;
    T* const v_out = a.residual ? static_cast<T*>(a.v_out) + row * width : nullptr;
    auto read = [&](int c, float(&v)[V]) {
        sel_load<T, V>(static_cast<const T*>(a.x) + row * a.x_stride + c, v);
        if (a.residual) {
            float r[V];
            sel_load<T, V>(static_cast<const T*>(a.residual) + row * a.residual_stride + c, r);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += r[i];
        }
    };
    // over the channels of this lane: f(channel, values), which are read again where registers do not hold them
    float v[kHeld][V];
    auto each = [&](auto first, auto&& f) {
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int c = (r * L + lane) * V;
                if (c < width) {
                    if constexpr (decltype(first)::value) read(c, v[r]);
                    f(c, v[r]);
                }
            }
        } else {
            for (int c = lane * V; c < width; c += L * V) {
                read(c, v[0]);
                f(c, v[0]);
            }
        }
    };
    float sum = 0.0f, squares = 0.0f;
    each(std::true_type(), [&](int c, float(&u)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += u[i];
        if (v_out) sel_store<T, V>(v_out + c, u);
    });
    const float mean = norm_sum<L>(sum, s) / (float)width;
    each(std::false_type(), [&](int c, float(&u)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) squares = fmaf(u[i] - mean, u[i] - mean, squares);
    });
    const float inv = 1.0f / sqrtf(norm_sum<L>(squares, s + 4) / (float)width + a.eps);
    each(std::false_type(), [&](int c, float(&u)[V]) {
        float w[V], b[V], y[V];
        sel_load<float, V>(a.weight + c, w);
        if (a.bias) sel_load<float, V>(a.bias + c, b);
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = fmaf((u[i] - mean) * inv, w[i], a.bias ? b[i] : 0.0f);
        sel_store<T, V>(out + c, y);
    });
}

// Each group of lanes keeps its channels over its rows (every gridDim.x-th) and the sums for weight and bias with them; a
// second launch adds the groups' sums up in their order.  The next row is on its way while one is worked on.
template <class T, int V, int L, int R>
__global__ __launch_bounds__(NHIP_WG, 2) void layer_norm_grad_kernel(nhip_layer_norm_args a, float* parts) {
    __shared__ float s[16];
    __shared__ float both[R > 0 && L == NHIP_WAVE ? 4 * NHIP_WAVE * V : 1];
    constexpr int kWaves = NHIP_WG / L;  // rows side by side
    const int lane = threadIdx.x % L, mine = threadIdx.x / L, width = a.channels;
    float* const row_w = parts + (long long)blockIdx.x * 2 * width;
    float* const row_b = row_w + width;
    const long long step = (long long)gridDim.x * kWaves, row0 = (long long)blockIdx.x * kWaves + mine;

    struct Raw {
        SelPack<T, V> x, residual, dout, dv;
    };
    // loads are unconditional, from channels and rows cut to those that exist: one under a condition is waited
    // for where its branch ends
    auto fetch = [&](Raw& raw, long long row, int c) {
        const long long r = min(row, a.rows - 1);
        const int at = min(c, width - V);
        auto get = [&](const void* p, long long stride) {
            return *reinterpret_cast<const SelPack<T, V>*>(static_cast<const T*>(p) + r * stride + at);
        };
        raw.x = get(a.x, a.x_stride);
        raw.dout = get(a.dout, a.dout_stride);
        if (a.residual) raw.residual = get(a.residual, a.residual_stride);
        if (a.dv) raw.dv = get(a.dv, a.dv_stride);
    };
    struct Values {
        float v[V], d[V];  // what the norm is taken of, dout
    };
    auto open = [&](const Raw& raw, Values& u) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            u.v[i] = (float)raw.x.v[i];
            if (a.residual) u.v[i] += (float)raw.residual.v[i];
            u.d[i] = (float)raw.dout.v[i];
        }
    };
    auto weights = [&](int c, float(&w)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = a.weight[min(c, width - V) + i];
    };
    auto close = [&](long long row, int c, const Values& u, const Raw& raw, const float(&w)[V], float mean, float inv, float m_e,
                     float m_eu, float(&dw)[V], float(&db)[V]) {
        if (c >= width) return;
        float d[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float n = (u.v[i] - mean) * inv;
            dw[i] = fmaf(u.d[i], n, dw[i]);
            db[i] += u.d[i];
            d[i] = inv * (fmaf(-n, m_eu, u.d[i] * w[i]) - m_e);
            if (a.dv) d[i] += (float)raw.dv.v[i];
        }
        sel_store<T, V>(static_cast<T*>(a.dx) + row * width + c, d);
    };
    auto channel = [&](int r) { return (r * L + lane) * V; };
    auto sum_v = [&](int c, const Values& u, float& sum) {
        if (c >= width) return;
#pragma unroll
        for (int i = 0; i < V; ++i) sum += u.v[i];
    };
    auto sum_rest = [&](int c, const Values& u, const float(&w)[V], float mean, float& squares, float& e, float& eu) {
        if (c >= width) return;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float off = u.v[i] - mean, t = u.d[i] * w[i];
            squares = fmaf(off, off, squares);
            e += t;
            eu = fmaf(t, off, eu);
        }
    };
    const float per = 1.0f / (float)width;
    // A row's sums, between waves through words of `s` that the sums before them do not use: one barrier each, since whoever
    // writes there again has passed the other one in between.  (The norm of 8192 x 2048 in bfloat16 with four barriers to
    // a sum, 46 us; with one to all three, 41.)
    auto first_sum = [&](float v) {
        v = sel_wave_sum(v);
        if constexpr (L > NHIP_WAVE) {
            if (lane % NHIP_WAVE == 0) s[threadIdx.x / NHIP_WAVE] = v;
            __syncthreads();
            v = (s[0] + s[1]) + (s[2] + s[3]);
        }
        return v;
    };
    auto finish = [&](float& squares, float& e, float& eu) {
        squares = sel_wave_sum(squares);
        e = sel_wave_sum(e);
        eu = sel_wave_sum(eu);
        if constexpr (L > NHIP_WAVE) {
            const int w = threadIdx.x / NHIP_WAVE;
            if (lane % NHIP_WAVE == 0) {
                s[4 + w] = squares;
                s[8 + w] = e;
                s[12 + w] = eu;
            }
            __syncthreads();
            squares = (s[4] + s[5]) + (s[6] + s[7]);
            e = (s[8] + s[9]) + (s[10] + s[11]);
            eu = (s[12] + s[13]) + (s[14] + s[15]);
        }
        const float inv = 1.0f / sqrtf(squares / (float)width + a.eps);
        e *= per;
        eu *= inv * per;
        return inv;
    };

    if constexpr (R > 0) {
        constexpr bool kAhead = R * V * sizeof(T) <= 32;
        float w[R][V], dw[R][V], db[R][V];
        Raw raw[R], next[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            weights(channel(r), w[r]);
            if (a.rows) fetch(next[r], row0, channel(r));
#pragma unroll
            for (int i = 0; i < V; ++i) dw[r][i] = db[r][i] = 0.0f;
        }
        for (long long row = row0; row < a.rows; row += step) {
            Values u[R];
            float sum = 0.0f, squares = 0.0f, e = 0.0f, eu = 0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (kAhead || row == row0) raw[r] = next[r];
                else fetch(raw[r], row, channel(r));
                open(raw[r], u[r]);
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (kAhead) fetch(next[r], row + step, channel(r));
#pragma unroll
            for (int r = 0; r < R; ++r) sum_v(channel(r), u[r], sum);
            const float mean = first_sum(sum) / (float)width;
#pragma unroll
            for (int r = 0; r < R; ++r) sum_rest(channel(r), u[r], w[r], mean, squares, e, eu);
            const float inv = finish(squares, e, eu);
#pragma unroll
            for (int r = 0; r < R; ++r) close(row, channel(r), u[r], raw[r], w[r], mean, inv, e, eu, dw[r], db[r]);
        }
        // the waves' sums, or the group's own
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                float* const to = which ? row_b : row_w;
                const int c = channel(r);
                if constexpr (L == NHIP_WAVE) {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < V; ++i) both[(mine * NHIP_WAVE + lane) * V + i] = which ? db[r][i] : dw[r][i];
                    __syncthreads();
                    if (mine == 0 && c < width)
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const int q = lane * V + i;
                            to[c + i] = (both[q] + both[NHIP_WAVE * V + q]) +
                                        (both[2 * NHIP_WAVE * V + q] + both[3 * NHIP_WAVE * V + q]);
                        }
                } else if (c < width) {
#pragma unroll
                    for (int i = 0; i < V; ++i) to[c + i] = which ? db[r][i] : dw[r][i];
                }
            }
    } else {
        for (int c = lane * V; c < width; c += L * V)
#pragma unroll
            for (int i = 0; i < V; ++i) row_w[c + i] = row_b[c + i] = 0.0f;
        for (long long row = row0; row < a.rows; row += step) {
            float sum = 0.0f, squares = 0.0f, e = 0.0f, eu = 0.0f, w[V], dw[V], db[V];
            Raw raw;
            Values u;
            for (int c = lane * V; c < width; c += L * V) {
                fetch(raw, row, c);
                open(raw, u);
                sum_v(c, u, sum);
            }
            const float mean = first_sum(sum) / (float)width;
            for (int c = lane * V; c < width; c += L * V) {
                weights(c, w);
                fetch(raw, row, c);
                open(raw, u);
                sum_rest(c, u, w, mean, squares, e, eu);
            }
            const float inv = finish(squares, e, eu);
            for (int c = lane * V; c < width; c += L * V) {
                weights(c, w);
                fetch(raw, row, c);
                open(raw, u);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    dw[i] = row_w[c + i];
                    db[i] = row_b[c + i];
                }
                close(row, c, u, raw, w, mean, inv, e, eu, dw, db);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    row_w[c + i] = dw[i];
                    row_b[c + i] = db[i];
                }
            }
        }
    }
}

// Whether every row begins at a multiple of 16 bytes and holds whole packs of 16
bool wide(const nhip_layer_norm_args& a) {
    const int v = 16 / sel_size(a.type);
    if (a.channels % v) return false;
    for (const void* p : {a.x, a.residual, (const void*)a.weight, (const void*)a.bias, (const void*)a.out, (const void*)a.v_out,
                          a.dout, a.dv, (const void*)a.dx})
        if (!sel_aligned(p, 16)) return false;
    for (long long s : {a.x_stride, a.residual ? a.residual_stride : 0, a.dout ? a.dout_stride : 0, a.dv ? a.dv_stride : 0})
        if (s % v) return false;
    return true;
}

int check(const nhip_layer_norm_args* a) {
    if (!a || a->channels <= 0 || a->channels >= 1 << 27 || a->rows < 0 || a->rows > 0x7fffffffLL) return NHIP_E_BADARG;
    if (a->type < NHIP_F32 || a->type > NHIP_F16 || !a->weight || !(a->eps >= 0.0f)) return NHIP_E_BADARG;
    if (a->rows && !a->x) return NHIP_E_BADARG;
    return 0;
}

// Rows of the table of sums: one per group of waves along the rows; eight rows each at least, or the table costs more
// than the rows.
int sum_rows(long long rows, int groups) {
    const long long n = rows / 8;
    return (int)(n > groups ? groups : n < 1 ? 1 : n);
}
constexpr int kMostGroups = 2048;
template <class T, int V, int R> constexpr int groups_at_once() {
    return 256 * (V == 1 || R < 2 ? 8 : R == 2 && sizeof(T) == 2 ? 3 : 2);
}

}  // namespace

extern "C" int nhip_layer_norm(void* stream, const nhip_layer_norm_args* args) {
    if (int e = check(args)) return e;
    const nhip_layer_norm_args& a = *args;
    if (a.rows == 0) return 0;
    if (!a.out || (a.residual && !a.v_out)) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        constexpr int V16 = 16 / sizeof(T);
        norm_with_shape(wide(a), V16, a.channels, [&](auto vec, auto lanes, auto held) {
            constexpr int V = decltype(vec)::value ? V16 : 1, L = decltype(lanes)::value, R = decltype(held)::value;
            constexpr int per = NHIP_WG / L;
            // (an axis of a grid has fewer than 2^32 threads)
            const long long n = (a.rows + per - 1) / per, across = n < 65536 ? n : 65536;
            NHIP_LAUNCH((layer_norm_kernel<T, V, L, R>), dim3((unsigned)across, (unsigned)((n + across - 1) / across)),
                        dim3(NHIP_WG), 0, static_cast<hipStream_t>(stream), a);
            rc = (int)hipGetLastError();
        });
    });
    return rc;
}

extern "C" int nhip_layer_norm_grad_workspace(const nhip_layer_norm_args* args, long long* bytes_out) {
    if (int e = check(args)) return e;
    if (!bytes_out || 2LL * args->channels > SEL_MAX_SUMS) return NHIP_E_BADARG;
    *bytes_out = (long long)sum_rows(args->rows, kMostGroups) * 2 * args->channels * 4;
    return 0;
}

extern "C" int nhip_layer_norm_grad(void* stream, const nhip_layer_norm_args* args) {
    long long need = 0;
    if (int e = nhip_layer_norm_grad_workspace(args, &need)) return e;
    const nhip_layer_norm_args& a = *args;
    if (!a.dweight || (a.bias && !a.dbias)) return NHIP_E_BADARG;
    if (a.rows && (!a.dout || !a.dx || (a.dv && !a.residual))) return NHIP_E_BADARG;
    if (need > a.workspace_bytes) return NHIP_E_TOOBIG;
    if (!a.workspace) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG, rows = 0;
    float* parts = static_cast<float*>(a.workspace);
    hipStream_t st = static_cast<hipStream_t>(stream);
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        constexpr int V16 = 4;  // (8 bytes of 16-bit types: what a lane holds of eight channels leaves too few waves)
        norm_with_shape(wide(a), V16, a.channels, [&](auto vec, auto lanes, auto held) {
            constexpr int V = decltype(vec)::value ? V16 : 1, L = decltype(lanes)::value, R = decltype(held)::value;
            rows = sum_rows(a.rows, groups_at_once<T, V, R>());
            NHIP_LAUNCH_FIRST((layer_norm_grad_kernel<T, V, L, R>), dim3((unsigned)rows), dim3(NHIP_WG), 0, st, a, parts);
            rc = (int)hipGetLastError();
        });
    });
    if (rc) return rc;
    return sel_reduce(st, SelReduce{parts, 2LL * a.channels, rows, a.channels, 2LL * a.channels, a.dweight, a.channels, 1,
                                    a.bias ? a.dbias : nullptr, nullptr});
}
