// The short causal convolution along a sequence, channel by channel (a filter with `width`
// taps per channel in front of a selective scan), its gradient and its step for single tokens.
//
//     u[t, d] = bias[d] + sum_k weight[d, k] x[t - width + 1 + k, d],   y = u  or  u sigmoid(u)
//
// The operators move memory: 2 width + 6 operations per element of 2 or 4 bytes.  A lane
// takes 16 bytes of neighbouring channels and goes along a strip of tokens with the window in
// registers, so that each input is read once (and width - 1 rows again where strips meet, from
// the caches).  8 x 2048 tokens, 2304 channels, four taps, bfloat16: 151 MB in 30.9 us, 4.9 TB/s, where a copy
// reaches 5.1; its gradient 54 us for 226 MB, 4.2 TB/s.
#include <type_traits>

#include "selective_common.h"

namespace {

constexpr int kStrip = 16;           // tokens that a wave goes along
constexpr int kChunk = 4 * kStrip;   // tokens of a work-group: four waves
constexpr int kMaxWidth = 8;

// lane's channels: c0 ... c0 + V - 1
template <class T, int V>
__device__ __forceinline__ int first_channel() {
    return (blockIdx.y * NHIP_WAVE + (threadIdx.x & (NHIP_WAVE - 1))) * V;
}

// Input of token t of the sequence: of `initial` in front of its first token, zero beyond both
// ends.
template <class T, int V, int K>
__device__ __forceinline__ void load_token(const nhip_conv_args& a, const SelSeq& s, int t, int c0,
                                           float (&v)[V]) {
    if (t >= 0 && t < s.n) {
        sel_load<T, V>(sel_row<T>(a.x, a.tokens, s, t) + c0, v);
    } else if (t < 0 && a.initial && t >= 1 - K) {
        sel_load<T, V>(static_cast<const T*>(a.initial) +
                           ((long long)s.seq * (K - 1) + (K - 1 + t)) * a.channels + c0, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.0f;
    }
}

// Taps and bias of this lane's channels.  The group's lie back to back, V K floats to a lane: read by neighbouring
// threads and handed over through the LDS (a lane's own V K reads touch as many lines as the inputs of
// its whole strip).
template <int V, int K> struct Taps {
    static constexpr int kRow = NHIP_WAVE + 1;
    float at[V * K][kRow];
};
template <int V, int K>
__device__ __forceinline__ void load_taps(const nhip_conv_args& a, int c0, Taps<V, K>& s, float (&w)[K][V], float (&b)[V]) {
    const long long first = (long long)blockIdx.y * NHIP_WAVE * V * K, end = (long long)a.channels * K;
    constexpr int kAll = NHIP_WAVE * V * K;
#pragma unroll
    for (int q0 = 0; q0 < kAll; q0 += NHIP_WG) {
        const int q = q0 + threadIdx.x;
        const float v = a.weight[min(first + q, end - 1)];
        if (q < kAll) s.at[q % (V * K)][q / (V * K)] = v;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = a.bias ? a.bias[min(c0 + i, a.channels - 1)] : 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = s.at[i * K + k][threadIdx.x & (NHIP_WAVE - 1)];
}

template <class T, int V, int K>
__global__ __launch_bounds__(NHIP_WG) void conv_kernel(nhip_conv_args a) {
    const SelSeq s = sel_seq_of_chunk(a.tokens, blockIdx.x, kChunk);
    if (s.seq < 0) return;
    __shared__ Taps<V, K> taps;
    const int c0 = first_channel<T, V>();
    const int t0 = s.chunk * kChunk + (threadIdx.x / NHIP_WAVE) * kStrip;
    float w[K][V], b[V];
    load_taps<V, K>(a, c0, taps, w, b);
    if (c0 >= a.channels) return;
    const int t1 = min(t0 + kStrip, s.n);
    if (t0 < t1) {
        // All tokens of the strip are under way before the first is used.  (The loads are unconditional, the last
        // token again where the strip ends early: one under a condition is waited for where its branch ends.)
        SelPack<T, V> in[kStrip];
        const T* const from = sel_row<T>(a.x, a.tokens, s, t0) + c0;
#pragma unroll
        for (int k = 0; k < kStrip; ++k)
            in[k] = *reinterpret_cast<const SelPack<T, V>*>(from + min(k, t1 - 1 - t0) * a.x.token);
        float x[K][V];  // the window: x[k] is token t - K + 1 + k
#pragma unroll
        for (int k = 0; k < K - 1; ++k) load_token<T, V, K>(a, s, t0 - K + 1 + k, c0, x[k]);
        T* const out = static_cast<T*>(a.y) + (s.row0 + t0) * a.channels + c0;
#pragma unroll
        for (int q = 0; q < kStrip; ++q) {
            float u[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x[K - 1][i] = (float)in[q].v[i];
                u[i] = b[i];
#pragma unroll
                for (int k = 0; k < K; ++k) u[i] = fmaf(w[k][i], x[k][i], u[i]);
                if (a.silu) u[i] *= sel_sigmoid(u[i]);
            }
            if (q < t1 - t0) sel_store_past<T, V>(out + (long long)q * a.channels, u);
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) x[k][i] = x[k + 1][i];
        }
    }
    // the last chunk's first wave hands on the end of the sequence
    if (a.final && K > 1 && threadIdx.x < NHIP_WAVE && s.chunk == sel_chunks(s.n, kChunk) - 1) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            float v[V];
            load_token<T, V, K>(a, s, s.n + j - (K - 1), c0, v);
            sel_store<T, V>(static_cast<T*>(a.final) + ((long long)s.seq * (K - 1) + j) * a.channels + c0, v);
        }
    }
}

// dx[t] = sum_k weight[k] g[t + K - 1 - k], g = dy f'(u).  A strip goes on over the K - 1 tokens
// behind it, whose g its last tokens need; g is zero outside the sequence.  The sums for the
// taps go to a row of the workspace per chunk, [K + 1][channels], and are added up by a second
// launch in the order of the chunks: the same result on every call.  5003 tokens in seven sequences, 1100
// channels, 32 bits: 21.2 us for 66 MB, and 4.0 for the sums; 425 work-groups, not two to a compute unit, of which
// each has 19 tokens of a strip to get through, eight under way at once (the next four behind those that are worked on:
// 8 x 2048 tokens, 2304 channels, bfloat16, 67 us without, 56 with; the waves' sums handed over all at once, 54).
template <class T, int V, int K>
__global__ __launch_bounds__(NHIP_WG) void conv_grad_kernel(nhip_conv_args a, float* parts) {
    __shared__ union {
        Taps<V, K> taps;
        float sums[K + 1][4][NHIP_WAVE * V];
    } lds;
    const int chunk = blockIdx.x;
    const SelSeq s = sel_seq_of_chunk(a.tokens, chunk, kChunk);
    const int c0 = first_channel<T, V>();
    const bool here = s.seq >= 0 && c0 < a.channels;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NHIP_WAVE), lane = threadIdx.x & (NHIP_WAVE - 1);
    float w[K][V], b[V], dw[K + 1][V];
    load_taps<V, K>(a, c0, lds.taps, w, b);
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = 0.0f;
    if (here) {
        const int t0 = s.chunk * kChunk + wave * kStrip;
        const int t1 = min(t0 + kStrip, s.n);
        // the sequence's first strip also forms what goes to `initial`: rows of t < 0
        const int from = s.chunk == 0 && wave == 0 && a.dinitial ? 1 - K : t0;
        if (from < t1 || from < 0) {
            float x[K][V], g[K][V];  // x[k], g[k]: token t - K + 1 + k
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (k < K - 1) load_token<T, V, K>(a, s, t0 - K + 1 + k, c0, x[k]);
#pragma unroll
                for (int i = 0; i < V; ++i) g[k][i] = 0.0f;
            }
            constexpr int kAhead = 4;  // tokens fetched at once, from places cut to those that exist
            const T* const x_at = s.n ? sel_row<T>(a.x, a.tokens, s, 0) + c0 : nullptr;
            const T* const dy_at = s.n ? sel_row<T>(a.dy, a.tokens, s, 0) + c0 : nullptr;
            const int t_end = max(t1, t0) + K - 1;
            SelPack<T, V> next_x[kAhead], next_dy[kAhead];
            auto fetch = [&](int t_first) {
#pragma unroll
                for (int q = 0; q < kAhead; ++q) {
                    const long long at = min(t_first + q, s.n - 1);
                    next_x[q] = *reinterpret_cast<const SelPack<T, V>*>(x_at + at * a.x.token);
                    next_dy[q] = *reinterpret_cast<const SelPack<T, V>*>(dy_at + at * a.dy.token);
                }
            };
            if (s.n) fetch(t0);
            for (int t_first = t0; t_first < t_end; t_first += kAhead) {
                SelPack<T, V> xs[kAhead], dys[kAhead];
#pragma unroll
                for (int q = 0; q < kAhead; ++q) {
                    xs[q] = next_x[q];
                    dys[q] = next_dy[q];
                }
                if (s.n) fetch(t_first + kAhead);
#pragma unroll
                for (int q = 0; q < kAhead; ++q) {
                    const int t = t_first + q;
                    const bool in = t < s.n;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        x[K - 1][i] = in ? (float)xs[q].v[i] : 0.0f;
                        float d = (float)dys[q].v[i];
                        if (a.silu) {
                            float u = b[i];
#pragma unroll
                            for (int k = 0; k < K; ++k) u = fmaf(w[k][i], x[k][i], u);
                            const float sg = sel_sigmoid(u);
                            d *= sg * fmaf(u, 1.0f - sg, 1.0f);
                        }
                        g[K - 1][i] = in ? d : 0.0f;
                    }
                    if (t < t1) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
#pragma unroll
                            for (int k = 0; k < K; ++k) dw[k][i] = fmaf(g[K - 1][i], x[k][i], dw[k][i]);
                            dw[K][i] += g[K - 1][i];
                        }
                    }
                    const int td = t - (K - 1);  // the token whose gradient is complete
                    if (td >= from && t < t_end) {
                        float dx[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            dx[i] = 0.0f;
#pragma unroll
                            for (int k = 0; k < K; ++k) dx[i] = fmaf(w[k][i], g[K - 1 - k][i], dx[i]);
                        }
                        const int j = td + (K - 1) - s.n;  // its place among the last K - 1 inputs
                        if (a.dfinal && j >= 0) {
                            float more[V];
                            sel_load<T, V>(static_cast<const T*>(a.dfinal) +
                                               ((long long)s.seq * (K - 1) + j) * a.channels + c0, more);
#pragma unroll
                            for (int i = 0; i < V; ++i) dx[i] += more[i];
                        }
                        T* out = td >= 0 ? static_cast<T*>(a.dx) + (s.row0 + td) * a.channels + c0
                                         : static_cast<T*>(a.dinitial) +
                                               ((long long)s.seq * (K - 1) + (K - 1 + td)) * a.channels + c0;
                        sel_store<T, V>(out, dx);
                    }
#pragma unroll
                    for (int k = 0; k < K - 1; ++k)
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            x[k][i] = x[k + 1][i];
                            g[k][i] = g[k + 1][i];
                        }
                }
            }
        }
    }
    __syncthreads();  // (the taps have been read)
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) lds.sums[k][wave][lane * V + i] = dw[k][i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k <= K; ++k)
        for (int c = threadIdx.x; c < NHIP_WAVE * V; c += NHIP_WG) {
            const int d = blockIdx.y * NHIP_WAVE * V + c;
            if (d < a.channels)
                parts[((long long)chunk * (K + 1) + k) * a.channels + d] =
                    (lds.sums[k][0][c] + lds.sums[k][1][c]) + (lds.sums[k][2][c] + lds.sums[k][3][c]);
        }
}

// One token each: width - 1 rows of a slot and the input are read, the rows written one place on.  A launch's own
// time at any number of requests that is served at once (64, 2304 channels, bfloat16: 4.7 us for 2.4 MB).
template <class T, int V, int K>
__global__ __launch_bounds__(NHIP_WG) void conv_step_kernel(nhip_conv_step_args a) {
    const int per = (a.channels + V - 1) / V;
    const long long i0 = (long long)blockIdx.x * NHIP_WG + threadIdx.x;
    if (i0 >= (long long)a.n * per) return;
    const int r = (int)(i0 / per), c0 = (int)(i0 % per) * V;
    const int slot = a.slots ? a.slots[r] : r;
    float u[V];
    if (slot >= 0 && slot < a.n_slots) {
        T* state = static_cast<T*>(a.state) + slot * a.state_stride + c0;
        float x[K][V];
#pragma unroll
        for (int k = 0; k < K - 1; ++k) sel_load<T, V>(state + (long long)k * a.channels, x[k]);
        sel_load<T, V>(static_cast<const T*>(a.x) + r * a.x_stride + c0, x[K - 1]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            u[i] = a.bias ? a.bias[c0 + i] : 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k)
                u[i] = fmaf(a.weight[(long long)(c0 + i) * K + k], x[k][i], u[i]);
            if (a.silu) u[i] *= sel_sigmoid(u[i]);
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k) sel_store<T, V>(state + (long long)k * a.channels, x[k + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = 0.0f;
    }
    sel_store<T, V>(static_cast<T*>(a.y) + (long long)r * a.channels + c0, u);
}

template <class F> bool with_width(int width, F&& f) {
    switch (width) {
        case 1: f(std::integral_constant<int, 1>()); return true;
        case 2: f(std::integral_constant<int, 2>()); return true;
        case 3: f(std::integral_constant<int, 3>()); return true;
        case 4: f(std::integral_constant<int, 4>()); return true;
        case 5: f(std::integral_constant<int, 5>()); return true;
        case 6: f(std::integral_constant<int, 6>()); return true;
        case 7: f(std::integral_constant<int, 7>()); return true;
        case 8: f(std::integral_constant<int, 8>()); return true;
    }
    return false;
}

// A lane reads 16 bytes of neighbouring channels where every row begins at a multiple of 16 bytes,
// otherwise one channel.  (The gradient's lanes, which take 8 bytes of 16-bit types, go by the same rule.)
bool wide(int type, int channels, std::initializer_list<const void*> pointers,
          std::initializer_list<long long> strides) {
    const int v = 16 / sel_size(type);
    if (channels % v) return false;
    for (const void* p : pointers)
        if (!sel_aligned(p, 16)) return false;
    for (long long s : strides)
        if (s % v) return false;
    return true;
}

int check(const nhip_conv_args* a) {
    if (!a || !a->weight || a->channels <= 0 || a->width < 1 || a->width > kMaxWidth) return NHIP_E_BADARG;
    if (a->type < NHIP_F32 || a->type > NHIP_F16 || !sel_tokens_ok(a->tokens)) return NHIP_E_BADARG;
    if (a->tokens.n_tokens && !a->x.p) return NHIP_E_BADARG;
    if (sel_max_chunks(a->tokens, kChunk) > SEL_MAX_GROUPS || a->channels > SEL_MAX_GRID_Y * NHIP_WAVE)
        return NHIP_E_BADARG;
    return 0;
}

bool grid(const nhip_conv_args& a, int v, dim3* g) {
    const long long chunks = sel_max_chunks(a.tokens, kChunk);
    *g = dim3((unsigned)chunks, (unsigned)((a.channels + NHIP_WAVE * v - 1) / (NHIP_WAVE * v)));
    return chunks > 0;
}

}  // namespace

extern "C" int nhip_causal_conv(void* stream, const nhip_conv_args* args) {
    if (int e = check(args)) return e;
    const nhip_conv_args& a = *args;
    if (a.tokens.n_tokens && !a.y) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        with_width(a.width, [&](auto k) {
            constexpr int K = decltype(k)::value, V = 16 / sizeof(T);
            dim3 g;
            hipStream_t st = static_cast<hipStream_t>(stream);
            if (wide(a.type, a.channels, {a.x.p, a.initial, a.y, a.final}, {a.x.seq, a.x.token})) {
                if (grid(a, V, &g)) NHIP_LAUNCH((conv_kernel<T, V, K>), g, dim3(NHIP_WG), 0, st, a);
            } else {
                if (grid(a, 1, &g)) NHIP_LAUNCH((conv_kernel<T, 1, K>), g, dim3(NHIP_WG), 0, st, a);
            }
            rc = (int)hipGetLastError();
        });
    });
    return rc;
}

extern "C" int nhip_causal_conv_grad_workspace(const nhip_conv_args* args, long long* bytes_out) {
    if (int e = check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    *bytes_out = sel_max_chunks(args->tokens, kChunk) * (args->width + 1) * args->channels * 4;
    return 0;
}

extern "C" int nhip_causal_conv_grad(void* stream, const nhip_conv_args* args) {
    long long need = 0;
    if (int e = nhip_causal_conv_grad_workspace(args, &need)) return e;
    const nhip_conv_args& a = *args;
    if (a.tokens.n_tokens && (!a.dy.p || !a.dx)) return NHIP_E_BADARG;
    if (!a.dweight || !a.dbias) return NHIP_E_BADARG;
    if (need > a.workspace_bytes) return NHIP_E_TOOBIG;
    if (need && !a.workspace) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    hipStream_t st = static_cast<hipStream_t>(stream);
    float* parts = static_cast<float*>(a.workspace);
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        with_width(a.width, [&](auto k) {
            // (four channels of 16 bits too: the window, its gradient and the sums of eight take all registers)
            constexpr int K = decltype(k)::value, V = 4;
            dim3 g;
            if (wide(a.type, a.channels, {a.x.p, a.dy.p, a.initial, a.dfinal, a.dx, a.dinitial},
                     {a.x.seq, a.x.token, a.dy.seq, a.dy.token})) {
                if (grid(a, V, &g))
                    NHIP_LAUNCH_FIRST((conv_grad_kernel<T, V, K>), g, dim3(NHIP_WG), 0, st, a, parts);
            } else {
                if (grid(a, 1, &g))
                    NHIP_LAUNCH_FIRST((conv_grad_kernel<T, 1, K>), g, dim3(NHIP_WG), 0, st, a, parts);
            }
            rc = (int)hipGetLastError();
        });
    });
    if (rc) return rc;
    const int rows = (int)sel_max_chunks(a.tokens, kChunk);
    const long long taps = (long long)a.width * a.channels, n = taps + a.channels;
    // columns of a row of `parts`: tap k of channel d at k * channels + d; dweight is [channels, width]
    return sel_reduce(st, SelReduce{parts, n, rows, taps, n, a.dweight, a.channels, a.width, a.dbias, nullptr});
}

extern "C" int nhip_causal_conv_step(void* stream, const nhip_conv_step_args* args) {
    if (!args || !args->weight || args->channels <= 0 || args->width < 1 || args->width > kMaxWidth ||
        args->n < 0 || args->n_slots < 0)
        return NHIP_E_BADARG;
    const nhip_conv_step_args& a = *args;
    if (a.type < NHIP_F32 || a.type > NHIP_F16) return NHIP_E_BADARG;
    if (a.n == 0) return 0;
    if (!a.x || !a.y || (!a.state && a.width > 1)) return NHIP_E_BADARG;
    const bool w = wide(a.type, a.channels, {a.x, a.state, a.y}, {a.x_stride, a.state_stride});
    const long long lanes = (long long)a.n * (w ? a.channels / (16 / sel_size(a.type)) : a.channels);
    const long long groups = (lanes + NHIP_WG - 1) / NHIP_WG;
    if (groups > SEL_MAX_GROUPS) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        with_width(a.width, [&](auto k) {
            constexpr int K = decltype(k)::value, V = 16 / sizeof(T);
            hipStream_t st = static_cast<hipStream_t>(stream);
            const dim3 g((unsigned)groups);
            if (w) NHIP_LAUNCH((conv_step_kernel<T, V, K>), g, dim3(NHIP_WG), 0, st, a);
            else NHIP_LAUNCH((conv_step_kernel<T, 1, K>), g, dim3(NHIP_WG), 0, st, a);
            rc = (int)hipGetLastError();
        });
    });
    return rc;
}
