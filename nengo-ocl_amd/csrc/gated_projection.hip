// The gated projection of a feed-forward block, y = act(x gate') (x up'), and its gradient:
//
//     g = x gate',  u = x up',  y = act(g) u
//     dg = dy u act'(g),  du = dy act(g);   dx = dg gate + du up,   dgate = dg' x,   dup = du' x
//
// A wave's tile holds equal features of both weights, so that activation and product happen in its registers.  The
// backward pass forms g and u again and keeps dg and du, in the type of x, for the two products that read them.
#include <algorithm>
#include <optional>

#include "token_layout.h"

namespace {

constexpr long long kMostRows = 1 << 20, kMostChannels = 1 << 20, kMostFeatures = 1 << 20;

// act(g) and its derivative
__device__ __forceinline__ void activate(int kind, float g, float& f, float& slope) {
    if (kind == NHIP_ACT_SILU) {
        const float s = sel_sigmoid(g);
        f = g * s;
        slope = s * fmaf(g, 1.0f - s, 1.0f);
    } else {
        const float cdf = 0.5f * erfcf(g * -0.70710678118654752f);
        f = g * cdf;
        slope = fmaf(g * 0.39894228040143268f, sel_exp(-0.5f * g * g), cdf);
    }
}

struct Forward {
    void* y;
    long long features, f0, n_features;  // of a row; the piece's first, and how many it has
    int activation;
    template <class T, class S> __device__ __forceinline__ void run(const TokPlace& at, sel_f4 (&acc)[S::MI][S::NI]) const {
        constexpr int H = S::MI / 2;
        const bool wide = tok_fours(y, features, sizeof(T));
        const bool lines = features % 8 == 0 && ((uintptr_t)y & 15) == 0;
        static_assert(sizeof(T) == 4 || H % 4 || H == 4, "tok_put has four tiles");
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            const long long n = (long long)at.n_tile * S::BN + at.wave_n * S::kWaveN + 16 * j + at.l;
            auto value = [&](int i, float(&v)[4]) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float act, slope;
                    activate(activation, acc[i][j][r], act, slope);
                    v[r] = act * acc[i + H][j][r];
                }
            };
            if constexpr (sizeof(T) == 2 && H % 4 == 0) {
                if (lines) {
                    const long long c = ((long long)at.m_tile * S::BM + at.wave_m * S::kWaveM) / 2;
                    tok_put<T>(at, static_cast<T*>(y) + (n - at.l) * features + f0 + c, features,
                               (int)max(0LL, min(16LL, at.live - (n - at.l))), (int)max(0LL, min(64LL, n_features - c)), value);
                    continue;
                }
            }
            if (n >= at.live) continue;
            T* const to = static_cast<T*>(y) + n * features + f0;
#pragma unroll
            for (int i = 0; i < H; ++i) {
                const long long f = ((long long)at.m_tile * S::BM + at.wave_m * S::kWaveM) / 2 + 16 * i + 4 * at.g;
                float v[4];
                value(i, v);
                if (wide && f + 4 <= n_features) {
                    sel_store<T, 4>(to + f, v);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (f + r < n_features) to[f + r] = (T)v[r];
                }
            }
        }
    }
};

// dg and du of the tile, in both layouts: columns (rows) of du come `second` behind those of dg.  They are rounded to the
// type of x, the type in which the matrix cores multiply them with x and the weights: once, to half a step.  (A gradient in
// bfloat16 is off by 0.0023 of its norm, 0.0017 of it the rounding of the result; two parts to each of them would
// save that and double two of the three products.)
//
// Float16 holds less than their range: 2000 times an activation of 40 is beyond it.  A wave leaves the largest of its tile, and where
// the largest of all is beyond the type, or so small that what matters is among its subnormal numbers, the product is formed
// once more, and they are stored by a power of two that brings the largest to 2^14 ... 2^15 (Range).  Others are stored as they are:
// the launches that look for the largest and that then do nothing take 28 us of 1056 (8192 rows, 2048 channels, 5504 features;
// 6 of 63 with 700, 512, 1376), the product once more 370.  (A kernel of its own for each: one that does both spills ten registers.)
enum class Kept { plain, measured, scaled };
template <Kept KEPT> struct Backward {
    const void* dy;
    long long dy_ld, f0, n_features, second;
    void *g, *gt;
    long long g_ld, gt_ld;
    int activation;
    int m_tiles;
    float* most;         // measured: [tiles, waves], the largest finite magnitude
    const float* scale;  // scaled
    template <class T, class S> __device__ __forceinline__ void run(const TokPlace& at, sel_f4 (&acc)[S::MI][S::NI]) const {
        constexpr int H = S::MI / 2;
        float top = 0.0f;
        const float k = KEPT == Kept::scaled ? *scale : 1.0f;
        const bool wide = tok_fours(dy, dy_ld, sizeof(T));
        const long long c = ((long long)at.m_tile * S::BM + at.wave_m * S::kWaveM) / 2;  // of the piece's features
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            const long long n = (long long)at.n_tile * S::BN + at.wave_n * S::kWaveN + 16 * j + at.l;
            const bool counts = n < at.live;
            const T* const from = static_cast<const T*>(dy) + (counts ? n : 0) * dy_ld + f0;
            float d[H][4];
            if (wide && c + 16 * H <= n_features) {
#pragma unroll
                for (int i = 0; i < H; ++i) sel_load<T, 4>(from + c + 16 * i + 4 * at.g, d[i]);
            } else {
#pragma unroll
                for (int i = 0; i < H; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) d[i][r] = (float)from[min(c + 16 * i + 4 * at.g + r, n_features - 1)];
            }
            // g and u become dg and du in their places
#pragma unroll
            for (int i = 0; i < H; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float act, slope;
                    activate(activation, acc[i][j][r], act, slope);
                    const bool is = counts && c + 16 * i + 4 * at.g + r < n_features;
                    acc[i][j][r] = is ? d[i][r] * acc[i + H][j][r] * slope : 0.0f;
                    acc[i + H][j][r] = is ? d[i][r] * act : 0.0f;
                }
            if constexpr (KEPT != Kept::plain) {
#pragma unroll
                for (int i = 0; i < S::MI; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = acc[i][j][r];
                        if (KEPT == Kept::measured) top = fabsf(v) < INFINITY ? fmaxf(top, fabsf(v)) : top;
                        else acc[i][j][r] = v * k;
                    }
                asm volatile("" : "+v"(top));  // (a column at a time: with all of them at once registers are spilled)
            }
            if constexpr (sizeof(T) == 2 && H % 4 == 0) {
                if (!gt) {
#pragma unroll
                    for (int which = 0; which < 2; ++which)
                        tok_put<T>(at, static_cast<T*>(g) + (n - at.l) * g_ld + which * second + c, g_ld, 16, 64,
                                   [&](int i, float(&v)[4]) {
#pragma unroll
                                       for (int r = 0; r < 4; ++r) v[r] = acc[i + which * H][j][r];
                                   });
                    continue;
                }
            }
#pragma unroll
            for (int i = 0; i < S::MI; ++i) {
                const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                tok_store_both<T>(static_cast<T*>(g), g_ld, static_cast<T*>(gt), gt_ld, n,
                                  (i < H ? 0 : second) + c + 16 * (i % H) + 4 * at.g, v);
            }
        }
        if constexpr (KEPT == Kept::measured) {
#pragma unroll
            for (int e = 1; e < NHIP_WAVE; e *= 2) top = fmaxf(top, __shfl_xor(top, e));
            if (at.l + at.g == 0) most[((long long)at.n_tile * m_tiles + at.m_tile) * S::kWaves + at.wave_n * S::WM + at.wave_m] = top;
        }
    }
};

// Float16: from the tiles' largest magnitudes what dg and du are scaled by (and the reverse), and the rows that are formed once
// more: none where the type holds the largest, and nothing above 2^-6 of it is subnormal (elements of a normal distribution's
// product, a thirtieth of the largest, are rounded to as much as their results are).
struct Range {
    const float* most;
    long long n;
    int rows;
    float* scale;  // [2]
    int* live;
};
constexpr float kLeastRange = 0x1p-8f, kMostRange = 65504.0f;

__global__ __launch_bounds__(1024) void range_kernel(Range a) {
    __shared__ float s[16];
    float top = 0.0f;
    for (long long i = threadIdx.x; i < a.n; i += 1024) top = fmaxf(top, a.most[i]);
#pragma unroll
    for (int d = 1; d < NHIP_WAVE; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    if (threadIdx.x % NHIP_WAVE == 0) s[threadIdx.x / NHIP_WAVE] = top;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 16; ++w) top = fmaxf(top, s[w]);
    const bool fits = top == 0.0f || (top >= kLeastRange && top <= kMostRange);
    const int e = fits ? 0 : 14 - max(ilogbf(top), -100);
    a.scale[0] = ldexpf(1.0f, e);
    a.scale[1] = ldexpf(1.0f, -e);
    *a.live = fits ? 0 : a.rows;
}

int check(const nhip_gated_args* a) {
    if (!a || a->channels <= 0 || a->features <= 0 || a->rows < 0) return NHIP_E_BADARG;
    if (a->type < NHIP_F32 || a->type > NHIP_F16) return NHIP_E_BADARG;
    if (a->activation != NHIP_ACT_SILU && a->activation != NHIP_ACT_GELU) return NHIP_E_BADARG;
    if (a->rows > kMostRows || a->channels > kMostChannels || a->features > kMostFeatures) return NHIP_E_BADARG;
    return 0;
}

struct Space : TokSpace {
    long long x_ld, piece;
    long long x = 0, gate = 0, up = 0, most = 0, scale = 0;
    bool pad_x, pad_w;
    std::optional<TokGradient> gradient;
    Space(const nhip_gated_args& a, bool grad) {
        const long long size = sel_size(a.type), d = a.channels, rows = a.rows > 0 ? a.rows : 1;
        x_ld = tok_round(d, 64);
        if (grad) {
            gradient.emplace(*this, a.rows, d, 2 * tok_round(a.features, 128), size);
            piece = gradient->piece / 2;
            if (a.type == NHIP_F16 && a.rows) {
                const long long last = a.features % piece;  // (of the last piece, whose shape may be another one)
                most = take(std::max(waves(a, std::min<long long>(a.features, piece)), last ? waves(a, last) : 0) * 4);
                scale = take(256);
            }
        } else {
            // as many features as a launch's tiles reach
            piece = std::min(tok_round(a.features, 128), (1LL << 21) / (tok_round(rows, 256) / 256) * 64);
        }
        pad_x = !tok_rows_wide(a.x, a.x_stride * size, d * size);
        pad_w = !tok_rows_wide(a.gate, a.gate_stride * size, d * size) || !tok_rows_wide(a.up, a.up_stride * size, d * size) ||
                a.gate_stride != a.up_stride;
        if (pad_x) x = take(rows * x_ld * size);
        if (pad_w) {
            gate = take(piece * x_ld * size);
            up = take(piece * x_ld * size);
        }
    }
    // of all tiles that form dg and du for n features
    static long long waves(const nhip_gated_args& a, long long n) {
        return tok_with_shape(2 * n, a.rows, sel_size(a.type), 1, [&](auto shape) {
            using S = decltype(shape);
            return (2 * n + S::BM - 1) / S::BM * ((a.rows + S::BN - 1) / S::BN) * S::kWaves;
        });
    }
};

#define TOK_TRY(call) do { if (int e_ = (call)) return e_; } while (0)

// x as the products read it
template <class T> int x_rows(hipStream_t st, const nhip_gated_args& a, const Space& s, char* w, TokRows& rows) {
    rows = TokRows{static_cast<const char*>(a.x), nullptr, a.x_stride * (long long)sizeof(T), a.rows};
    if (s.pad_x) {
        TOK_TRY(tok_pad<T>(st, TokPad{a.x, a.x_stride, w + s.x, s.x_ld, a.rows, a.channels}));
        rows.p = w + s.x;
        rows.ld = s.x_ld * (long long)sizeof(T);
    }
    return 0;
}

// n features from f0 on, of both weights
template <class T>
int weight_rows(hipStream_t st, const nhip_gated_args& a, const Space& s, char* w, long long f0, long long n, TokRows& rows) {
    const T* const gate = static_cast<const T*>(a.gate) + f0 * a.gate_stride;
    const T* const up = static_cast<const T*>(a.up) + f0 * a.up_stride;
    rows = TokRows{reinterpret_cast<const char*>(gate), reinterpret_cast<const char*>(up), a.gate_stride * (long long)sizeof(T), n};
    if (s.pad_w) {
        TOK_TRY(tok_pad<T>(st, TokPad{gate, a.gate_stride, w + s.gate, s.x_ld, n, a.channels}));
        TOK_TRY(tok_pad<T>(st, TokPad{up, a.up_stride, w + s.up, s.x_ld, n, a.channels}));
        rows.p = w + s.gate;
        rows.p2 = w + s.up;
        rows.ld = s.x_ld * (long long)sizeof(T);
    }
    return 0;
}

template <class T> int forward(hipStream_t st, const nhip_gated_args& a, const Space& s) {
    char* const w = static_cast<char*>(a.workspace);
    if (!a.rows) return 0;
    TokRows x, rows;
    TOK_TRY(x_rows<T>(st, a, s, w, x));
    for (long long f0 = 0; f0 < a.features; f0 += s.piece) {
        const long long n = a.features - f0 < s.piece ? a.features - f0 : s.piece;
        TOK_TRY(weight_rows<T>(st, a, s, w, f0, n, rows));
        TokProduct p{rows, x, nullptr, nullptr, a.channels * (long long)sizeof(T), 0, 0, 1};
        p.last = f0 + n == a.features;
        const Forward e{a.y, a.features, f0, n, a.activation};
        if (a.rows <= TOK_FEW) {
            TOK_TRY((tok_few<T, 2, 1>(st, p, e)));
            continue;
        }
        TOK_TRY(tok_with_many(2 * n, a.rows, sizeof(T), 1, [&](auto shape) {
            using S = decltype(shape);
            p.m_tiles = (int)((2 * n + S::BM - 1) / S::BM);
            p.n_tiles = (int)((a.rows + S::BN - 1) / S::BN);
            return tok_product<T, S, S::kWaveM / 2>(st, p, e);
        }));
    }
    return 0;
}

template <class T> int backward(hipStream_t st, const nhip_gated_args& a, const Space& s) {
    constexpr long long size = sizeof(T);
    char* const w = static_cast<char*>(a.workspace);
    const long long d = a.channels;
    TokRows x, rows;
    TOK_TRY(x_rows<T>(st, a, s, w, x));
    const TokGradient& gr = *s.gradient;
    TOK_TRY(gr.lay_out_x<T>(st, w, a.x, a.x_stride, nullptr));
    for (long long f0 = 0; f0 < a.features; f0 += s.piece) {
        const long long n = a.features - f0 < s.piece ? a.features - f0 : s.piece;
        // the second weights' part begins behind the last tile of the first one's, whose zeros lie between
        const long long second = tok_round(n, tok_with_shape(2 * n, a.rows, sizeof(T), 1, [](auto shape) { return decltype(shape)::BM / 2; }));
        const long long both = second + tok_round(n, 64);
        TOK_TRY(weight_rows<T>(st, a, s, w, f0, n, rows));
        constexpr bool kRange = std::is_same<T, _Float16>::value;
        float* const most = reinterpret_cast<float*>(w + s.most);
        float* const scale = reinterpret_cast<float*>(w + s.scale);
        int* const live = reinterpret_cast<int*>(scale + 2);
        auto form = [&](auto kept) {
            return tok_with_shape(2 * n, a.rows, sizeof(T), 1, [&](auto shape) {
                using S = decltype(shape);
                constexpr Kept k = decltype(kept)::value;
                TokProduct p{rows, x, k == Kept::scaled ? live : nullptr, nullptr, d * size, (int)((2 * n + S::BM - 1) / S::BM),
                             (int)((a.rows + S::BN - 1) / S::BN), 1};
                return tok_product<T, S, S::kWaveM / 2>(st, p, Backward<k>{a.dy, a.dy_stride, f0, n, second, w + gr.g, gr.gt_of<T>(w),
                                                                           gr.g_ld, gr.gt_ld, a.activation, p.m_tiles, most, scale});
            });
        };
        if (a.rows) {
            TOK_TRY(form(std::integral_constant<Kept, kRange ? Kept::measured : Kept::plain>()));
            if constexpr (kRange) {
                const Range r{most, Space::waves(a, n), (int)a.rows, scale, live};
                TOK_LAUNCH(false, range_kernel, dim3(1), dim3(1024), 0, st, r);
                NHIP_LAUNCH_CHECK();
                TOK_TRY(form(std::integral_constant<Kept, Kept::scaled>()));
            }
        }
        const float* const back = kRange && a.rows ? scale + 1 : nullptr;
        TOK_TRY(gr.weights<T>(st, w, x, nullptr, second + n, n, second, static_cast<T*>(a.dgate) + f0 * d,
                              static_cast<T*>(a.dup) + f0 * d, back));
        if (a.rows) TOK_TRY((gr.inputs<T, kRange>(st, w, rows, nullptr, both, n, second, f0 > 0, back)));
    }
    return gr.finish<T>(st, w, nullptr, nullptr, nullptr, a.dx);
}

int run(void* stream, const nhip_gated_args* args, bool grad) {
    if (int e = check(args)) return e;
    const nhip_gated_args& a = *args;
    if (!a.gate || !a.up || (a.rows && !a.x)) return NHIP_E_BADARG;
    if (grad ? !a.dgate || !a.dup || (a.rows && (!a.dy || !a.dx)) : a.rows && !a.y) return NHIP_E_BADARG;
    const Space s(a, grad);
    if (s.bytes > a.workspace_bytes) return NHIP_E_TOOBIG;
    if (s.bytes && (!a.workspace || !sel_aligned(a.workspace, 256))) return NHIP_E_BADARG;
    int rc = NHIP_E_BADARG;
    sel_with_type(a.type, [&](auto t) {
        using T = decltype(t);
        rc = grad ? backward<T>(static_cast<hipStream_t>(stream), a, s) : forward<T>(static_cast<hipStream_t>(stream), a, s);
    });
    return tok_end(static_cast<hipStream_t>(stream), rc);
}

}  // namespace

extern "C" int nhip_gated_projection_workspace(const nhip_gated_args* args, long long* bytes_out) {
    if (int e = check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    *bytes_out = Space(*args, false).bytes;
    return 0;
}

extern "C" int nhip_gated_projection(void* stream, const nhip_gated_args* args) { return run(stream, args, false); }

extern "C" int nhip_gated_projection_grad_workspace(const nhip_gated_args* args, long long* bytes_out) {
    if (int e = check(args)) return e;
    if (!bytes_out) return NHIP_E_BADARG;
    *bytes_out = Space(*args, true).bytes;
    return 0;
}

extern "C" int nhip_gated_projection_grad(void* stream, const nhip_gated_args* args) { return run(stream, args, true); }
