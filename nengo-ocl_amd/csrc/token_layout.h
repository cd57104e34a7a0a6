// Layouts that the products of token_products.h read: rows without the tokens that do not count, rows of whole stages,
// transposed matrices; and the sum of the parts of a product's result.
#pragma once

#include "token_products.h"

static inline long long tok_round(long long v, long long to) { return (v + to - 1) / to * to; }
// Elements of a row in the workspace: rows whose distance is a power of two meet in few channels of the memory
static inline long long tok_ld(long long v) { return tok_round(v, 64) + 64; }

// Whether rows may be read 16 bytes at a time
static inline bool tok_rows_wide(const void* p, long long ld_bytes, long long row_bytes) {
    return sel_aligned(p, 16) && ld_bytes % 16 == 0 && row_bytes % 16 == 0 && ld_bytes <= TOK_MOST_LD;
}

// Whether rows of elements of `size` bytes may be read and written four at a time, from columns that are multiples of four
static __host__ __device__ __forceinline__ bool tok_fours(const void* p, long long ld, int size) {
    return ld % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(4 * size - 1)) == 0;
}

// Offsets of a workspace
struct TokSpace {
    long long bytes = 0;
    long long take(long long n) {
        const long long at = bytes;
        bytes += tok_round(n, 256);
        return at;
    }
};

// ------------------------------------------------------------------------------------ transposed
// out[c, r] = in[r, c] for r < rows (or *live of them) and c < cols; zeros for rows up to out_rows (a multiple of 64).
struct TokTranspose {
    const void* in;
    long long ld;
    void* out;
    long long out_ld;
    long long rows, cols, out_rows;
    const int* live;
    int wide;
};

template <class T> __global__ __launch_bounds__(NHIP_WG) void tok_transpose_kernel(TokTranspose a) {
    constexpr int V = 16 / (int)sizeof(T), kPacks = 64 / V;
    __shared__ T s[64][64 + 2];
    const long long r0 = (long long)blockIdx.x * 64, c0 = (long long)blockIdx.y * 64;
    const long long rows = a.live ? min((long long)*a.live, a.rows) : a.rows;
    const T* const in = static_cast<const T*>(a.in);
    for (int q = threadIdx.x; q < 64 * kPacks; q += NHIP_WG) {
        const int r = q / kPacks, c = q % kPacks * V;
        SelPack<T, V> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.v[e] = (T)0.0f;
        if (r0 + r < rows) {
            const T* const from = in + (r0 + r) * a.ld + c0 + c;
            if (a.wide && c0 + c + V <= a.cols) {
                v = *reinterpret_cast<const SelPack<T, V>*>(from);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (c0 + c + e < a.cols) v.v[e] = from[e];
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) s[c + e][r] = v.v[e];
    }
    __syncthreads();
    T* const out = static_cast<T*>(a.out);
    for (int q = threadIdx.x; q < 64 * kPacks; q += NHIP_WG) {
        const int c = q / kPacks, r = q % kPacks * V;
        if (c0 + c >= a.cols) continue;
        SelPack<T, V> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.v[e] = s[c][r + e];
        *reinterpret_cast<SelPack<T, V>*>(out + (c0 + c) * a.out_ld + r0 + r) = v;
    }
}

template <class T> static inline int tok_transpose(hipStream_t stream, TokTranspose a) {
    if (a.cols <= 0 || a.out_rows <= 0) return 0;
    const long long x = a.out_rows / 64, y = (a.cols + 63) / 64;
    if (x > 0xffffff || y > SEL_MAX_GRID_Y) return NHIP_E_BADARG;
    a.wide = tok_rows_wide(a.in, a.ld * (long long)sizeof(T), 16);
    TOK_LAUNCH(false, (tok_transpose_kernel<T>), dim3((unsigned)x, (unsigned)y), dim3(NHIP_WG), 0, stream, a);
    NHIP_LAUNCH_CHECK();
    return 0;
}

// ------------------------------------------------------------------------------- rows of whole stages
// out[r, c] = in[r, c], zeros for c up to out_ld (a multiple of 64)
struct TokPad {
    const void* in;
    long long ld;
    void* out;
    long long out_ld, rows, cols;
};

template <class T> __global__ __launch_bounds__(NHIP_WG) void tok_pad_kernel(TokPad a) {
    constexpr int V = 16 / (int)sizeof(T);
    const long long packs = a.out_ld / V, all = a.rows * packs;
    for (long long q = (long long)blockIdx.x * NHIP_WG + threadIdx.x; q < all; q += (long long)gridDim.x * NHIP_WG) {
        const long long r = q / packs, c = q % packs * V;
        const T* const from = static_cast<const T*>(a.in) + r * a.ld + c;
        SelPack<T, V> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.v[e] = c + e < a.cols ? from[e] : (T)0.0f;
        *reinterpret_cast<SelPack<T, V>*>(static_cast<T*>(a.out) + r * a.out_ld + c) = v;
    }
}

template <class T> static inline int tok_pad(hipStream_t stream, const TokPad& a) {
    if (a.rows <= 0) return 0;
    const long long groups = (a.rows * (a.out_ld * (long long)sizeof(T) / 16) + NHIP_WG - 1) / NHIP_WG;
    TOK_LAUNCH(false, (tok_pad_kernel<T>), dim3((unsigned)(groups < 16384 ? groups : 16384)), dim3(NHIP_WG), 0, stream, a);
    NHIP_LAUNCH_CHECK();
    return 0;
}

// --------------------------------------------------------------------------- gradients of x and of the weights
// dW[w, d] = sum_n G[n, w] x[n, d] for the rows w of a piece of the weights: rows below `first` of them go to out, those from
// `second` on (the other weights of a gated projection) to out2.
struct TokStoreRows {
    void *out, *out2;
    long long ld, rows, second;  // ld: elements of a row of the result, its channels; rows: of each
    const float* scale;          // 1 / that of G, or NULL
    template <class T, class S> __device__ __forceinline__ void run(const TokPlace& at, sel_f4 (&acc)[S::MI][S::NI]) const {
        const float k = scale ? *scale : 1.0f;
        const bool lines = ld % 8 == 0 && (((uintptr_t)out | (uintptr_t)out2) & 15) == 0;
        const bool wide = tok_fours(out, ld, sizeof(T)) && (!out2 || tok_fours(out2, ld, sizeof(T)));
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            long long w = (long long)at.n_tile * S::BN + at.wave_n * S::kWaveN + 16 * j + at.l;
            T* to = static_cast<T*>(out);
            if (second && w >= second) {
                w -= second;
                to = static_cast<T*>(out2);
            }
            if constexpr (sizeof(T) == 2 && S::MI % 4 == 0) {
                if (lines) {  // (all lanes' columns are of the same matrix: `second` is a multiple of 16)
                    const long long w0 = w - at.l, d0 = (long long)at.m_tile * S::BM + at.wave_m * S::kWaveM;
                    const int some = (int)max(0LL, min(16LL, rows - w0));
#pragma unroll
                    for (int i = 0; i < S::MI; i += 4)
                        tok_put<T>(at, to + w0 * ld + d0 + 16 * i, ld, some, (int)max(0LL, min(64LL, ld - d0 - 16 * i)),
                                   [&](int e, float(&v)[4]) {
#pragma unroll
                                       for (int r = 0; r < 4; ++r) v[r] = acc[i + e][j][r] * k;
                                   });
                    continue;
                }
            }
            if (w >= rows) continue;
            to += w * ld;
#pragma unroll
            for (int i = 0; i < S::MI; ++i) {
                const long long d = (long long)at.m_tile * S::BM + at.wave_m * S::kWaveM + 16 * i + 4 * at.g;
                const float v[4] = {acc[i][j][0] * k, acc[i][j][1] * k, acc[i][j][2] * k, acc[i][j][3] * k};
                if (wide && d + 4 <= ld) {
                    sel_store<T, 4>(to + d, v);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (d + r < ld) to[d + r] = (T)v[r];
                }
            }
            asm volatile("" ::: "memory");
        }
    }
};

// dx[n, d] = sum_w G[n, w] W[w, d], added up over pieces of the weights in 32 bits, in parts (splits of k)
// (SCALED: pieces of G have a scale each.  A kernel of its own: the others take 3 % more of a gradient's time with it.)
template <bool SCALED> struct TokAddParts {
    float* parts;
    long long ld, part;  // elements of a row, of a part
    int add;
    const float* scale;  // 1 / that of G
    template <class T, class S> __device__ __forceinline__ void run(const TokPlace& at, sel_f4 (&acc)[S::MI][S::NI]) const {
        const float k = SCALED ? *scale : 1.0f;
        float* const mine = parts + at.split * part;
#pragma unroll
        for (int j = 0; j < S::NI; ++j) {
            const long long n = (long long)at.n_tile * S::BN + at.wave_n * S::kWaveN + 16 * j + at.l;
            if (n >= at.live) continue;
#pragma unroll
            for (int i = 0; i < S::MI; ++i) {
                const long long d = (long long)at.m_tile * S::BM + at.wave_m * S::kWaveM + 16 * i + 4 * at.g;
                sel_f4* const to = reinterpret_cast<sel_f4*>(mine + n * ld + d);
                const sel_f4 v = SCALED ? acc[i][j] * k : acc[i][j];
                *to = add ? *to + v : v;
            }
            asm volatile("" ::: "memory");  // (a column's sums at a time: all of them at once are more than the registers hold)
        }
    }
};

// dx[r] = the sum of the parts of row where[r] (zeros where it is below zero; NULL: r)
struct TokJoin {
    const float* parts;
    long long ld, part;
    int n_parts;
    const int* where;
    const float* scale;
    void* out;
    long long rows, cols;
    const int* live = nullptr;  // not NULL: as many parts as the product had by its tiles of live rows (tok_parts), n_parts at most
    int slots = 0, m_tiles = 0, bn = 1;
    bool last = false;  // the entry point's last launch
};

template <class T, int V> __global__ __launch_bounds__(NHIP_WG) void tok_join_kernel(TokJoin a) {
    const float k = a.scale ? *a.scale : 1.0f;
    const int n_parts = a.live ? tok_parts(a.slots, a.m_tiles * ((*a.live + a.bn - 1) / a.bn), a.n_parts) : a.n_parts;
    const long long packs = (a.cols + V - 1) / V, all = a.rows * packs;
    for (long long q = (long long)blockIdx.x * NHIP_WG + threadIdx.x; q < all; q += (long long)gridDim.x * NHIP_WG) {
        const long long r = q / packs, c = q % packs * V, from = a.where ? a.where[r] : r;
        float v[V], sum[V];
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] = 0.0f;
        if (from >= 0) {
            const float* p = a.parts + from * a.ld + c;
            for (int s = 0; s < n_parts; ++s) {
                sel_load<float, V>(p + s * a.part, v);
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] += v[e];
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] *= k;
        sel_store<T, V>(static_cast<T*>(a.out) + r * a.cols + c, sum);
    }
}

template <class T> static inline int tok_join(hipStream_t stream, const TokJoin& a) {
    if (a.rows <= 0) return 0;
    const int v = tok_fours(a.out, a.cols, sizeof(T)) ? 4 : 1;
    const long long groups = (a.rows * (a.cols / v) + NHIP_WG - 1) / NHIP_WG;
    const dim3 grid((unsigned)(groups < 16384 ? groups : 16384));
    if (v == 4) TOK_LAUNCH(a.last, (tok_join_kernel<T, 4>), grid, dim3(NHIP_WG), 0, stream, a);
    else TOK_LAUNCH(a.last, (tok_join_kernel<T, 1>), grid, dim3(NHIP_WG), 0, stream, a);
    NHIP_LAUNCH_CHECK();
    return 0;
}

// The two products behind G: dW = G' x and dx = G W, for the rows of a piece of W.  16-bit elements in large tiles are read as
// they lie, G and x by columns for dW, W for dx; others go through transposed copies, which for small products cost less than
// they are.  (8192 tokens, 65536 words, 2048 channels: the copies took 7 % of the gradient's time.)
struct TokGradient {
    long long rows, d, size;
    long long padded, piece, g_ld, gt_ld, dx_ld;
    long long g = 0, gt = 0, xt = 0, wt = 0, dx = 0, dw = 0, dw_parts;  // in the workspace
    int dx_splits, dx_most, dw_splits;
    bool across;

    // tiles of 256 from which on operands are read as they lie: fewer do not go round.  (700 tokens, 6400 words, 1024 channels: 85 us,
    // through copies by small tiles 90; 300 tokens, 9001 words, 520 channels, 102 tiles: 73 and 69.)
    static constexpr int kLeastAcross = 96;

    // `weights`: rows of W (of both, whole tiles of each); they are gone through in equal pieces whose G takes 512 MB at most
    TokGradient(TokSpace& space, long long rows_, long long d_, long long weights, long long size_)
        : rows(rows_), d(d_), size(size_) {
        padded = tok_round(rows > 0 ? rows : 1, TOK_MOST_TILE);
        long long most = (512LL << 20) / (padded * size) / 256 * 256;
        most = most < 256 ? 256 : most;
        const long long pieces = (weights + most - 1) / most;
        piece = tok_round((weights + pieces - 1) / pieces, 256);
        g_ld = tok_ld(piece);
        gt_ld = tok_ld(padded);
        dx_ld = tok_round(d, TOK_MOST_TILE);
        const long long dw_bytes = piece * dx_ld * 4, dx_bytes = padded * dx_ld * 4, room = 256LL << 20;
        // (rows that do not count leave work-groups to the others' parts: room for more parts than all rows need)
        dx_splits = tok_splits(d, rows, (int)size, piece * size);
        dx_most = (int)tok_most_splits(piece * size);
        dw_splits = tok_splits(d, piece, (int)size, rows * size);
        if (dx_most > 1 && dx_most * dx_bytes > room) dx_most = room / dx_bytes > 1 ? (int)(room / dx_bytes) : 1;
        if (dx_splits > dx_most) dx_splits = dx_most;
        if (dw_splits > 1 && dw_splits * dw_bytes > room) dw_splits = room / dw_bytes > 1 ? (int)(room / dw_bytes) : 1;
        across = size == 2 && tok_is_large(d, rows, 2, dx_splits, kLeastAcross) && tok_is_large(d, piece, 2, dw_splits, kLeastAcross);
        g = space.take(padded * g_ld * size);
        if (!across) {
            gt = space.take(piece * gt_ld * size);
            xt = space.take(d * gt_ld * size);
            wt = space.take(d * g_ld * size);
        }
        dx = space.take(dx_most * dx_bytes);
        dw_parts = dw_splits > 1 ? dw_splits * dw_bytes : 0;
        long long n0;
        if (const int s = tail(weights < piece ? tok_round(weights, 64) : piece, n0, room)) dw_parts = s * tok_round(piece - n0, 256) * dx_ld * 4;
        if (dw_parts) dw = space.take(dw_parts);
    }

    // Tiles go round 256 compute units whole times and then some: the last columns of G, from n0 on, whose tiles are the rest of the
    // last round, are cut along k into parts that fill it.  0 where that gives nothing: no whole round, or a rest that fills it, or
    // too short a k for what the parts' sums take.  (8192 tokens, 2 x 5504 features, 2048 channels, 344 tiles: 405 us; 256, and 88 in
    // two parts, 330.)
    int tail(long long n, long long& n0, long long room) const {
        if (!across || dw_splits > 1) return 0;
        const long long m_tiles = (d + 255) / 256, n_tiles = (n + 255) / 256, whole = m_tiles * n_tiles / 256 * 256 / m_tiles;
        const long long rest = m_tiles * (n_tiles - whole), parts = rest > 0 ? (256 / rest < 8 ? 256 / rest : 8) : 0;
        n0 = whole * 256;
        if (whole < 1 || parts < 2 || rows * size / TOK_KB < 48 || parts * tok_round(n - n0, 256) * dx_ld * 4 > room) return 0;
        return (int)parts;
    }
    template <class T> T* gt_of(char* w) const { return across ? nullptr : reinterpret_cast<T*>(w + gt); }

    // x (its rows that count) by channels, once for all pieces
    template <class T> int lay_out_x(hipStream_t st, char* w, const void* x, long long ld, const int* live) const {
        return across ? 0 : tok_transpose<T>(st, TokTranspose{x, ld, w + xt, gt_ld, rows, d, padded, live, 0});
    }

    // dW: `n` rows of G's columns, of which those below `first` go to out and `first` from `second` on to out2 (if there is one)
    template <class T>
    int weights(hipStream_t st, char* w, const TokRows& x, const int* live, long long n, long long first, long long second,
                T* out, T* out2, const float* scale) const {
        TokRows a{w + xt, nullptr, gt_ld * size, d};
        if (across) {
            a = x;
            a.across = tok_round(d * size, 16);
        }
        // columns from ... to - 1 of G
        auto go = [&](long long from, long long to, int splits, const auto& epilogue) {
            TokRows b{w + gt + from * gt_ld * size, nullptr, gt_ld * size, to - from};
            if (across) {
                b = TokRows{w + g + from * size, nullptr, g_ld * size, to - from};
                b.across = (g_ld - from) * size;
            }
            // (large in every piece if in a whole one: G's layout goes by that)
            auto run = [&](auto shape) {
                using S = decltype(shape);
                constexpr int kAcross = std::is_same<S, TokLarge>::value && sizeof(T) == 2 ? 3 : 0;
                TokProduct p{a, b, nullptr, live, rows * size, (int)((d + S::BM - 1) / S::BM),
                             (int)((to - from + S::BN - 1) / S::BN), splits};
                if (kAcross && !across) return tok_product<T, S, 0>(st, p, epilogue);
                return tok_product<T, S, 0, kAcross>(st, p, epilogue);
            };
            return across ? run(TokLarge()) : tok_with_shape(d, to - from, (int)size, splits, run);
        };
        const TokStoreRows store{out, out2, d, first, out2 ? second : 0, scale};
        long long n0 = 0;
        int splits = dw_splits;
        if (splits == 1) {
            splits = tail(n, n0, dw_parts);
            if (!splits) return go(0, n, 1, store);
            if (int e = go(0, n0, 1, store)) return e;
        }
        float* const parts = reinterpret_cast<float*>(w + dw);
        const long long part = tok_round(n - n0, 256) * dx_ld;
        if (int e = go(n0, n, splits, TokAddParts<false>{parts, dx_ld, part, 0, nullptr})) return e;
        // the sums of columns from ... to - 1, which are rows of `to_rows` from its first on
        auto join = [&](long long from, long long to, long long base, T* to_rows) {
            from = from > n0 ? from : n0;
            if (from >= to) return 0;
            return tok_join<T>(st, TokJoin{parts + (from - n0) * dx_ld, dx_ld, part, splits, nullptr, scale,
                                           to_rows + (from - base) * d, to - from, d});
        };
        if (int e = join(0, first, 0, out)) return e;
        return out2 ? join(second, second + first, second, out2) : 0;
    }

    // dx += G W over `k` columns of G; W's rows (p2: from `second` on, `first` of each matrix) lie at the places that `rows_of` has
    template <class T, bool SCALED = false>
    int inputs(hipStream_t st, char* w, const TokRows& rows_of, const int* live, long long k, long long first, long long second,
               bool add, const float* scale = nullptr) const {
        TokRows a{w + wt, nullptr, g_ld * size, d};
        if (across) {
            a = rows_of;
            a.across = tok_round(d * size, 16);
            a.second = second;
            a.k_rows = first;
        } else {
            for (int part = 0; part < (rows_of.p2 ? 2 : 1); ++part)
                if (int e = tok_transpose<T>(st, TokTranspose{part ? rows_of.p2 : rows_of.p, rows_of.ld / size,
                                                              reinterpret_cast<T*>(w + wt) + part * second, g_ld, first, d,
                                                              rows_of.p2 && !part ? second : tok_round(first, 64), nullptr, 0}))
                    return e;
        }
        const TokRows b{w + g, nullptr, g_ld * size, rows};
        const TokAddParts<SCALED> epilogue{reinterpret_cast<float*>(w + dx), dx_ld, padded * dx_ld, add, scale};
        auto run = [&](auto shape) {
            using S = decltype(shape);
            constexpr int kAcross = std::is_same<S, TokLarge>::value && sizeof(T) == 2 ? 1 : 0;
            TokProduct p{a, b, live, nullptr, k * size, (int)((d + S::BM - 1) / S::BM), (int)((rows + S::BN - 1) / S::BN),
                         live ? dx_most : dx_splits, false, live ? 256 * S::kAtOnce : 0};
            if (kAcross && !across) return tok_product<T, S, 0>(st, p, epilogue);
            return tok_product<T, S, 0, kAcross>(st, p, epilogue);
        };
        return across ? run(TokLarge()) : tok_with_shape(d, rows, (int)size, dx_splits, run);
    }

    template <class T> int finish(hipStream_t st, char* w, const int* where, const int* live, const float* scale, void* out) const {
        TokJoin join{reinterpret_cast<float*>(w + dx), dx_ld, padded * dx_ld, live ? dx_most : dx_splits, where, scale, out, rows, d};
        auto shape_of = [&](auto shape) {
            using S = decltype(shape);
            join.live = live;
            join.slots = 256 * S::kAtOnce;
            join.m_tiles = (int)((d + S::BM - 1) / S::BM);
            join.bn = S::BN;
            return 0;
        };
        if (live) across ? shape_of(TokLarge()) : tok_with_shape(d, rows, (int)size, dx_splits, shape_of);
        join.last = true;
        return tok_join<T>(st, join);
    }
};
