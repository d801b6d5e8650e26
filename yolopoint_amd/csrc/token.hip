// Operators on tokens (rows of features: keypoint descriptors, descriptor-map cells, sequence entries): layer norm with its backward pass, the
// fused dropout + residual + layer norm, dropout from a counter-based generator, rotary positions.  All of them are bound by HBM: each reads
// its inputs once, keeps a row in registers, and writes its outputs once; sums, statistics and angles are held in 32 bits or more.
// Compiled with -ffp-contract=off: every fused multiply-add is written as one, so that the kernels for different operands and row shapes round alike
// (the fused operator's norm is the plain norm of its sum bit for bit).
#include "yp_internal.h"

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

template <int DT> struct Sc;
template <> struct Sc<YP_F16> { using t = _Float16; };
template <> struct Sc<YP_BF16> { using t = __bf16; };
template <> struct Sc<YP_F32> { using t = float; };

// ------------------------------------------------------------------------------------------------------------------ memory
// 16 bytes of a row.  Rows may start on any element (odd widths, slices of wider rows): the target's global loads and stores take any alignment,
// so there is no separate path for unaligned rows.
template <typename T> struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
    T e[N];
};

// How the end of a row of D elements is read (a template parameter: as run-time branches around the loads these cost a wait after each of them).
// No load leaves its row, none stands behind a branch: threads behind the end read the row's last 16 bytes and drop them.
enum Tail { WHOLE,      // D % N == 0
            CUT,        // D > N: the last chunk is read from the 16 bytes that end with the row and moved to its place
            SHORT };    // D < N: element by element

// elements c .. c + N - 1 of a row of D elements, zeros behind its end
template <typename T, Tail TAIL> __device__ __forceinline__ Vec<T> load_vec(const T* row, int c, int D) {
    constexpr int N = Vec<T>::N;
    Vec<T> v;
    if constexpr (TAIL == SHORT) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const T e = row[min(c + j, D - 1)];
            v.e[j] = c + j < D ? e : (T)0.f;
        }
    } else {
        const int at = min(c, D - N);
        u32x4 r;
        __builtin_memcpy(&r, row + at, 16);
        const unsigned back = (unsigned)(c - at) * sizeof(T);        // bytes to move down
        if constexpr (TAIL == CUT) {
            if (back & 8) { r.x = r.z; r.y = r.w; r.z = r.w = 0u; }
            if (back & 4) { r.x = r.y; r.y = r.z; r.z = r.w; r.w = 0u; }
            if constexpr (sizeof(T) == 2) {
                if (back & 2) {
                    r.x = __builtin_amdgcn_alignbit(r.y, r.x, 16); r.y = __builtin_amdgcn_alignbit(r.z, r.y, 16); r.z = __builtin_amdgcn_alignbit(r.w, r.z, 16); r.w >>= 16;
                }
            }
        }
        if (back >= 16) r = u32x4{0u, 0u, 0u, 0u};
        __builtin_memcpy(&v, &r, 16);
    }
    return v;
}

template <typename T> __device__ __forceinline__ void store_vec(T* p, const Vec<T>& v, int n) {
    if (n == Vec<T>::N) {
        __builtin_memcpy(p, &v, 16);
    } else if (n) {
#pragma unroll
        for (int j = 0; j < Vec<T>::N; ++j)
            if (j < n) p[j] = v.e[j];
    }
}

// the compiler may not carry what it computed from v over this point (it computes nothing itself)
template <typename T> __device__ __forceinline__ void hold(Vec<T>& v) {
    u32x4 r;
    __builtin_memcpy(&r, &v, 16);
    asm volatile("" : "+v"(r));
    __builtin_memcpy(&v, &r, 16);
}

// fp32 -> T.  For f16 the compiler would merge some multiply-adds with the conversion (one rounding instead of two) and leave others alone, by the
// registers it has in hand: the empty asm keeps them apart, so that every kernel rounds alike.
template <typename T> __device__ __forceinline__ T to(float f) {
    if constexpr (__is_same(T, _Float16)) asm("" : "+v"(f));
    return (T)f;
}

// N consecutive weights (fp32 or the rows' type) as fp32, zeros behind them; `none` where there are no weights
template <typename T, Tail TAIL> __device__ __forceinline__ void load_weights(const void* w, bool w32, int c, int D, float none, float (&out)[Vec<T>::N]) {
    constexpr int N = Vec<T>::N;
    if (w == nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = none;
    } else if (w32) {
#pragma unroll
        for (int h = 0; h < N; h += 4) {
            const Vec<float> v = load_vec<float, TAIL>((const float*)w, c + h, D);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[h + j] = v.e[j];
        }
    } else {
        const Vec<T> v = load_vec<T, TAIL>((const T*)w, c, D);
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = (float)v.e[j];
    }
}

// ------------------------------------------------------------------------------------------------------------------ sums over the threads of a row
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// sum over groups of G <= 64 neighbouring lanes, in all of them (butterflies through the lane-permuting operand reads and the row swaps: no LDS)
template <int G> __device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (G >= 2) v = dpp_add<0xB1>(v);        // lane ^ 1
    if constexpr (G >= 4) v = dpp_add<0x4E>(v);        // lane ^ 2
    if constexpr (G >= 8) v = dpp_add<0x141>(v);       // mirror inside 8 (quads hold one value by now)
    if constexpr (G >= 16) v = dpp_add<0x140>(v);      // mirror inside 16
    if constexpr (G >= 32) {
        const u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s.x) + __uint_as_float(s.y);
    }
    if constexpr (G >= 64) {
        const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s.x) + __uint_as_float(s.y);
    }
    return v;
}

// one or two sums over the G threads of a row.  G > 64: the row has the whole workgroup; `slot` alternates between calls, so that one barrier a call is
// enough (a wave writes slot s again only behind the barrier of the call on slot 1 - s, which every wave passes after reading s).
template <int G> __device__ __forceinline__ void row_sum2(float& a, float& b, float2 (*sh)[16], int slot) {
    if constexpr (G <= 64) {
        a = lanes_sum<G>(a);
        b = lanes_sum<G>(b);
    } else {
        a = lanes_sum<64>(a);
        b = lanes_sum<64>(b);
        if ((threadIdx.x & 63) == 0) sh[slot][threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) {
            const float2 s = sh[slot][i];
            a += s.x;
            b += s.y;
        }
    }
}

template <int G> __device__ __forceinline__ float row_sum(float a, float2 (*sh)[16], int slot) {
    if constexpr (G <= 64) return lanes_sum<G>(a);
    float none = 0.f;
    row_sum2<G>(a, none, sh, slot);
    return a;
}

// ------------------------------------------------------------------------------------------------------------------ dropout
// Element i of a tensor (flat, row-major) is kept where half i % 8 of the 128 bits that Philox4x32-10 gives for the counter (i / 8, offset) is
// >= threshold = round(65536 p).  16 bits an element: the rate moves in steps of 2^-16, and one call of the generator (20 multiplications of
// quarter rate) serves eight elements.
struct Drop {
    unsigned long long seed, offset;
    unsigned threshold;
    float scale;
};

__device__ __forceinline__ Drop drop_state(unsigned long long seed, unsigned long long offset, const int64_t* __restrict__ rng, unsigned threshold, float scale) {
    if (rng != nullptr) { seed = (unsigned long long)rng[0]; offset = (unsigned long long)rng[1]; }
    return Drop{seed, offset, threshold, scale};
}

// the bits of N = 4 or 8 elements from flat index i on, two to a word
template <int N> __device__ __forceinline__ void drop_bits(const Drop& d, unsigned long long i, unsigned (&w)[N / 2]) {
    const unsigned sh = (unsigned)i & 7u;
    const YpU4 a = yp_philox4x32(d.seed, i >> 3, d.offset);
    if (N == 8 && sh == 0) {
        w[0] = a.x; w[1] = a.y; w[N / 2 - 2] = a.z; w[N / 2 - 1] = a.w;
        return;
    }
    if (N == 4 && (sh == 0 || sh == 4)) {
        w[0] = sh ? a.z : a.x; w[1] = sh ? a.w : a.y;
        return;
    }
    // the elements straddle two counters: shift the eight words right by sh halves
    const YpU4 b = yp_philox4x32(d.seed, (i >> 3) + 1, d.offset);
    unsigned v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (sh & 4) {
#pragma unroll
        for (int k = 0; k < 6; ++k) v[k] = v[k + 2];
    }
    if (sh & 2) {
#pragma unroll
        for (int k = 0; k < 7; ++k) v[k] = v[k + 1];
    }
#pragma unroll
    for (int k = 0; k < N / 2; ++k) w[k] = (sh & 1) ? __builtin_amdgcn_alignbit(v[k + 1], v[k], 16) : v[k];
}

template <int N> __device__ __forceinline__ bool drop_kept(const Drop& d, const unsigned (&w)[N / 2], int j) {
    return ((j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu) >= d.threshold;
}

// out = res + (kept ? x * scale : 0): one fused multiply-add in fp32, rounded to T
template <typename T, bool DROP> __device__ __forceinline__ void drop_add(const Drop& d, unsigned long long i, const Vec<T>& x, const Vec<T>& res, Vec<T>& out) {
    constexpr int N = Vec<T>::N;
    unsigned w[N / 2];
    if constexpr (DROP) drop_bits<N>(d, i, w);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float r = (float)res.e[j];
        if constexpr (DROP) out.e[j] = to<T>(drop_kept<N>(d, w, j) ? fmaf((float)x.e[j], d.scale, r) : r);
        else out.e[j] = to<T>(r + (float)x.e[j]);
    }
}

// out = kept ? v * scale : 0
template <typename T> __device__ __forceinline__ void drop_only(const Drop& d, unsigned long long i, const float (&v)[Vec<T>::N], Vec<T>& out) {
    constexpr int N = Vec<T>::N;
    unsigned w[N / 2];
    drop_bits<N>(d, i, w);
#pragma unroll
    for (int j = 0; j < N; ++j) out.e[j] = to<T>(drop_kept<N>(d, w, j) ? v[j] * d.scale : 0.f);
}

template <typename T, bool RES, bool DROP, Tail TAIL>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y, int64_t n, unsigned long long seed,
                                                      unsigned long long offset, const int64_t* __restrict__ rng, unsigned threshold, float scale) {
    constexpr int N = Vec<T>::N;
    const Drop d = drop_state(seed, offset, rng, threshold, scale);
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N; i < n; i += (int64_t)gridDim.x * 256 * N) {
        // the tensor as one row that ends 2 N elements behind this thread's at the latest
        const int64_t at = max((int64_t)0, min(i, n - 2 * N));
        const int c = (int)(i - at), D = (int)min(n - at, (int64_t)(2 * N));
        const Vec<T> v = load_vec<T, TAIL>(x + at, c, D);
        Vec<T> o;
        if constexpr (RES) {
            drop_add<T, DROP>(d, i, v, load_vec<T, TAIL>(res + at, c, D), o);
        } else if constexpr (DROP) {
            float f[N];
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] = (float)v.e[j];
            drop_only<T>(d, i, f, o);
        } else {
            o = v;
        }
        store_vec<T>(y + i, o, min(N, D - c));
    }
}

// ------------------------------------------------------------------------------------------------------------------ layer norm
// A row of D features is held in the registers of G threads, E <= 16 features each in chunks of 16 bytes (thread t of a row: chunks t, t + G, ...):
// neighbouring threads read neighbouring 16 bytes, and the weights of a thread's columns stay in its registers over all of its rows.  G <= 64: one
// row or several a wave, sums without LDS; wider rows have a workgroup of G threads.
constexpr int ln_block(int G) { return G <= 64 ? 256 : G; }

struct LnFwd {
    const void *x, *res, *weight, *bias;
    void *z, *y;
    float *mean, *rstd;
    int64_t rows, xs, rs;
    int D;
    float eps;
    bool w32;
    unsigned long long seed, offset;
    const int64_t* rng;
    unsigned threshold;
    float scale;
};

// mean = sum x / D;  then, around that mean, d = x - mean: delta = sum d / D (what rounding left of the mean), var = sum d^2 / D - delta^2;
// y = (d - delta) rstd w + b.
// The next row is on its way while this one is worked on (the first before the weights are read).
template <typename T, int G, int E, bool RES, bool DROP, Tail TAIL>
__global__ __launch_bounds__(ln_block(G)) void ln_fwd_kernel(const LnFwd a) {
    constexpr int N = Vec<T>::N, NC = E / N, ROWS = ln_block(G) / G;
    __shared__ float2 sh[2][16];
    const T *x = (const T*)a.x, *res = (const T*)a.res;
    T *z = (T*)a.z, *y = (T*)a.y;
    const int t = threadIdx.x % G;
    const float inv_d = 1.0f / (float)a.D;
    const Drop d = drop_state(a.seed, a.offset, a.rng, a.threshold, a.scale);
    int c[NC], n[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) { c[k] = (t + k * G) * N; n[k] = max(0, min(N, a.D - c[k])); }
    const int64_t first = (int64_t)blockIdx.x * ROWS + threadIdx.x / G, step = (int64_t)gridDim.x * ROWS;
    Vec<T> nx[NC], nr[NC];
    auto fetch = [&](int64_t row) {
        row = min(row, a.rows - 1);
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            nx[k] = load_vec<T, TAIL>(x + row * a.xs, c[k], a.D);
            if (RES) nr[k] = load_vec<T, TAIL>(res + row * a.rs, c[k], a.D);
        }
    };
    fetch(first);
    float w[NC][N], b[NC][N];
#pragma unroll
    for (int k = 0; k < NC; ++k) { load_weights<T, TAIL>(a.weight, a.w32, c[k], a.D, 1.f, w[k]); load_weights<T, TAIL>(a.bias, a.w32, c[k], a.D, 0.f, b[k]); }
    for (int64_t row = first; row < a.rows; row += step) {
        Vec<T> v[NC];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            v[k] = nx[k];
            if constexpr (RES) {
                drop_add<T, DROP>(d, (unsigned long long)row * a.D + c[k], nx[k], nr[k], v[k]);
                store_vec<T>(z + row * a.D + c[k], v[k], n[k]);
            }
        }
        fetch(row + step);
        float f[NC][N], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) { f[k][j] = j < n[k] ? (float)v[k].e[j] : 0.f; s1 += f[k][j]; }
        const float mean = row_sum<G>(s1, sh, 0) * inv_d;
        s1 = 0.f;
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) {
                f[k][j] = j < n[k] ? f[k][j] - mean : 0.f;
                s1 += f[k][j];
                s2 = fmaf(f[k][j], f[k][j], s2);
            }
        row_sum2<G>(s1, s2, sh, 1);
        const float delta = s1 * inv_d;
        float var = fmaf(-delta, delta, s2 * inv_d);
        var = var < 0.f ? 0.f : var;                // (not fmaxf: a NaN stays one)
        const float rstd = 1.0f / sqrtf(var + a.eps);
        if (a.mean != nullptr && t == 0) { a.mean[row] = mean + delta; a.rstd[row] = rstd; }
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            Vec<T> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.e[j] = to<T>(fmaf((f[k][j] - delta) * rstd, w[k][j], b[k][j]));
            store_vec<T>(y + row * a.D + c[k], o, n[k]);
        }
    }
}

struct LnBwd {
    const void *z, *dy, *dz, *weight;
    const float *mean, *rstd;
    void *dres, *dx;
    float* partial;                                 // [gridDim.x][2][D]: dy xhat | dy summed over a workgroup's rows
    int64_t rows, zs, dys, dzs;
    int D;
    bool w32;
    unsigned long long seed, offset;
    const int64_t* rng;
    unsigned threshold;
    float scale;
};

// h = dy w, c1 = mean h, c2 = mean (h xhat);  dres = [dz +] rstd (h - c1 - xhat c2);  dx = kept ? dres scale : 0.
// dweight / dbias: a thread owns the same columns of every row it meets, so it sums them in its registers; a workgroup joins its rows through LDS and
// writes one line of partial sums; ln_columns_kernel adds the lines in order (no atomics: two passes give the same bits).
// Between the sums and the result the row waits in the type it was loaded in, and xhat and h are formed again (the empty asm keeps the compiler from
// holding them in fp32 instead: 2 E registers more a thread).
template <typename T, int G, int E, bool RES, bool DROP, Tail TAIL>
__global__ __launch_bounds__(ln_block(G)) void ln_bwd_kernel(const LnBwd a) {
    constexpr int N = Vec<T>::N, NC = E / N, BLOCK = ln_block(G), ROWS = BLOCK / G;
    __shared__ float2 sh[2][16];
    __shared__ float join[ROWS > 1 ? BLOCK * N : 1];
    const T *z = (const T*)a.z, *dy = (const T*)a.dy, *dz = (const T*)a.dz;
    T *dres = (T*)a.dres, *dx = (T*)a.dx;
    const int t = threadIdx.x % G;
    const float inv_d = 1.0f / (float)a.D;
    const Drop d = drop_state(a.seed, a.offset, a.rng, a.threshold, a.scale);
    int c[NC], n[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) { c[k] = (t + k * G) * N; n[k] = max(0, min(N, a.D - c[k])); }
    const int64_t first = (int64_t)blockIdx.x * ROWS + threadIdx.x / G, step = (int64_t)gridDim.x * ROWS;
    Vec<T> nv[NC], ng[NC], ne[NC];
    float nmean, nrstd;
    auto fetch = [&](int64_t row) {
        row = min(row, a.rows - 1);
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            nv[k] = load_vec<T, TAIL>(z + row * a.zs, c[k], a.D);
            ng[k] = load_vec<T, TAIL>(dy + row * a.dys, c[k], a.D);
            if (RES) ne[k] = load_vec<T, TAIL>(dz + row * a.dzs, c[k], a.D);
        }
        nmean = a.mean[row];
        nrstd = a.rstd[row];
    };
    fetch(first);
    float w[NC][N], dw[NC][N], db[NC][N];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        load_weights<T, TAIL>(a.weight, a.w32, c[k], a.D, 1.f, w[k]);
#pragma unroll
        for (int j = 0; j < N; ++j) dw[k][j] = db[k][j] = 0.f;
    }
    int slot = 0;
    for (int64_t row = first; row < a.rows; row += step) {
        Vec<T> v[NC], g[NC], e[NC];
#pragma unroll
        for (int k = 0; k < NC; ++k) { v[k] = nv[k]; g[k] = ng[k]; if (RES) e[k] = ne[k]; }
        const float mean = nmean, rstd = nrstd;
        fetch(row + step);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float gj = (float)g[k].e[j], xh = j < n[k] ? ((float)v[k].e[j] - mean) * rstd : 0.f;     // (gj is 0 behind the row's end)
                const float h = gj * w[k][j];
                dw[k][j] = fmaf(gj, xh, dw[k][j]);
                db[k][j] += gj;
                s1 += h;
                s2 = fmaf(h, xh, s2);
            }
            hold(v[k]);
            hold(g[k]);
        }
        row_sum2<G>(s1, s2, sh, slot);
        slot ^= 1;
        const float c1 = s1 * inv_d, c2 = s2 * inv_d;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            float o[N];
            Vec<T> ov;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float xh = ((float)v[k].e[j] - mean) * rstd;
                const float s = fmaf(-xh, c2, fmaf((float)g[k].e[j], w[k][j], -c1));
                if constexpr (RES) o[j] = fmaf(rstd, s, (float)e[k].e[j]);
                else o[j] = rstd * s;
                ov.e[j] = to<T>(o[j]);
            }
            store_vec<T>(dres + row * a.D + c[k], ov, n[k]);
            if constexpr (DROP) {
                drop_only<T>(d, (unsigned long long)row * a.D + c[k], o, ov);
                store_vec<T>(dx + row * a.D + c[k], ov, n[k]);
            }
        }
    }
    if (a.partial == nullptr) return;
    float* line = a.partial + (size_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            float s[N];
#pragma unroll
            for (int j = 0; j < N; ++j) s[j] = which ? db[k][j] : dw[k][j];
            if constexpr (ROWS > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < N; ++j) join[j * BLOCK + threadIdx.x] = s[j];
                __syncthreads();
                if (threadIdx.x < G) {
#pragma nounroll
                    for (int r = 1; r < ROWS; ++r)
#pragma unroll
                        for (int j = 0; j < N; ++j) s[j] += join[j * BLOCK + r * G + threadIdx.x];
                }
            }
            if (threadIdx.x < G) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (j < n[k]) line[which * a.D + c[k] + j] = s[j];
            }
        }
    }
}

// dweight | dbias [D] = sum of the partial lines, in order: 32 columns a workgroup, 32 slices of the lines beside each other
template <typename W>
__global__ __launch_bounds__(1024) void ln_columns_kernel(const float* __restrict__ partial, int lines, int D, W* __restrict__ dw, W* __restrict__ db) {
    __shared__ float sh[32][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + col;            // [0, 2 D)
    float s = 0.f;
    if (i < 2 * D) {
        int l = slice;
        for (; l + 96 < lines; l += 128) {
            const float p0 = partial[(size_t)l * 2 * D + i], p1 = partial[(size_t)(l + 32) * 2 * D + i], p2 = partial[(size_t)(l + 64) * 2 * D + i],
                        p3 = partial[(size_t)(l + 96) * 2 * D + i];
            s += p0; s += p1; s += p2; s += p3;
        }
        for (; l < lines; l += 32) s += partial[(size_t)l * 2 * D + i];
    }
    sh[slice][col] = s;
    __syncthreads();
    if (slice == 0 && i < 2 * D) {
        s = sh[0][col];
#pragma unroll
        for (int r = 1; r < 32; ++r) s += sh[r][col];
        if (i < D) { if (dw != nullptr) dw[i] = to<W>(s); }
        else if (db != nullptr) db[i - D] = to<W>(s);
    }
}

// ------------------------------------------------------------------------------------------------------------------ rotary positions
struct Rot {
    const void *q, *k;
    void *qo, *ko;
    const void* positions;
    const double* freq;
    int64_t qs[3], ks[3], qos[3], kos[3];           // strides of batch, token, head
    int64_t ps[3];                                  // of the positions: batch, token, axis
    int64_t start;
    int T, tokens, Hq, Hk, D, R, ptype, axes, hs;
    float scale, sign;
    bool interleaved, in_place;
};

// cos and sin of `turns` turns: the quarter turn by 64-bit arithmetic (positions of a million leave 2^-33 of a turn there and nothing in 32 bits), the
// rest |theta| <= pi / 4 by the Taylor series, whose first term left out is below 2e-9
__device__ __forceinline__ void turn_cos_sin(double turns, float& c, float& s) {
    const double f = turns - rint(turns);
    const double q = rint(4.0 * f);
    const float th = (float)(fma(q, -0.25, f) * 6.283185307179586476925);
    const int iq = (int)q;
    const float t2 = th * th;
    const float ss = fmaf(th * t2, fmaf(t2, fmaf(t2, fmaf(t2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), th);
    const float cc = fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
    const float a = (iq & 1) ? ss : cc, b = (iq & 1) ? cc : ss;
    c = ((iq + 1) & 2) ? -a : a;
    s = (iq & 2) ? -b : b;
}

// A thread owns one chunk of a head's pairs (16 bytes of each half, or 32 bytes of interleaved pairs) of one token, and walks the heads slot, slot + hs,
// ... of q and then of k with the same cosines and sines.
template <typename T, Tail TAIL>
__global__ __launch_bounds__(256) void rotary_kernel(const Rot a) {
    constexpr int N = Vec<T>::N;
    const int half = a.R >> 1;
    const int turned = (half + N - 1) / N, copied = a.in_place ? 0 : (a.D - a.R + 2 * N - 1) / (2 * N), chunks = turned + copied;
    const int items = a.hs * chunks, per = 256 / items;
    const int lt = threadIdx.x / items, item = threadIdx.x - lt * items;
    if (lt >= per) return;
    const int slot = item / chunks, ch = item - slot * chunks;
    const int H = a.Hq + a.Hk;
    const bool turns = ch < turned;
    const int j0 = turns ? ch * N : 0;
    // the thread's two 16-byte pieces: elements c0 .. | c1 .. of the runs of `len` features that start at s0 | s1 of the head
    const int len = !turns ? a.D - a.R : a.interleaved ? a.R : half;
    const int s0 = turns ? 0 : a.R, s1 = turns && !a.interleaved ? half : s0;
    const int c0 = turns ? (a.interleaved ? 2 * j0 : j0) : (ch - turned) * 2 * N, c1 = s1 == s0 ? c0 + N : c0;
    const int n0 = max(0, min(N, len - c0)), n1 = max(0, min(N, len - c1));
    const int per_axis = half / a.axes;
    for (int64_t tok = (int64_t)blockIdx.x * per + lt; tok < a.tokens; tok += (int64_t)gridDim.x * per) {
        const unsigned bi = (unsigned)tok / (unsigned)a.T;
        const int ti = (int)((unsigned)tok - bi * (unsigned)a.T);
        float cs[N], sn[N];
        if (turns) {
            double p0, p1;
            if (a.positions == nullptr) {
                p0 = p1 = (double)(a.start + ti);
            } else {
                const int64_t at = bi * a.ps[0] + ti * a.ps[1];
                if (a.ptype == YP_POS_I64) { p0 = (double)((const int64_t*)a.positions)[at]; p1 = (double)((const int64_t*)a.positions)[at + (a.axes - 1) * a.ps[2]]; }
                else if (a.ptype == YP_POS_I32) { p0 = (double)((const int32_t*)a.positions)[at]; p1 = (double)((const int32_t*)a.positions)[at + (a.axes - 1) * a.ps[2]]; }
                else { p0 = (double)((const float*)a.positions)[at]; p1 = (double)((const float*)a.positions)[at + (a.axes - 1) * a.ps[2]]; }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int pair = min(j0 + j, half - 1);
                const double f = a.freq[pair] * 0.15915494309189533576888;        // radians -> turns
                turn_cos_sin((pair >= per_axis ? p1 : p0) * f, cs[j], sn[j]);
                cs[j] *= a.scale;
                sn[j] *= a.scale * a.sign;
            }
        }
        for (int h = slot; h < H; h += a.hs) {
            const bool isq = h < a.Hq;
            const int hh = isq ? h : h - a.Hq;
            const T* in = (const T*)(isq ? a.q : a.k) + bi * (isq ? a.qs[0] : a.ks[0]) + ti * (isq ? a.qs[1] : a.ks[1]) + hh * (isq ? a.qs[2] : a.ks[2]);
            T* out = (T*)(isq ? a.qo : a.ko) + bi * (isq ? a.qos[0] : a.kos[0]) + ti * (isq ? a.qos[1] : a.kos[1]) + hh * (isq ? a.qos[2] : a.kos[2]);
            Vec<T> u = load_vec<T, TAIL>(in + s0, c0, len), v = load_vec<T, TAIL>(in + s1, c1, len);
            if (turns && a.interleaved) {
                Vec<T> ou, ov;
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    const float x0 = (float)u.e[2 * j], x1 = (float)u.e[2 * j + 1], y0 = (float)v.e[2 * j], y1 = (float)v.e[2 * j + 1];
                    ou.e[2 * j] = to<T>(fmaf(x0, cs[j], -(x1 * sn[j])));
                    ou.e[2 * j + 1] = to<T>(fmaf(x1, cs[j], x0 * sn[j]));
                    ov.e[2 * j] = to<T>(fmaf(y0, cs[j + N / 2], -(y1 * sn[j + N / 2])));
                    ov.e[2 * j + 1] = to<T>(fmaf(y1, cs[j + N / 2], y0 * sn[j + N / 2]));
                }
                u = ou;
                v = ov;
            } else if (turns) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float x0 = (float)u.e[j], x1 = (float)v.e[j];
                    u.e[j] = to<T>(fmaf(x0, cs[j], -(x1 * sn[j])));
                    v.e[j] = to<T>(fmaf(x1, cs[j], x0 * sn[j]));
                }
            }
            store_vec<T>(out + s0 + c0, u, n0);
            store_vec<T>(out + s1 + c1, v, n1);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------ host
// the shapes of a row over threads (threads, features a thread), narrowest first; the first that holds the row is taken
#define LN_SHAPES(X) X(4, 8) X(8, 8) X(16, 8) X(32, 8) X(64, 8) X(64, 16) X(128, 16) X(256, 16) X(512, 16) X(1024, 16)
constexpr int LN_WIDEST = 1024 * 16;

struct LnShape { int G, E; };
LnShape ln_shape(int D) {
#define PICK(G_, E_) if (D <= G_ * E_) return LnShape{G_, E_};
    LN_SHAPES(PICK)
#undef PICK
    return LnShape{0, 0};
}
int ln_rows_per_block(int G) { return ln_block(G) / G; }

// workgroups of a backward pass: enough to fill the chip, few enough that their lines of partial sums stay small beside the rows
int ln_bwd_blocks(int64_t rows, int D) {
    const int per = ln_rows_per_block(ln_shape(D).G);
    const int64_t want = (rows + per - 1) / per;
    return (int)(want < 1024 ? want : 1024);
}

int drop_parameters(double p, unsigned* threshold, float* scale) {
    if (!(p >= 0.0 && p <= 1.0)) return 0;
    *threshold = (unsigned)(p * 65536.0 + 0.5);
    *scale = *threshold < 65536u ? (float)(65536.0 / (65536.0 - (double)*threshold)) : 0.f;
    return 1;
}

// KERNEL<T, G, E, RES, DROP, TAIL> for run-time shape, operands and row end
#define LN_RUN(KERNEL, G_, E_, ...) KERNEL<T, G_, E_, __VA_ARGS__><<<blocks, ln_block(G_), 0, st>>>(a)
#define LN_ENDS(KERNEL, G_, E_, RES_, DROP_) \
    if (a.D % Vec<T>::N == 0) LN_RUN(KERNEL, G_, E_, RES_, DROP_, WHOLE); \
    else if (a.D > Vec<T>::N) LN_RUN(KERNEL, G_, E_, RES_, DROP_, CUT); \
    else if constexpr (G_ == 4) LN_RUN(KERNEL, G_, E_, RES_, DROP_, SHORT);
#define LN_FWD(G_, E_) if (s.G == G_ && s.E == E_) { if (!res) { LN_ENDS(ln_fwd_kernel, G_, E_, false, false) } else if (!drop) { LN_ENDS(ln_fwd_kernel, G_, E_, true, false) } \
        else { LN_ENDS(ln_fwd_kernel, G_, E_, true, true) } return; }
#define LN_BWD(G_, E_) if (s.G == G_ && s.E == E_) { if (!res && !drop) { LN_ENDS(ln_bwd_kernel, G_, E_, false, false) } else if (!drop) { LN_ENDS(ln_bwd_kernel, G_, E_, true, false) } \
        else if (!res) { LN_ENDS(ln_bwd_kernel, G_, E_, false, true) } else { LN_ENDS(ln_bwd_kernel, G_, E_, true, true) } return; }
template <typename T> void ln_fwd_launch(const LnFwd& a, LnShape s, bool res, bool drop, int blocks, hipStream_t st) { LN_SHAPES(LN_FWD) }
template <typename T> void ln_bwd_launch(const LnBwd& a, LnShape s, bool res, bool drop, int blocks, hipStream_t st) { LN_SHAPES(LN_BWD) }

bool ln_types(const YpLayerNormDesc* d) {
    return (d->dtype == YP_F16 || d->dtype == YP_BF16 || d->dtype == YP_F32) && (d->wdtype == YP_F32 || d->wdtype == d->dtype);
}

}  // namespace

extern "C" int yp_layer_norm_max_width(int dtype) { return dtype == YP_F16 || dtype == YP_BF16 || dtype == YP_F32 ? LN_WIDEST : 0; }

extern "C" int yp_layer_norm_fwd(const YpLayerNormDesc* d, void* stream) {
    YP_REQUIRE(d != nullptr, "yp_layer_norm_fwd: no descriptor");
    YP_REQUIRE(ln_types(d), "yp_layer_norm_fwd: types %d / %d", d->dtype, d->wdtype);
    YP_REQUIRE(d->rows >= 0 && d->D >= 1 && d->D <= yp_layer_norm_max_width(d->dtype), "yp_layer_norm_fwd: %lld rows of %d", (long long)d->rows, d->D);
    if (d->rows == 0) return YP_OK;
    YP_REQUIRE(d->x && d->y && (d->res == nullptr || d->z) && (d->mean == nullptr) == (d->rstd == nullptr), "yp_layer_norm_fwd: a buffer is missing");
    YP_REQUIRE(d->x_stride >= 0 && d->res_stride >= 0, "yp_layer_norm_fwd: negative stride");
    LnFwd a{};
    YP_REQUIRE(drop_parameters(d->p, &a.threshold, &a.scale), "yp_layer_norm_fwd: a dropout rate of %g", d->p);
    YP_REQUIRE(d->res != nullptr || a.threshold == 0, "yp_layer_norm_fwd: dropout needs a residual");
    a.x = d->x; a.res = d->res; a.weight = d->weight; a.bias = d->bias; a.z = d->z; a.y = d->y; a.mean = d->mean; a.rstd = d->rstd;
    a.rows = d->rows; a.xs = d->x_stride; a.rs = d->res_stride; a.D = d->D; a.eps = d->eps; a.w32 = d->wdtype == YP_F32;
    a.seed = d->seed; a.offset = d->offset; a.rng = d->rng;
    const LnShape s = ln_shape(d->D);
    const int64_t per = ln_rows_per_block(s.G), want = (d->rows + per - 1) / per;
    const int blocks = (int)(want < 4096 ? want : 4096);
    hipStream_t st = (hipStream_t)stream;
    const bool drop = a.threshold != 0;
    if (d->dtype == YP_F16) ln_fwd_launch<_Float16>(a, s, d->res != nullptr, drop, blocks, st);
    else if (d->dtype == YP_BF16) ln_fwd_launch<__bf16>(a, s, d->res != nullptr, drop, blocks, st);
    else ln_fwd_launch<float>(a, s, d->res != nullptr, drop, blocks, st);
    YP_CHECK_HIP(hipGetLastError());
    return YP_OK;
}

extern "C" size_t yp_layer_norm_bwd_workspace_bytes(int64_t rows, int D, int dtype) {
    if (rows <= 0 || D < 1 || D > yp_layer_norm_max_width(dtype)) return 0;
    return (size_t)ln_bwd_blocks(rows, D) * 2 * (size_t)D * sizeof(float);
}

extern "C" int yp_layer_norm_bwd(const YpLayerNormDesc* d, void* stream) {
    YP_REQUIRE(d != nullptr, "yp_layer_norm_bwd: no descriptor");
    YP_REQUIRE(ln_types(d), "yp_layer_norm_bwd: types %d / %d", d->dtype, d->wdtype);
    YP_REQUIRE(d->rows >= 0 && d->D >= 1 && d->D <= yp_layer_norm_max_width(d->dtype), "yp_layer_norm_bwd: %lld rows of %d", (long long)d->rows, d->D);
    const bool sums = d->dweight != nullptr || d->dbias != nullptr;
    hipStream_t st = (hipStream_t)stream;
    int blocks = 0;
    if (d->rows > 0) {
        LnBwd a{};
        YP_REQUIRE(drop_parameters(d->p, &a.threshold, &a.scale), "yp_layer_norm_bwd: a dropout rate of %g", d->p);
        const bool drop = a.threshold != 0;
        YP_REQUIRE(d->x && d->dy && d->mean && d->rstd && d->dres && (!drop || d->dx), "yp_layer_norm_bwd: a buffer is missing");
        YP_REQUIRE(d->x_stride >= 0 && d->dy_stride >= 0 && d->dz_stride >= 0, "yp_layer_norm_bwd: negative stride");
        if (sums && (d->workspace == nullptr || d->workspace_bytes < yp_layer_norm_bwd_workspace_bytes(d->rows, d->D, d->dtype))) {
            yp_set_error("yp_layer_norm_bwd: workspace of %zu bytes, %zu needed", d->workspace_bytes, yp_layer_norm_bwd_workspace_bytes(d->rows, d->D, d->dtype));
            return YP_ERR_WORKSPACE;
        }
        a.z = d->x; a.dy = d->dy; a.dz = d->dz; a.weight = d->weight; a.mean = d->mean; a.rstd = d->rstd; a.dres = d->dres; a.dx = d->dx;
        a.partial = sums ? (float*)d->workspace : nullptr;
        a.rows = d->rows; a.zs = d->x_stride; a.dys = d->dy_stride; a.dzs = d->dz_stride; a.D = d->D; a.w32 = d->wdtype == YP_F32;
        a.seed = d->seed; a.offset = d->offset; a.rng = d->rng;
        const LnShape s = ln_shape(d->D);
        blocks = ln_bwd_blocks(d->rows, d->D);
        if (d->dtype == YP_F16) ln_bwd_launch<_Float16>(a, s, d->dz != nullptr, drop, blocks, st);
        else if (d->dtype == YP_BF16) ln_bwd_launch<__bf16>(a, s, d->dz != nullptr, drop, blocks, st);
        else ln_bwd_launch<float>(a, s, d->dz != nullptr, drop, blocks, st);
        YP_CHECK_HIP(hipGetLastError());
    }
    if (sums) {
        const int grid = (2 * d->D + 31) / 32;
        const float* p = (const float*)d->workspace;
        if (d->wdtype == YP_F32) ln_columns_kernel<float><<<grid, 1024, 0, st>>>(p, blocks, d->D, (float*)d->dweight, (float*)d->dbias);
        else if (d->wdtype == YP_F16) ln_columns_kernel<_Float16><<<grid, 1024, 0, st>>>(p, blocks, d->D, (_Float16*)d->dweight, (_Float16*)d->dbias);
        else ln_columns_kernel<__bf16><<<grid, 1024, 0, st>>>(p, blocks, d->D, (__bf16*)d->dweight, (__bf16*)d->dbias);
        YP_CHECK_HIP(hipGetLastError());
    }
    return YP_OK;
}

extern "C" int yp_dropout(const void* x, const void* res, void* y, int64_t n, int dtype, double p, uint64_t seed, uint64_t offset, const int64_t* rng, void* stream) {
    unsigned threshold = 0;
    float scale = 0.f;
    YP_REQUIRE(dtype == YP_F16 || dtype == YP_BF16 || dtype == YP_F32, "yp_dropout: type %d", dtype);
    YP_REQUIRE(drop_parameters(p, &threshold, &scale), "yp_dropout: a rate of %g", p);
    YP_REQUIRE(n >= 0, "yp_dropout: %lld elements", (long long)n);
    if (n == 0) return YP_OK;
    YP_REQUIRE(x && y, "yp_dropout: a buffer is missing");
    const int64_t per = 256 * (dtype == YP_F32 ? 4 : 8), want = (n + per - 1) / per;
    const unsigned blocks = (unsigned)(want < 16384 ? want : 16384);
    hipStream_t st = (hipStream_t)stream;
#define END(T_, RES_, DROP_) \
        if (n % Vec<T_>::N == 0) dropout_kernel<T_, RES_, DROP_, WHOLE><<<blocks, 256, 0, st>>>((const T_*)x, (const T_*)res, (T_*)y, n, seed, offset, rng, threshold, scale); \
        else if (n > Vec<T_>::N) dropout_kernel<T_, RES_, DROP_, CUT><<<blocks, 256, 0, st>>>((const T_*)x, (const T_*)res, (T_*)y, n, seed, offset, rng, threshold, scale); \
        else dropout_kernel<T_, RES_, DROP_, SHORT><<<blocks, 256, 0, st>>>((const T_*)x, (const T_*)res, (T_*)y, n, seed, offset, rng, threshold, scale)
#define RUN(T_) do { \
        if (res) { if (threshold) END(T_, true, true); else END(T_, true, false); } \
        else { if (threshold) END(T_, false, true); else END(T_, false, false); } } while (0)
    if (dtype == YP_F16) RUN(_Float16); else if (dtype == YP_BF16) RUN(__bf16); else RUN(float);
#undef RUN
#undef END
    YP_CHECK_HIP(hipGetLastError());
    return YP_OK;
}

extern "C" int yp_rotary(const YpRotaryDesc* d, void* stream) {
    YP_REQUIRE(d != nullptr, "yp_rotary: no descriptor");
    YP_REQUIRE(d->dtype == YP_F16 || d->dtype == YP_BF16 || d->dtype == YP_F32, "yp_rotary: type %d", d->dtype);
    YP_REQUIRE(d->B >= 0 && d->T >= 0 && d->Hq >= 0 && d->Hk >= 0 && (int64_t)d->B * d->T < (int64_t)1 << 31, "yp_rotary: %d x %d tokens, %d + %d heads", d->B, d->T, d->Hq, d->Hk);
    YP_REQUIRE(d->D >= 2 && d->D <= 1024 && d->R >= 2 && d->R <= d->D && d->R % 2 == 0, "yp_rotary: %d of %d features", d->R, d->D);
    YP_REQUIRE((d->axes == 1 || d->axes == 2) && d->R / 2 % d->axes == 0, "yp_rotary: %d axes over %d pairs", d->axes, d->R / 2);
    YP_REQUIRE(d->position_type == YP_POS_I32 || d->position_type == YP_POS_I64 || d->position_type == YP_POS_F32, "yp_rotary: positions of type %d", d->position_type);
    if (d->B == 0 || d->T == 0 || d->Hq + d->Hk == 0) return YP_OK;
    YP_REQUIRE((d->Hq == 0 || (d->q && d->q_out)) && (d->Hk == 0 || (d->k && d->k_out)) && d->inv_freq, "yp_rotary: a buffer is missing");
    YP_REQUIRE(d->positions || d->axes == 1, "yp_rotary: two axes need positions");
    Rot a{};
    a.q = d->q; a.k = d->k; a.qo = d->q_out; a.ko = d->k_out; a.positions = d->positions; a.freq = d->inv_freq;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = d->q_stride[i]; a.ks[i] = d->k_stride[i]; a.qos[i] = d->q_out_stride[i]; a.kos[i] = d->k_out_stride[i]; a.ps[i] = d->position_stride[i];
    }
    a.start = d->start; a.T = d->T; a.tokens = d->B * d->T; a.Hq = d->Hq; a.Hk = d->Hk; a.D = d->D; a.R = d->R; a.ptype = d->position_type; a.axes = d->axes;
    a.scale = d->scale; a.sign = d->inverse ? -1.f : 1.f; a.interleaved = d->interleaved != 0; a.in_place = d->q == d->q_out && d->k == d->k_out;
    const int N = d->dtype == YP_F32 ? 4 : 8, H = d->Hq + d->Hk;
    const int chunks = (d->R / 2 + N - 1) / N + (a.in_place ? 0 : (d->D - d->R + 2 * N - 1) / (2 * N));
    // heads beside each other: all of them while the tokens alone do not fill the chip, else four to a thread (they share its cosines)
    const bool few = (int64_t)a.tokens * H * chunks <= 256 * 2048;
    int hs = few ? H : (H + 3) / 4;
    if (hs > 256 / chunks) hs = 256 / chunks;
    a.hs = hs;
    const int per = 256 / (hs * chunks);
    const int64_t want = ((int64_t)a.tokens + per - 1) / per;
    const unsigned blocks = (unsigned)(want < 65536 ? want : 65536);
    hipStream_t st = (hipStream_t)stream;
    const int turned_run = a.interleaved ? a.R : a.R / 2, copied_run = a.in_place ? 0 : a.D - a.R;
    const Tail tail = turned_run % N == 0 && copied_run % N == 0 ? WHOLE : turned_run >= N && (copied_run == 0 || copied_run >= N) ? CUT : SHORT;
#define RUN(T_) do { if (tail == WHOLE) rotary_kernel<T_, WHOLE><<<blocks, 256, 0, st>>>(a); else if (tail == CUT) rotary_kernel<T_, CUT><<<blocks, 256, 0, st>>>(a); \
        else rotary_kernel<T_, SHORT><<<blocks, 256, 0, st>>>(a); } while (0)
    if (d->dtype == YP_F16) RUN(_Float16); else if (d->dtype == YP_BF16) RUN(__bf16); else RUN(float);
#undef RUN
    YP_CHECK_HIP(hipGetLastError());
    return YP_OK;
}
