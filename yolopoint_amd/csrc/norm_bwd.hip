// Layer norm, backward: the gradient of the rows (through residual and dropout where the forward pass had them) and the sums over the rows that are the
// gradients of weight and bias.  Bound by HBM: each row of each operand is read once, each gradient written once.
#include "norm.h"

namespace {

struct LnBwd {
    const void *z, *dy, *dz, *weight;
    const float *mean, *rstd, *rest;                // [rows] each, or with_rest: one behind the other in lines of three; rest is the means again without it
    void *dres, *dx;
    float* partial;                                 // [gridDim.x][2][D]: dy xhat | dy summed over a workgroup's rows
    int64_t rows, zs, dys, dzs;
    int D, waves, each;                             // G = 0: waves a row, rows a workgroup
    bool w32;
    unsigned long long seed, offset;
    const int64_t* rng;
    unsigned threshold;
    float scale, inv_width;                         // 1 / D (an argument: no register of the lanes)
    bool with_rest;
};

// h = dy w, c1 = mean h, c2 = mean (h xhat);  dres = [dz +] rstd (h - c1 - xhat c2);  dx = kept ? dres scale : 0.
// xhat is the forward pass's: z rstd + shift is one multiply-add, whose shift -mean rstd carries the rounding of the product and of the mean; `low` is what
// those left (without it a constant f32 row of 13730 had xhat 0.04, and dweight and dx got terms that do not exist).  Where xhat is formed a second
// time (TIGHT) it is formed without it, and the row's sums are moved instead.  One addition a value: nothing where HBM bounds, 3 - 5 % at odd 16-bit
// widths with dropout, 6 - 8 % at those of more than 8192 features.
// dweight / dbias: a thread owns the same columns of every row it meets, so it sums them in its registers; a workgroup of some 512 threads joins its rows
// through LDS and writes one line of partial sums; ln_columns_kernel adds the lines in order (no atomics: two passes give the same bits).
// E = 16 (rows that 16 waves of 8 features a thread do not hold): no registers are left for the next row, nor for the weights, which wait in LDS (as
// 16-byte pieces: no bank twice); between the sums and the result the row waits in the type it was loaded in, and xhat and h are formed again (the
// empty asm keeps the compiler from holding them in fp32 instead); one chunk after the other, so that only one's random numbers are live.
// Measured, 128 MiB a tensor: 79 - 106 us for widths 16 .. 16384 (3.8 - 5.1 TB/s over the two tensors read and one written; odd 16-bit widths over 4096: 115 -
// 135), through residual and dropout 129 - 164 us (4.1 - 5.2 over five); odd bf16 widths with dropout are bound by their instructions (777: 170, 2100: 217,
// 4099: 244, 12345: 257 us), rows of more than 8192 features by registers that do not suffice: all their fp32 kernels spill 12 - 55 (16384 with dropout:
// 204 us), the 16-bit ones with dropout up to 14.
template <typename T, int G, int E, bool RES, bool DROP, Tail TAIL>
__global__ __launch_bounds__(G ? 512 : 1024, 4) void ln_bwd_kernel(const LnBwd a) {
    constexpr int N = Vec<T>::N, NC = E / N;
    constexpr bool TIGHT = E > 8, SCALAR = TIGHT && sizeof(T) == 2;       // SCALAR: a row's numbers wait on the scalar unit (fp32 rows and narrower ones lose by it)
    constexpr bool EARLY = !TIGHT && !(sizeof(T) == 4 && RES && DROP);     // the next row is on its way while this one is worked on, where registers are left
    __shared__ float2 sh[2][16];
    extern __shared__ float lds[];                  // TIGHT: the weights; then the space in which a workgroup's rows join
    const T *z = (const T*)a.z, *dy = (const T*)a.dy, *dz = (const T*)a.dz;
    T *dres = (T*)a.dres, *dx = (T*)a.dx;
    // threads of a row, rows of the workgroup, this thread's place
    const int threads = G ? G : a.waves * 64, each = G ? 512 / G : a.each;
    const int sub = G ? row_in_block<G>() : __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) / a.waves), t = G ? threadIdx.x % G : threadIdx.x - sub * threads;
    const Drop d = drop_state(a.seed, a.offset, a.rng, a.threshold, a.scale);
    int c[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) c[k] = (t + k * threads) * N;
    // (G = 0: all rows of a workgroup take every step together, for its barriers; one behind the last row repeats that with a gradient of zero and
    // stores nothing)
    const int64_t first = (int64_t)blockIdx.x * each + sub, step = (int64_t)gridDim.x * each, end = G ? a.rows : (a.rows + each - 1) / each * each;
    Vec<T> nv[NC], ng[NC], ne[NC];
    float nmean, nrstd, nrest;
    int64_t at = min(first, a.rows - 1);
    const T *pz = z + at * a.zs, *pg = dy + at * a.dys, *pe = RES ? dz + at * a.dzs : nullptr;
    auto fetch = [&]() {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            nv[k] = fetch_vec<T, TAIL>(pz, c[k], a.D);
            ng[k] = fetch_vec<T, TAIL>(pg, c[k], a.D);
            if constexpr (RES) ne[k] = fetch_vec<T, TAIL>(pe, c[k], a.D);
        }
        const int64_t line = a.with_rest ? at * 3 : at;
        nmean = a.mean[line];
        nrstd = a.rstd[line];
        nrest = a.rest[line];
    };
    if constexpr (EARLY) fetch();
    float w[TIGHT ? 1 : NC][N], dw[NC][N], db[NC][N];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
        float wk[N];
        load_weights<T, TAIL>(a.weight, a.w32, c[k], a.D, 1.f, wk);
        if constexpr (TIGHT) {
#pragma unroll
            for (int h = 0; h < N; h += 4) *(float4*)&lds[((k * (N / 4) + h / 4) * threads + t) * 4] = make_float4(wk[h], wk[h + 1], wk[h + 2], wk[h + 3]);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            dw[k][j] = db[k][j] = 0.f;
            if constexpr (!TIGHT) w[k][j] = wk[j];
        }
    }
    auto weights = [&](int k, float (&wk)[N]) {     // (each thread reads what it wrote itself: no barrier)
        if constexpr (TIGHT) {
#pragma unroll
            for (int h = 0; h < N; h += 4) {
                const float4 q = *(const float4*)&lds[((k * (N / 4) + h / 4) * threads + t) * 4];
                wk[h] = q.x; wk[h + 1] = q.y; wk[h + 2] = q.z; wk[h + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) wk[j] = w[k][j];
        }
    };
    int slot = 0;
    for (int64_t row = first; row < end; row += step) {
        if constexpr (!EARLY) fetch();
        const bool real = G || row < a.rows;
        Vec<T> v[NC], g[NC], e[NC];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            v[k] = settle<T, TAIL>(nv[k], c[k], a.D);
            g[k] = settle<T, TAIL>(ng[k], c[k], a.D);
            if constexpr (RES) e[k] = settle<T, TAIL>(ne[k], c[k], a.D);
            if (!real) g[k] = Vec<T>{};
        }
        float rstd = nrstd, shift = -nmean * rstd, low = fmaf(a.with_rest ? -nrest : 0.f, rstd, -fmaf(nmean, rstd, shift));
        if constexpr (SCALAR) { rstd = of_wave(rstd); shift = of_wave(shift); low = of_wave(low); }
        if (row + step < end) {
            const int64_t next = min(row + step, a.rows - 1);
            pz += (next - at) * a.zs;
            pg += (next - at) * a.dys;
            if (RES) pe += (next - at) * a.dzs;
            at = next;
            if constexpr (EARLY) fetch();
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const float sk = c[k] < a.D ? shift : 0.f;
            float wk[N];
            weights(k, wk);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float gj = (float)g[k].e[j], xh = fmaf((float)v[k].e[j], rstd, sk) + low;  // (gj is 0 behind the row's end)
                const float h = gj * wk[j];
                dw[k][j] = fmaf(gj, xh, dw[k][j]);
                db[k][j] += gj;
                s1 += h;
                s2 = fmaf(h, xh, s2);
            }
            if constexpr (TIGHT) {
                hold(v[k]);
                hold(g[k]);
            }
        }
        row_sum2<G>(s1, s2, sh[slot], sub * a.waves, a.waves);
        slot ^= 1;
        float c1 = s1 * a.inv_width, c2 = s2 * a.inv_width;
        if constexpr (TIGHT) c1 = fmaf(low, c2, c1);           // (where xhat is formed again, it is formed without its low part)
        if constexpr (SCALAR) { c1 = of_wave(c1); c2 = of_wave(c2); }
        if (!real || (!DROP && a.dres == nullptr)) continue;    // (with dropout dres goes with dx: a branch around its store costs 13 of 227 us at 2100 features)
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            if (DROP && G == 0 && __ballot(c[k] < a.D) == 0ull) continue;           // (a wave behind the row's end makes no random numbers)
            const float sk = c[k] < a.D ? shift : 0.f;
            float o[N], wk[N];
            weights(k, wk);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float xh = TIGHT ? fmaf((float)v[k].e[j], rstd, sk) : fmaf((float)v[k].e[j], rstd, sk) + low;
                const float h = (float)g[k].e[j] * wk[j];
                const float s = fmaf(-xh, c2, h - c1);
                if constexpr (RES) o[j] = fmaf(rstd, s, (float)e[k].e[j]);
                else o[j] = rstd * s;
            }
            Vec<T> ov;
            if constexpr (DROP) {
                drop_only<T, TAIL != WHOLE, G == 0 || G == 64, sizeof(T) == 2 && !(TIGHT && TAIL != WHOLE)>(d, (unsigned long long)row * a.D + c[k], o, ov, last_lane<G>(), a.D - c[k]);
                store_vec<T, TAIL>(dx + row * a.D, c[k], a.D, ov);
            }
            store_vec<T, TAIL>(dres + row * a.D, c[k], a.D, to_vec<T>(o));
            if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
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
            if constexpr (G != 0) {                 // rows join two at a time: in every step the upper half hands its sums to the lower
#pragma unroll
                for (int half = 512 / (G ? G : 1) / 2; half > 0; half >>= 1) {
                    const int r = threadIdx.x / (G ? G : 1);
                    __syncthreads();
                    if (r >= half && r < 2 * half) {
#pragma unroll
                        for (int j = 0; j < N; ++j) lds[j * 256 + threadIdx.x - half * G] = s[j];
                    }
                    __syncthreads();
                    if (r < half) {
#pragma unroll
                        for (int j = 0; j < N; ++j) s[j] += lds[j * 256 + threadIdx.x];
                    }
                }
            } else {                                // four rows at the most: one after the other
                for (int r = 1; r < each; ++r) {
                    __syncthreads();
                    if (sub == r) {
#pragma unroll
                        for (int j = 0; j < N; ++j) lds[j * threads + t] = s[j];
                    }
                    __syncthreads();
                    if (sub == 0) {
#pragma unroll
                        for (int j = 0; j < N; ++j) s[j] += lds[j * threads + t];
                    }
                }
            }
            if (G ? threadIdx.x < G : sub == 0) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (c[k] + j < a.D) line[which * a.D + c[k] + j] = s[j];
            }
        }
    }
}

// dweight | dbias [D] = sum of the partial lines, in order: 32 columns a workgroup, 32 slices of the lines beside each other (512 lines of 2 x 1024: 3.9 us)
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

// The shape of a row: G threads with 8 features each, the first that holds it; G = 0: waves of 64 threads with 8 features each (16 where 16 waves do not
// hold the row: its sums for the weights' gradients are another 2 E registers a thread, and two waves a SIMD less cost more than the barrier), rows
// beside each other up to eight waves a workgroup (three waves: four rows, so that the four SIMDs hold as many waves each).
#define LN_SHAPES(X) X(4, 8) X(8, 8) X(16, 8) X(32, 8) X(64, 8) X(0, 8) X(0, 16)
struct LnShape { int G, E, waves, each, block; };
LnShape ln_shape(int D) {
#define PICK(G_, E_) if (G_ && D <= G_ * E_) return LnShape{G_, E_, 1, 512 / G_, 512};
    LN_SHAPES(PICK)
#undef PICK
    const int E = D <= 8192 ? 8 : 16, waves = (D + 64 * E - 1) / (64 * E), each = waves == 3 ? 4 : waves < 8 ? 8 / waves : 1;
    return LnShape{0, E, waves, each, waves * each * 64};
}

// Workgroups: what the chip holds beside each other, 24 waves a compute unit at the most (each writes a line of partial sums, so there are no more of them).
// `fit`: workgroups that a compute unit holds, by the kernel's registers; unknown (the workspace's size): 24 waves.  A grid that a part of the
// compute units hold twice and the others once leaves those idle for half of the time: 84 against 90 us for 87381 x 384 fp32.
int ln_bwd_blocks(int64_t rows, int D, int fit) {
    const LnShape s = ln_shape(D);
    const int cap = 24 * 64 / s.block > 1 ? 24 * 64 / s.block : 1, per_cu = fit > 0 && fit < cap ? fit : cap;
    const int64_t want = (rows + s.each - 1) / s.each, most = 256 * per_cu;
    return (int)(want < most ? want : most);
}

// one kernel's workgroups a compute unit, asked for once for each workgroup size
struct Fit { std::atomic<int> waves[17]; };
int ln_fit(Fit& f, const void* kernel, int block, int shared) {
    const int known = f.waves[block / 64].load(std::memory_order_relaxed);
    if (known) return known;
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, block, shared) != hipSuccess || n < 1) {
        (void)hipGetLastError();
        n = 1;
    }
    f.waves[block / 64].store(n, std::memory_order_relaxed);
    return n;
}

template <typename T> hipError_t ln_bwd_launch(const LnBwd& args, bool res, bool drop, int* lines, hipStream_t st) {
    const LnShape s = ln_shape(args.D);
    LnBwd a = args;
    a.waves = s.waves;
    a.each = s.each;
    const int weights = s.E > 8 ? s.waves * 64 * s.E * 4 : 0, join = s.G ? 256 * Vec<T>::N * 4 : s.each > 1 ? s.waves * 64 * Vec<T>::N * 4 : 0;
    const int shared = weights > join ? weights : join;
#define RUN(G_, E_, RES_, DROP_, TAIL_) do { \
        const void* kernel = (const void*)ln_bwd_kernel<T, G_, E_, RES_, DROP_, TAIL_>; \
        static YpLdsAttr lds_limit; \
        static Fit fit; \
        if (shared > 32768) { \
            const hipError_t e = yp_set_max_lds(lds_limit, kernel, LN_WIDEST * 4); \
            if (e != hipSuccess) return e; \
        } \
        *lines = ln_bwd_blocks(a.rows, a.D, ln_fit(fit, kernel, s.block, shared)); \
        ln_bwd_kernel<T, G_, E_, RES_, DROP_, TAIL_><<<*lines, s.block, shared, st>>>(a); \
        return hipGetLastError(); \
    } while (0)
#define ENDS(G_, E_, RES_, DROP_) \
    if (a.D % Vec<T>::N == 0) RUN(G_, E_, RES_, DROP_, WHOLE); \
    else if (a.D > Vec<T>::N) RUN(G_, E_, RES_, DROP_, CUT); \
    else if constexpr (G_ == 4) RUN(G_, E_, RES_, DROP_, SHORT);
#define SHAPE(G_, E_) if (s.G == G_ && s.E == E_) { if (!res && !drop) { ENDS(G_, E_, false, false) } else if (!drop) { ENDS(G_, E_, true, false) } \
        else if (!res) { ENDS(G_, E_, false, true) } else { ENDS(G_, E_, true, true) } }
    LN_SHAPES(SHAPE)
#undef SHAPE
#undef ENDS
#undef RUN
    return hipErrorInvalidValue;                    // (not reached: the shapes and row ends above are all there are)
}

}  // namespace

extern "C" size_t yp_layer_norm_bwd_workspace_bytes(int64_t rows, int D, int dtype) {
    if (rows <= 0 || D < 1 || D > yp_layer_norm_max_width(dtype)) return 0;
    return (size_t)ln_bwd_blocks(rows, D, 0) * 2 * (size_t)D * sizeof(float);
}

extern "C" int yp_layer_norm_bwd(const YpLayerNormDesc* d, void* stream) {
    YP_REQUIRE(d != nullptr, "yp_layer_norm_bwd: no descriptor");
    YP_REQUIRE(ln_types(d), "yp_layer_norm_bwd: types %d / %d", d->dtype, d->wdtype);
    YP_REQUIRE(d->rows >= 0 && d->D >= 1 && d->D <= LN_WIDEST, "yp_layer_norm_bwd: %lld rows of %d", (long long)d->rows, d->D);
    const bool sums = d->dweight != nullptr || d->dbias != nullptr;
    hipStream_t st = (hipStream_t)stream;
    int lines = 0;
    if (d->rows > 0) {
        LnBwd a{};
        YP_REQUIRE(drop_parameters(d->p, &a.threshold, &a.scale), "yp_layer_norm_bwd: a dropout rate of %g", d->p);
        const bool res = d->dz != nullptr, drop = a.threshold != 0;
        YP_REQUIRE(d->x && d->dy && (d->stats || (d->mean && d->rstd)) && (!drop || (d->dx && d->dres)), "yp_layer_norm_bwd: a buffer is missing");
        YP_REQUIRE(d->x_stride >= 0 && d->dy_stride >= 0 && d->dz_stride >= 0, "yp_layer_norm_bwd: negative stride");
        if (sums && (d->workspace == nullptr || d->workspace_bytes < yp_layer_norm_bwd_workspace_bytes(d->rows, d->D, d->dtype))) {
            yp_set_error("yp_layer_norm_bwd: workspace of %zu bytes, %zu needed", d->workspace_bytes, yp_layer_norm_bwd_workspace_bytes(d->rows, d->D, d->dtype));
            return YP_ERR_WORKSPACE;
        }
        a.z = d->x; a.dy = d->dy; a.dz = d->dz; a.weight = d->weight; a.with_rest = d->stats != nullptr;
        a.mean = a.with_rest ? d->stats : d->mean; a.rstd = a.with_rest ? d->stats + 1 : d->rstd; a.rest = a.with_rest ? d->stats + 2 : d->mean;
        a.dres = d->dres; a.dx = d->dx;
        a.partial = sums ? (float*)d->workspace : nullptr;
        a.rows = d->rows; a.zs = d->x_stride; a.dys = d->dy_stride; a.dzs = d->dz_stride; a.D = d->D; a.inv_width = 1.0f / (float)d->D; a.w32 = d->wdtype == YP_F32;
        a.seed = d->seed; a.offset = d->offset; a.rng = d->rng;
        YP_CHECK_HIP(d->dtype == YP_F16 ? ln_bwd_launch<_Float16>(a, res, drop, &lines, st) : d->dtype == YP_BF16 ? ln_bwd_launch<__bf16>(a, res, drop, &lines, st)
                                                                                             : ln_bwd_launch<float>(a, res, drop, &lines, st));
    }
    if (sums) {
        const int grid = (2 * d->D + 31) / 32;
        const float* p = (const float*)d->workspace;
        if (d->wdtype == YP_F32) ln_columns_kernel<float><<<grid, 1024, 0, st>>>(p, lines, d->D, (float*)d->dweight, (float*)d->dbias);
        else if (d->wdtype == YP_F16) ln_columns_kernel<_Float16><<<grid, 1024, 0, st>>>(p, lines, d->D, (_Float16*)d->dweight, (_Float16*)d->dbias);
        else ln_columns_kernel<__bf16><<<grid, 1024, 0, st>>>(p, lines, d->D, (__bf16*)d->dweight, (__bf16*)d->dbias);
        YP_CHECK_HIP(hipGetLastError());
    }
    return YP_OK;
}
