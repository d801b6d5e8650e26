// Layer norm over the rows of a token tensor, forward: alone, or behind residual + dropout in the same pass.  Bound by HBM: a row is read once, stays in
// registers while its statistics are formed, and is written once.
#include "norm.h"

namespace {

struct LnFwd {
    const void *x, *res, *weight, *bias;
    void *z, *y;
    float* stats;                                   // of a row from row * line on: the mean, 1 / deviation (`rstd` elements on) and the mean's rest (two on):
    int64_t rows, xs, rs, rstd;                     // as many of them as `parts`
    int D, line, parts;
    float eps, width, inv_width;                    // D and 1 / D (as arguments: no register of the lanes)
    bool w32;
    unsigned long long seed, offset;
    const int64_t* rng;
    unsigned threshold;
    float scale;
};

// mean = sum x / D;  var = sum (x - mean)^2 / D;  y = (x - mean) / sqrt(var + eps) w + b.  Behind the mean, delta is what rounding left of it, and is taken
// off as well: where a row hardly varies (a constant one has rstd = 316), that rounding would become the result.
//   f32, f16   delta = sum (x - mean) / D: a fp32 row of mean 4096 and deviation 1 keeps 1e-7 instead of 1e-3, a f16 row of mean 1000 and deviation 1/4 (one
//              step of its type) 1e-7 instead of its half step
//   bf16       delta = (sum x - mean D) / D, what the division left, for nothing a value (the sum over x - mean takes 10 % at 1091 features): the sum itself
//              is exact in 24 bits while no value is below 2^-16 D of the largest, as 8 bits a value and D <= 2^14 of them fit.  Where one is, it stands
//              apart from the largest, the deviation is half of that / sqrt(D) at least, and the sum's rounding moves y by 4e-4 at the most.
// (16-bit rows over several waves: held to the registers of five waves a SIMD, which the compiler misses by three with dropout at odd widths: 4100 features
// 143 us against 170.)
// The next row is on its way while this one is worked on (the first before the weights are read): its registers are not touched before its turn, or the
// wait for them would stand right behind the loads.
// Measured, 128 MiB a tensor, with the statistics: 44 - 67 us for widths 16 .. 16384 (4.0 - 6.2 TB/s), with residual and dropout 100 - 130 us (4.1 - 5.4; a
// large copy: 5.2 - 5.4); widths just over a border with dropout are bound by their instructions (bf16 4100: 142 us, 4099: 158, 12345: 160).
template <typename T, int G, int E, bool RES, bool DROP, Tail TAIL>
__global__ __launch_bounds__(G ? 256 : 1024, G == 0 && sizeof(T) == 2 ? 5 : 1) void ln_fwd_kernel(const LnFwd a) {
    constexpr int N = Vec<T>::N, NC = E / N, ROWS = G ? 256 / G : 1;
    constexpr bool FINE = !__is_same(T, __bf16);
    __shared__ float2 sh[2][16];
    const T *x = (const T*)a.x, *res = (const T*)a.res;
    T *z = (T*)a.z, *y = (T*)a.y;
    const int threads = G ? G : blockDim.x, t = G ? threadIdx.x % G : threadIdx.x;
    const Drop d = drop_state(a.seed, a.offset, a.rng, a.threshold, a.scale);
    int c[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) c[k] = (t + k * threads) * N;
    const int64_t first = (int64_t)blockIdx.x * ROWS + row_in_block<G>(), step = (int64_t)gridDim.x * ROWS;
    Vec<T> nx[NC], nr[NC];
    const T *px = x + min(first, a.rows - 1) * a.xs, *pr = RES ? res + min(first, a.rows - 1) * a.rs : nullptr;
    auto fetch = [&]() {
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            nx[k] = fetch_vec<T, TAIL>(px, c[k], a.D);
            if constexpr (RES) nr[k] = fetch_vec<T, TAIL>(pr, c[k], a.D);
        }
    };
    fetch();
    float w[NC][N], b[NC][N];
#pragma unroll
    for (int k = 0; k < NC; ++k) { load_weights<T, TAIL>(a.weight, a.w32, c[k], a.D, 1.f, w[k]); load_weights<T, TAIL>(a.bias, a.w32, c[k], a.D, 0.f, b[k]); }
    for (int64_t row = first; row < a.rows; row += step) {
        Vec<T> v[NC];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            v[k] = settle<T, TAIL>(nx[k], c[k], a.D);
            if constexpr (RES) {
                const Vec<T> r = settle<T, TAIL>(nr[k], c[k], a.D), s = v[k];
                if (DROP && G == 0 && __ballot(c[k] < a.D) == 0ull) continue;       // (a wave behind the row's end makes no random numbers)
                drop_add<T, DROP, TAIL != WHOLE, G == 0 || G == 64>(d, (unsigned long long)row * a.D + c[k], s, r, v[k], last_lane<G>(), a.D - c[k]);
                store_vec<T, TAIL>(z + row * a.D, c[k], a.D, v[k]);
            }
        }
        if (row + step < a.rows) {
            px += step * a.xs;
            if (RES) pr += step * a.rs;
            fetch();
        }
        float f[NC][N], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j) { f[k][j] = (float)v[k].e[j]; s1 += f[k][j]; }
        const float sum = row_sum<G>(s1, sh[0]), mean = sum * a.inv_width;
        s1 = 0.f;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            const float m = c[k] < a.D ? mean : 0.f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                f[k][j] -= m;
                if constexpr (TAIL != WHOLE) f[k][j] = c[k] + j < a.D ? f[k][j] : 0.f;
                if constexpr (FINE) s1 += f[k][j];
                s2 = fmaf(f[k][j], f[k][j], s2);
            }
        }
        if constexpr (FINE) row_sum2<G>(s1, s2, sh[1]);
        else s2 = row_sum<G>(s2, sh[1]);
        const float delta = (FINE ? s1 : fmaf(-mean, a.width, sum)) * a.inv_width;
        float var = fmaf(-delta, delta, s2 * a.inv_width);
        var = var < 0.f ? 0.f : var;                // (not fmaxf: a NaN stays one)
        const float rstd = rsqrtf(var + a.eps), shift = -delta * rstd;
        // (Rows of a wave or less: one store by as many lanes, three take 70 us against 63 for bf16 rows of 16.  Wider ones: three by one lane, the other
        // way takes 138 us against 125 at 2100 features with dropout, and a branch for each 172; a rest that has no place is written under the mean.)
        const float nearest = mean + delta, rest = delta - (nearest - mean);            // (exact: |delta| is some steps of the mean)
        if constexpr (G != 0) {
            if (t < a.parts) a.stats[row * a.line + (t == 1 ? a.rstd : t)] = t == 0 ? nearest : t == 1 ? rstd : rest;
        } else if (a.parts != 0 && t == 0) {
            float* s = a.stats + row * a.line;
            s[a.line - 1] = rest;
            s[a.rstd] = rstd;
            s[0] = nearest;
        }
#pragma unroll
        for (int k = 0; k < NC; ++k) {
            float o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) o[j] = fmaf(fmaf(f[k][j], rstd, shift), w[k][j], b[k][j]);
            store_vec<T, TAIL>(y + row * a.D, c[k], a.D, to_vec<T>(o));
        }
    }
}

// The shape of a row: G threads with E features each, the first that holds it; G = 0: 64 * waves threads.  16 features a thread where 8 would need a
// second wave (513 .. 1024 features: no barrier.  65536 x 1024 bf16: 44.6 us against 47.5, 129055 x 520: 49 against 61), or more than four waves.
#define LN_SHAPES(X) X(4, 8) X(8, 8) X(16, 8) X(32, 8) X(64, 8) X(64, 16) X(0, 8) X(0, 16)
struct LnShape { int G, E, threads; };
LnShape ln_shape(int D) {
#define PICK(G_, E_) if (G_ && D <= G_ * E_) return LnShape{G_, E_, G_};
    LN_SHAPES(PICK)
#undef PICK
    const int E = D <= 2048 ? 8 : 16;
    return LnShape{0, E, (D + 64 * E - 1) / (64 * E) * 64};
}

template <typename T> hipError_t ln_fwd_launch(const LnFwd& a, bool res, bool drop, hipStream_t st) {
    const LnShape s = ln_shape(a.D);
    const int block = s.G ? 256 : s.threads;
    const int64_t per = s.G ? block / s.G : 1, want = (a.rows + per - 1) / per, most = 256 * 64 * 64 / block;     // (twice what the chip holds: the second half evens out)
    const int blocks = (int)(want < most ? want : most);
#define RUN(G_, E_, RES_, DROP_, TAIL_) do { ln_fwd_kernel<T, G_, E_, RES_, DROP_, TAIL_><<<blocks, block, 0, st>>>(a); return hipGetLastError(); } while (0)
#define ENDS(G_, E_, RES_, DROP_) \
    if (a.D % Vec<T>::N == 0) RUN(G_, E_, RES_, DROP_, WHOLE); \
    else if (a.D > Vec<T>::N) RUN(G_, E_, RES_, DROP_, CUT); \
    else if constexpr (G_ == 4) RUN(G_, E_, RES_, DROP_, SHORT);
#define SHAPE(G_, E_) if (s.G == G_ && s.E == E_) { if (!res) { ENDS(G_, E_, false, false) } else if (!drop) { ENDS(G_, E_, true, false) } else { ENDS(G_, E_, true, true) } }
    LN_SHAPES(SHAPE)
#undef SHAPE
#undef ENDS
#undef RUN
    return hipErrorInvalidValue;                    // (not reached: the shapes and row ends above are all there are)
}

}  // namespace

extern "C" int yp_layer_norm_max_width(int dtype) { return dtype == YP_F16 || dtype == YP_BF16 || dtype == YP_F32 ? LN_WIDEST : 0; }

extern "C" int yp_layer_norm_fwd(const YpLayerNormDesc* d, void* stream) {
    YP_REQUIRE(d != nullptr, "yp_layer_norm_fwd: no descriptor");
    YP_REQUIRE(ln_types(d), "yp_layer_norm_fwd: types %d / %d", d->dtype, d->wdtype);
    YP_REQUIRE(d->rows >= 0 && d->D >= 1 && d->D <= LN_WIDEST, "yp_layer_norm_fwd: %lld rows of %d", (long long)d->rows, d->D);
    if (d->rows == 0) return YP_OK;
    YP_REQUIRE(d->x && d->y && (d->res == nullptr || d->z) && (d->mean == nullptr) == (d->rstd == nullptr), "yp_layer_norm_fwd: a buffer is missing");
    YP_REQUIRE(d->x_stride >= 0 && d->res_stride >= 0, "yp_layer_norm_fwd: negative stride");
    LnFwd a{};
    YP_REQUIRE(drop_parameters(d->p, &a.threshold, &a.scale), "yp_layer_norm_fwd: a dropout rate of %g", d->p);
    YP_REQUIRE(d->res != nullptr || a.threshold == 0, "yp_layer_norm_fwd: dropout needs a residual");
    a.x = d->x; a.res = d->res; a.weight = d->weight; a.bias = d->bias; a.z = d->z; a.y = d->y;
    if (d->stats) { a.stats = d->stats; a.line = a.parts = 3; a.rstd = 1; }
    else if (d->mean) { a.stats = d->mean; a.line = 1; a.parts = 2; a.rstd = ((intptr_t)d->rstd - (intptr_t)d->mean) / (intptr_t)sizeof(float); }
    a.rows = d->rows; a.xs = d->x_stride; a.rs = d->res_stride; a.D = d->D; a.eps = d->eps; a.width = (float)d->D; a.inv_width = 1.0f / a.width; a.w32 = d->wdtype == YP_F32;
    a.seed = d->seed; a.offset = d->offset; a.rng = d->rng;
    hipStream_t st = (hipStream_t)stream;
    const bool res = d->res != nullptr, drop = a.threshold != 0;
    YP_CHECK_HIP(d->dtype == YP_F16 ? ln_fwd_launch<_Float16>(a, res, drop, st) : d->dtype == YP_BF16 ? ln_fwd_launch<__bf16>(a, res, drop, st) : ln_fwd_launch<float>(a, res, drop, st));
    return YP_OK;
}
