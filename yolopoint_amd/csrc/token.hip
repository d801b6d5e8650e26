// Operators on tokens (rows of features: keypoint descriptors, descriptor-map cells, sequence entries): dropout from a counter-based generator and rotary
// positions (layer norm: csrc/norm.hip, csrc/norm_bwd.hip).  All of them are bound by HBM: each reads its inputs once and writes its outputs once;
// sums, statistics and angles are held in 32 bits or more.
#include "token_common.h"

namespace {

// Bound by HBM: 67.1 M bf16 elements take 42 us (6.4 TB/s), with a residual 74 us (5.5 TB/s; a large copy 5.2 - 5.4).  Eight bf16 elements a thread are
// one call of the generator (some 85 instructions), four fp32 ones use half of theirs, for the same 16 bytes: 40.4 us for the same 256 MB.
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
        store_vec<T, TAIL>(y + at, c, D, o);
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

// Bound by HBM from two heads a thread on: 4 x 8192 tokens of 20 x 128 bf16 (335 MB moved) take 65 us, 5.2 TB/s, as a large copy.  A single head of bf16
// is bound by its cosines instead (some 40 instructions a pair, half of them 64-bit: 3.8 TB/s).  The angles are formed here and not read from a table of
// cosines: such a table is another 2 x 4 bytes a pair and token, as much as one bf16 head moves, and ends at the longest context it was made for.
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
            if (turns) {
                float fu[N], fv[N];
                if (a.interleaved) {
#pragma unroll
                    for (int j = 0; j < N / 2; ++j) {
                        const float x0 = (float)u.e[2 * j], x1 = (float)u.e[2 * j + 1], y0 = (float)v.e[2 * j], y1 = (float)v.e[2 * j + 1];
                        fu[2 * j] = fmaf(x0, cs[j], -(x1 * sn[j]));
                        fu[2 * j + 1] = fmaf(x1, cs[j], x0 * sn[j]);
                        fv[2 * j] = fmaf(y0, cs[j + N / 2], -(y1 * sn[j + N / 2]));
                        fv[2 * j + 1] = fmaf(y1, cs[j + N / 2], y0 * sn[j + N / 2]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float x0 = (float)u.e[j], x1 = (float)v.e[j];
                        fu[j] = fmaf(x0, cs[j], -(x1 * sn[j]));
                        fv[j] = fmaf(x1, cs[j], x0 * sn[j]);
                    }
                }
                u = to_vec<T>(fu);
                v = to_vec<T>(fv);
            }
            store_vec<T, TAIL>(out + s0, c0, len, u);
            store_vec<T, TAIL>(out + s1, c1, len, v);
        }
    }
}

}  // namespace

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
    // (a thread's next head is its head + up to 256, in 32 bits)
    YP_REQUIRE((int64_t)d->Hq + d->Hk <= (int64_t)1 << 30 && (int64_t)d->B * d->T * ((int64_t)d->Hq + d->Hk) < (int64_t)1 << 53, "yp_rotary: %d + %d heads of %d x %d tokens", d->Hq, d->Hk, d->B, d->T);
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
    // heads beside each other: all of them while even that does not fill the chip (64 tokens of 20 x 128 bf16: 3.8 us against 5.2 with four to a thread),
    // else four to a thread, which share its cosines (4096 tokens: 10.8 us against 17.6; the two meet at some 150 thousand threads)
    const bool few = (int64_t)a.tokens * H * chunks <= 256 * 512;
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
