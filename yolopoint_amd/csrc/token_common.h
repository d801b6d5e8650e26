// What the token operators share (csrc/token.hip, csrc/norm.hip, csrc/norm_bwd.hip): 16-byte pieces of rows, sums over lanes, dropout's random bits.
// Compiled with -ffp-contract=off: every fused multiply-add is written as one, so that the kernels for different operands and row shapes round alike
// (the fused operator's norm is the plain norm of its sum bit for bit).
#pragma once
#include "yp_internal.h"

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

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

// elements c .. c + N - 1 of a row of D elements in two steps, so that a row can be fetched long before it is used: `settle` is the first to touch
// the loaded registers; it leaves zeros behind the row's end
template <typename T, Tail TAIL> __device__ __forceinline__ Vec<T> fetch_vec(const T* row, int c, int D) {
    constexpr int N = Vec<T>::N;
    Vec<T> v;
    if constexpr (TAIL == SHORT) {
#pragma unroll
        for (int j = 0; j < N; ++j) v.e[j] = row[min(c + j, D - 1)];
    } else {
        __builtin_memcpy(&v, row + min(c, D - N), 16);
    }
    return v;
}
template <typename T, Tail TAIL> __device__ __forceinline__ Vec<T> settle(Vec<T> v, int c, int D) {
    constexpr int N = Vec<T>::N;
    if constexpr (TAIL == SHORT) {
#pragma unroll
        for (int j = 0; j < N; ++j) v.e[j] = c + j < D ? v.e[j] : (T)0.f;
    } else {
        u32x4 r;
        __builtin_memcpy(&r, &v, 16);
        const unsigned back = (unsigned)(c - min(c, D - N)) * sizeof(T);        // bytes to move down
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
template <typename T, Tail TAIL> __device__ __forceinline__ Vec<T> load_vec(const T* row, int c, int D) { return settle<T, TAIL>(fetch_vec<T, TAIL>(row, c, D), c, D); }

// elements c .. of a row of D elements (none behind its end)
template <typename T, Tail TAIL> __device__ __forceinline__ void store_vec(T* row, int c, int D, const Vec<T>& v) {
    constexpr int N = Vec<T>::N;
    T* p = row + c;
    if constexpr (TAIL == WHOLE) {
        if (c < D) __builtin_memcpy(p, &v, 16);
    } else {
        const int n = D - c;
        if (n >= N) {
            __builtin_memcpy(p, &v, 16);
        } else if (n > 0) {                         // the set bits of n, largest first
            u32x4 r;
            __builtin_memcpy(&r, &v, 16);
            if (n & (N / 2)) {
                const u32x2 h = {r.x, r.y};
                __builtin_memcpy(p, &h, 8);
                p += N / 2;
                r.x = r.z; r.y = r.w;
            }
            if (n & (N / 4)) {
                const unsigned h = r.x;
                __builtin_memcpy(p, &h, 4);
                p += N / 4;
                r.x = r.y;
            }
            if constexpr (sizeof(T) == 2) {
                if (n & 1) {
                    const unsigned short h = (unsigned short)r.x;
                    __builtin_memcpy(p, &h, 2);
                }
            }
        }
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
template <typename T> __device__ __forceinline__ Vec<T> to_vec(float (&f)[Vec<T>::N]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    Vec<T> v;
    if constexpr (sizeof(T) == 4) {
        __builtin_memcpy(&v, f, 16);
    } else {
        typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < Vec<T>::N; j += 2) {    // (two at a time: the packed conversion)
            if constexpr (__is_same(T, _Float16)) asm("" : "+v"(f[j]), "+v"(f[j + 1]));
            const t2 h = __builtin_convertvector((f2){f[j], f[j + 1]}, t2);
            v.e[j] = h.x;
            v.e[j + 1] = h.y;
        }
    }
    return v;
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

// ------------------------------------------------------------------------------------------------------------------ dropout
// Element i of a tensor (flat, row-major) is kept where half i % 8 of the 128 bits that Philox4x32-10 gives for the counter (i / 8, offset) is
// >= threshold = round(65536 p).  16 bits an element: the rate moves in steps of 2^-16, and one call of the generator (some 85
// instructions) serves eight elements.
struct Drop {
    unsigned long long seed, offset;
    unsigned threshold;
    float scale;
};

__device__ __forceinline__ Drop drop_state(unsigned long long seed, unsigned long long offset, const int64_t* __restrict__ rng, unsigned threshold, float scale) {
    if (rng != nullptr) { seed = (unsigned long long)rng[0]; offset = (unsigned long long)rng[1]; }
    return Drop{seed, offset, threshold, scale};
}

// The bits of N = 4 or 8 elements from flat index i on, two to a word.  STRADDLE: i may stand anywhere, so that the elements may need the next counter's
// words too (rows of odd widths).  Those are what the next lane has just made of the counter after this one, so they come from there; `edge`: this
// lane is the last of its row's lanes in the wave; `left`: elements of the row from i on.  A wave that holds one row (WAVE) makes the words of its last
// lane's next counter on the scalar unit, beside the other waves' vector work.
template <int N, bool STRADDLE, bool WAVE, bool MAD> __device__ __forceinline__ void drop_bits(const Drop& d, unsigned long long i, bool edge, int left, unsigned (&w)[N / 2]) {
    const unsigned sh = WAVE && N == 8 ? __builtin_amdgcn_readfirstlane((unsigned)i & 7u) : (unsigned)i & 7u;       // (chunks of 8: the same for a row)
    const YpU4 a = yp_philox4x32<false, MAD>(d.seed, i >> 3, d.offset);
    if constexpr (!STRADDLE) {                      // i % N == 0
        if constexpr (N == 8) { w[0] = a.x; w[1] = a.y; w[N / 2 - 2] = a.z; w[N / 2 - 1] = a.w; }
        else { w[0] = sh ? a.z : a.x; w[1] = sh ? a.w : a.y; }
    } else {
        auto from_next = [](unsigned v) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x130, 0xf, 0xf, true); };     // (the wave shifted by a lane)
        YpU4 b{from_next(a.x), from_next(a.y), from_next(a.z), from_next(a.w)};
        if (__ballot(edge && left > 0 && (int)sh + min(N, left) > 8)) {
            YpU4 s;
            if constexpr (WAVE) {
                const unsigned lo = __builtin_amdgcn_readlane((unsigned)(i >> 3), 63), hi = __builtin_amdgcn_readlane((unsigned)(i >> 35), 63);
                s = yp_philox4x32<true, MAD>(d.seed, (((unsigned long long)hi << 32) | lo) + 1, d.offset);
            } else {
                s = yp_philox4x32<false, MAD>(d.seed, (i >> 3) + 1, d.offset);
            }
            b.x = edge ? s.x : b.x; b.y = edge ? s.y : b.y; b.z = edge ? s.z : b.z; b.w = edge ? s.w : b.w;
        }
        // the eight words moved down by sh halves
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
}

template <int N> __device__ __forceinline__ bool drop_kept(const Drop& d, const unsigned (&w)[N / 2], int j) {
    return ((j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu) >= d.threshold;
}

// out = res + (kept ? x * scale : 0): one fused multiply-add in fp32, rounded to T
template <typename T, bool DROP, bool STRADDLE = false, bool WAVE = false>
__device__ __forceinline__ void drop_add(const Drop& d, unsigned long long i, const Vec<T>& x, const Vec<T>& res, Vec<T>& out, bool edge = false, int left = 0) {
    constexpr int N = Vec<T>::N;
    unsigned w[N / 2];
    if constexpr (DROP) drop_bits<N, STRADDLE, WAVE, false>(d, i, edge, left, w);
    float s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float r = (float)res.e[j];
        if constexpr (DROP) s[j] = drop_kept<N>(d, w, j) ? fmaf((float)x.e[j], d.scale, r) : r;
        else s[j] = r + (float)x.e[j];
    }
    out = to_vec<T>(s);
}

// out = kept ? v * scale : 0.  MAD: the generator's products as 64-bit multiply-adds, for eight 16-bit elements, which its instructions bound (backward of
// 31956 x 2100 bf16 224 us against 239, 86369 x 777 192 against 203, 13421 x 5000 132 against 150; at worst 16372 x 4099 245 against 235; dropout of
// 8.4 M elements 8.4 against 8.9).  As halves where the pairs of registers cost more than the products: four fp32 elements (8186 x 4099: 148 against
// 157), odd rows of more than 8192 features (5436 x 12345 bf16: 257 against 280, 8201 features 279 against 308), and drop_add (forward of 16372 x 4099
// bf16: 159 against 187).
template <typename T, bool STRADDLE = false, bool WAVE = false, bool MAD = sizeof(T) == 2>
__device__ __forceinline__ void drop_only(const Drop& d, unsigned long long i, const float (&v)[Vec<T>::N], Vec<T>& out, bool edge = false, int left = 0) {
    constexpr int N = Vec<T>::N;
    unsigned w[N / 2];
    drop_bits<N, STRADDLE, WAVE, MAD>(d, i, edge, left, w);
    float s[N];
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = drop_kept<N>(d, w, j) ? v[j] * d.scale : 0.f;
    out = to_vec<T>(s);
}

int drop_parameters(double p, unsigned* threshold, float* scale) {
    if (!(p >= 0.0 && p <= 1.0)) return 0;
    *threshold = (unsigned)(p * 65536.0 + 0.5);
    *scale = *threshold < 65536u ? (float)(65536.0 / (65536.0 - (double)*threshold)) : 0.f;
    return 1;
}

}  // namespace
