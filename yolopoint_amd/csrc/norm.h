// What the two passes of the layer norm share (csrc/norm.hip, csrc/norm_bwd.hip).
//
// A row of D features is held in the registers of its threads, E = 8 | 16 features each in chunks of 16 bytes (thread t of G: chunks t, t + G, ...):
// neighbouring threads read neighbouring 16 bytes, and the weights of a thread's columns stay where they are over all of its rows.  G <= 64: one row
// or several a wave, sums without LDS.  G = 0: one wave or more a row, as many as it fills; their sums meet in LDS.
#pragma once
#include "token_common.h"

namespace {

constexpr int LN_WIDEST = 1024 * 16;

template <int G> __device__ __forceinline__ int row_in_block() {
    if constexpr (G == 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / 64);     // (a wave's row: its addresses on the scalar unit)
    return G ? threadIdx.x / G : 0;
}

// a value that is the same in the whole wave, on the scalar unit (it frees a register of each lane)
__device__ __forceinline__ float of_wave(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }

// whether a thread is the last of its row's lanes in its wave
template <int G> __device__ __forceinline__ bool last_lane() { return ((threadIdx.x + 1) & (G && G < 64 ? G - 1 : 63)) == 0; }

// Sums over the threads of a row: G <= 64 neighbouring lanes, or (G = 0) `of` waves from wave `from` on (default: the workgroup's).  Calls alternate between
// two areas of LDS, so that one barrier a call is enough: a wave writes an area again only behind the barrier of the call on the other one, which
// every wave passes after reading the first.
template <int G> __device__ __forceinline__ void row_sum2(float& a, float& b, float2* area, int from = 0, int of = 0) {
    if constexpr (G > 0) {
        a = lanes_sum<G>(a);
        b = lanes_sum<G>(b);
    } else {
        a = lanes_sum<64>(a);
        b = lanes_sum<64>(b);
        if ((threadIdx.x & 63) == 0) area[threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        const int lane = threadIdx.x & 15, n = of ? of : blockDim.x >> 6;               // (16 waves at the most: each row of lanes adds them)
        const float2 s = area[min(from + lane, 15)];
        a = lanes_sum<16>(lane < n ? s.x : 0.f);
        b = lanes_sum<16>(lane < n ? s.y : 0.f);
    }
}
template <int G> __device__ __forceinline__ float row_sum(float a, float2* area) {
    if constexpr (G > 0) return lanes_sum<G>(a);
    a = lanes_sum<64>(a);
    if ((threadIdx.x & 63) == 0) area[threadIdx.x >> 6].x = a;
    __syncthreads();
    const int lane = threadIdx.x & 15;
    return lanes_sum<16>(lane < (int)(blockDim.x >> 6) ? area[lane].x : 0.f);
}

bool ln_types(const YpLayerNormDesc* d) {
    return (d->dtype == YP_F16 || d->dtype == YP_BF16 || d->dtype == YP_F32) && (d->wdtype == YP_F32 || d->wdtype == d->dtype);
}

}  // namespace
