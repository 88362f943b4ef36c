// What the decoding kernels share: loads of a lane's consecutive elements and the reduction that leaves each lane with one total.
#pragma once

#include "kda_common.cuh"

namespace kda {

template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = ldf(p + i);
}
template <>
__device__ __forceinline__ void load_n<__nv_bfloat16, 4>(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(r.x << 16); v[1] = __uint_as_float(r.x & 0xffff0000u);
    v[2] = __uint_as_float(r.y << 16); v[3] = __uint_as_float(r.y & 0xffff0000u);
}
template <>
__device__ __forceinline__ void load_n<float, 4>(const float* p, float (&v)[4]) {
    const float4 r = *reinterpret_cast<const float4*>(p);
    v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
}

// vec: the caller's rows start on a four-element boundary
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, float (&v)[N], int vec) {
    if (vec) {
        load_n(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = ldf(p + i);
    }
}

// Sums val[0..M) over the LD lanes that differ in the given lane bits (bit0, 2 bit0, ..., LD / 2 * bit0), halving the
// number of values a lane carries at every level: afterwards val[0] of a lane is the total of value `which`
// (the lane bits read from the lowest level up as the most significant bit of the index first).
template <int M, int LD, int BIT0>
struct TransposeSum {
    static __device__ __forceinline__ void run(float (&val)[M], int lane, int& which) {
        if constexpr (LD > 1) {
            const bool up = lane & BIT0;
            if constexpr (M > 1) {
                float half[M / 2];
#pragma unroll
                for (int i = 0; i < M / 2; ++i) {
                    const float keep = up ? val[M / 2 + i] : val[i], send = up ? val[i] : val[M / 2 + i];
                    half[i] = keep + __shfl_xor_sync(0xffffffffu, send, BIT0);
                }
                which = 2 * which + (up ? 1 : 0);
                TransposeSum<M / 2, LD / 2, 2 * BIT0>::run(half, lane, which);
                val[0] = half[0];
            } else {
                val[0] += __shfl_xor_sync(0xffffffffu, val[0], BIT0);
                TransposeSum<1, LD / 2, 2 * BIT0>::run(val, lane, which);
            }
        }
    }
};

}  // namespace kda
