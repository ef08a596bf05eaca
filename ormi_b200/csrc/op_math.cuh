// Device helpers shared by the transformer-block kernels: conversions between the storage types and fp32, reductions in a
// fixed order.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace ormi_b200 {

using bf16 = __nv_bfloat16;
using e4m3 = __nv_fp8_e4m3;

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<bf16>(bf16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ e4m3 from_f32<e4m3>(float v) { e4m3 r; r.__x = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); return r; }

__device__ __forceinline__ float bf16_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum / maximum over the block in warp order; every thread gets it.  `box` holds 33 floats of shared memory.
__device__ __forceinline__ float block_sum(float v, float* box) {
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, n = (blockDim.x + 31) >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) box[warp] = v;
    __syncthreads();
    float t = 0.f;
    for (int w = 0; w < n; ++w) t += box[w];
    return t;
}
// Largest magnitude as the bits of |v|: ordered like the values, and a NaN is above everything, so it is not lost.
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float block_max_mag(uint32_t m, uint32_t* box) {
    m = __reduce_max_sync(0xffffffffu, m);
    const int warp = threadIdx.x >> 5, n = (blockDim.x + 31) >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) box[warp] = m;
    __syncthreads();
    for (int w = 0; w < n; ++w) m = max(m, box[w]);
    return __uint_as_float(m);
}

}  // namespace ormi_b200
