// The e4m3 block quantizers' arithmetic on eight elements of a lane
// (bcjr_fp8.cu has the definition), for bcjr_fp8.cu and bcjr_mm.cuh.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace bcjr {
namespace mm {

constexpr float kMax = 448.f;

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float block_amax(float a) { return max_nan(a, 0x1p-100f); }
__device__ __forceinline__ float block_scale(float amax) { return __fmul_rn(amax, 1.f / kMax); }
__device__ __forceinline__ float block_inv(float amax) { return __fmul_rn(kMax, __frcp_rn(amax)); }

template <typename T> __device__ __forceinline__ void load8(const T *p, float (&v)[8]);
template <> __device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4 a = __ldcs(reinterpret_cast<const float4 *>(p));
    const float4 b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T> __device__ __forceinline__ void unpack8(uint4 u, float (&v)[8]);
template <> __device__ __forceinline__ void unpack8<__nv_bfloat16>(uint4 u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <> __device__ __forceinline__ void unpack8<__half>(uint4 u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <> __device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) {
    unpack8<__nv_bfloat16>(__ldcs(reinterpret_cast<const uint4 *>(p)), v);
}
template <> __device__ __forceinline__ void load8(const __half *p, float (&v)[8]) {
    unpack8<__half>(__ldcs(reinterpret_cast<const uint4 *>(p)), v);
}

__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
    return m;
}
__device__ __forceinline__ uint2 to_e4m3(const float (&v)[8], float inv) {
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
            : "=h"(h[i])
            : "f"(__fmul_rn(v[2 * i + 1], inv)), "f"(__fmul_rn(v[2 * i], inv)));
    return make_uint2(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16);
}

}  // namespace mm
}  // namespace bcjr
