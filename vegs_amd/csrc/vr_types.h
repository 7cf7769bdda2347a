// vr_types.h -- the storage types of gradients and tables (VrDataType) and their conversions; all arithmetic is fp32.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vr {

struct bf16 { uint16_t bits; };

__device__ __forceinline__ float load_f32(const float* p) { return *p; }
__device__ __forceinline__ float load_f32(const bf16* p) { return __uint_as_float((uint32_t)p->bits << 16); }
__device__ __forceinline__ float load_f32(const __half* p) { return __half2float(*p); }

// rounded once, to nearest with ties to even; NaN stays NaN
__device__ __forceinline__ void store_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_f32(bf16* p, float x)
{
    const uint32_t u = __float_as_uint(x);
    p->bits = (u & 0x7fffffffu) > 0x7f800000u ? (uint16_t)((u >> 16) | 0x40u) : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ void store_f32(__half* p, float x) { *p = __float2half_rn(x); }

}  // namespace vr
