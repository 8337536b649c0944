// The codec of compressed rows: feature_len one-byte codes (int8 or e4m3), one fp32 scale, zeros up to a multiple of 16 bytes.
#pragma once
#include "common.cuh"

#include <cuda_fp8.h>

namespace legion {

__host__ __device__ __forceinline__ int64_t code_row_bytes(int64_t feature_len) { return (feature_len + 4 + 15) / 16 * 16; }

// Four codes of one row, first value in the low byte.  SAFE: any row; otherwise a row whose values and whose factor
// are finite, where |x * inv| < 128 and the nearest integer is what adding 1.5 * 2^23 leaves in the low bits.
template <int CODEC, bool SAFE>
__device__ __forceinline__ uint32_t encode4(const float4 &x, float inv)
{
    const float p[4] = { __fmul_rn(x.x, inv), __fmul_rn(x.y, inv), __fmul_rn(x.z, inv), __fmul_rn(x.w, inv) };
    if (CODEC == LEGION_CODEC_INT8) {
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            q[i] = SAFE ? (uint32_t)max(-127, min(127, __float2int_rn(p[i]))) : __float_as_uint(__fadd_rn(p[i], 12582912.0f));
        return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(p[0], p[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(p[2], p[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

__device__ __forceinline__ float max_nan(float a, float b)   // NaN when either is
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

}  // namespace legion
