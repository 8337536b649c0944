// Rows of fp32 / fp16 / bf16 elements: vectors of VE elements moved by the widest loads that fit, arithmetic in fp32.
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <initializer_list>

namespace legion {

constexpr int kSms = 148;  // what grids are sized for

// The call's device for as long as the call takes; the caller's current device is put back.
struct OnDevice {
    int before = -1;
    cudaError_t err;
    explicit OnDevice(int dev)
    {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != dev) err = cudaSetDevice(dev);
        else before = -1;
    }
    ~OnDevice() { if (before >= 0) cudaSetDevice(before); }
};

__host__ __device__ __forceinline__ int dtype_bytes(int dtype) { return dtype == LEGION_F32 ? 4 : 2; }
__host__ __forceinline__ bool dtype_known(int dtype) { return dtype >= LEGION_F32 && dtype <= LEGION_BF16; }

template <int BYTES> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<8> { typedef uint2 type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<2> { typedef uint16_t type; };

// VE elements as they lie in memory, in words of at most 16 bytes.
template <typename T, int VE>
struct Vec {
    static constexpr int kBytes = VE * (int)sizeof(T);
    static constexpr int kWord = kBytes > 16 ? 16 : kBytes;
    static constexpr int kWords = kBytes / kWord;
    typedef typename Raw<kWord>::type word;
    union {
        word w[kWords];
        T e[VE];
    };
    __device__ __forceinline__ Vec() {}
    __device__ __forceinline__ void load(const T *p)
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const word *>(p)[i];
    }
    __device__ __forceinline__ void load_stream(const T *p)  // read once
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = __ldcs(reinterpret_cast<const word *>(p) + i);
    }
    __device__ __forceinline__ void store(T *p) const
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) reinterpret_cast<word *>(p)[i] = w[i];
    }
    __device__ __forceinline__ void store_stream(T *p) const
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) __stcs(reinterpret_cast<word *>(p) + i, w[i]);
    }
    __device__ __forceinline__ void zero()
    {
#pragma unroll
        for (int i = 0; i < VE; ++i) e[i] = T(0.0f);
    }
    __device__ __forceinline__ float get(int i) const;
    __device__ __forceinline__ void set(const float *x);
};

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T, int VE>
__device__ __forceinline__ float Vec<T, VE>::get(int i) const { return as_float(e[i]); }

__device__ __forceinline__ void round_to(float x, float &y) { y = x; }
__device__ __forceinline__ void round_to(float x, __half &y) { y = __float2half_rn(x); }
__device__ __forceinline__ void round_to(float x, __nv_bfloat16 &y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void round_pair(float a, float b, float *y) { y[0] = a; y[1] = b; }
__device__ __forceinline__ void round_pair(float a, float b, __half *y) { *reinterpret_cast<__half2 *>(y) = __floats2half2_rn(a, b); }
__device__ __forceinline__ void round_pair(float a, float b, __nv_bfloat16 *y) { *reinterpret_cast<__nv_bfloat162 *>(y) = __floats2bfloat162_rn(a, b); }

template <typename T, int VE>
__device__ __forceinline__ void Vec<T, VE>::set(const float *x)
{
    if (VE == 1) {
        round_to(x[0], e[0]);
    } else {
#pragma unroll
        for (int i = 0; i + 1 < VE; i += 2) round_pair(x[i], x[i + 1], &e[i]);
    }
}

// Element i of an array whose type is known at run time.
__device__ __forceinline__ float load_any(const void *p, int dtype, int64_t i)
{
    if (dtype == LEGION_F32) return static_cast<const float *>(p)[i];
    if (dtype == LEGION_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_any(void *p, int dtype, int64_t i, float x)
{
    if (dtype == LEGION_F32) static_cast<float *>(p)[i] = x;
    else if (dtype == LEGION_F16) static_cast<__half *>(p)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(x);
}

// Largest of `most`, most / 2, ... 1 that divides what is given.
__host__ __forceinline__ int common_vector(int most, std::initializer_list<int64_t> counts)
{
    for (; most > 1; most >>= 1) {
        bool ok = true;
        for (int64_t c : counts) ok = ok && c % most == 0;
        if (ok) break;
    }
    return most;
}
// Elements that a vector at p may have as far as the address goes (a multiple of its element's size).
__host__ __forceinline__ int64_t aligned_elements(const void *p, int dtype) { return (int64_t)((uintptr_t)p / dtype_bytes(dtype)); }

// x / d by one multiplication: x * m >> 64 with m = floor((2^64 - 1) / d) + 1 is exact for all 32-bit x and d, because m is at
// most one above 2^64 / d and x < 2^64 / d.
struct FastDiv {
    uint32_t d;
    uint64_t m;
    explicit FastDiv(uint32_t v) : d(v), m(v > 1 ? ~0ull / v + 1 : 0) {}
    __device__ __forceinline__ uint32_t div(uint32_t x) const { return d > 1 ? (uint32_t)__umul64hi(m, (uint64_t)x) : x; }
};

}  // namespace legion
