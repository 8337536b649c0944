// RMS norm with the residual's addition, its output as it is or as compressed rows, and its gradient.
//
//   h = x + r,   s = 1 / sqrt(mean(h^2) + eps),   y = h * w * s
//   compressed: a = max |y|, scale = a / top, code = y * (top / a) rounded (the quantiser of the caches; top = 127 or 448)
//   gradient, g = dy * w:   dx = s * g - h * s^3 * mean(g * h) (+ dres),   dw = sum over rows of dy * h * s
//   worked out as dx = s * g - (h * s) * (s * (s * mean(g * h))): s^3 is no normal fp32 number for rows below 1.4e-13 and above 4e12,
//   while h * s and s * mean(g * h) are of the order of 1 and of g whatever the size of the row
//
// A row is read once: a group of threads (8 or 32 lanes of a warp, or a CTA) holds it in registers from the loads through
// the sums to the stores.  s is positive and rounding is monotone, so max |y| is s * max |h * w| to the bit, and the norm
// and the codec share one reduction.  Sums are fp32, h is kept in fp32 until y is rounded; what
// residual_out receives is h rounded once.  What bounds all of it is HBM.
#include "async.cuh"
#include "codec.cuh"
#include "typed.cuh"

#include <utility>

namespace legion {

static constexpr unsigned kFull = 0xFFFFFFFFu;

__device__ int32_t g_norm_error = 0;
__device__ __forceinline__ void raise_operator_error() { atomicCAS(&g_norm_error, 0, LEGION_E_TIMEOUT); }
cudaError_t norm_error_word(void **word) { return cudaGetSymbolAddress(word, g_norm_error); }

// Two fp32 values that one instruction works on, each rounded as it would be alone.
struct Two {
    uint64_t v;
    __device__ __forceinline__ static Two of(float a, float b)
    {
        Two t;
        asm("mov.b64 %0, {%1, %2};" : "=l"(t.v) : "f"(a), "f"(b));
        return t;
    }
    __device__ __forceinline__ float low() const { return __uint_as_float((uint32_t)v); }
    __device__ __forceinline__ float high() const { return __uint_as_float((uint32_t)(v >> 32)); }
    __device__ __forceinline__ float sum() const { return low() + high(); }
};
__device__ __forceinline__ Two operator*(const Two &a, const Two &b)
{
    Two t;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.v) : "l"(a.v), "l"(b.v));
    return t;
}
__device__ __forceinline__ Two fma(const Two &a, const Two &b, const Two &c)
{
    Two t;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return t;
}
// 1 / sqrt(x): rsqrtf's value, off by up to two units in the last place, after one of Newton's steps, which leaves the roundings of x r and
// of the result; at 0 and infinity as rsqrtf has it.
__device__ __forceinline__ float inverse_root(float x)
{
    const float r = rsqrtf(x);
    return r > 0.0f && r < INFINITY ? fmaf(0.5f * r, fmaf(-x * r, r, 1.0f), r) : r;
}

// Sum and, WITH_MAX, NaN-keeping maximum over the threads of a row.  GROUP lanes of a warp, or (0) the CTA.
template <int GROUP>
struct RowReduce {
    float *smem;   // 2 x 2 x 32 words: two buffers used in turn, so that one barrier per row is enough
    int flip = 0;
    __device__ __forceinline__ explicit RowReduce(float *s) : smem(s) {}
    __device__ __forceinline__ void two(float &a, float &b, bool second_is_max)
    {
        constexpr int kLanes = GROUP == 0 ? 32 : GROUP;
#pragma unroll
        for (int d = kLanes / 2; d > 0; d >>= 1) {
            a += __shfl_xor_sync(kFull, a, d);
            const float o = __shfl_xor_sync(kFull, b, d);
            b = second_is_max ? max_nan(b, o) : b + o;
        }
        if (GROUP == 0) {
            const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
            float *sa = smem + flip * 64, *sb = sa + 32;
            flip ^= 1;
            if (lane == 0) {
                sa[warp] = a;
                sb[warp] = b;
            }
            __syncthreads();
            a = lane < warps ? sa[lane] : 0.0f;
            b = lane < warps ? sb[lane] : 0.0f;   // a maximum here is one of absolute values
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                a += __shfl_xor_sync(kFull, a, d);
                const float o = __shfl_xor_sync(kFull, b, d);
                b = second_is_max ? max_nan(b, o) : b + o;
            }
        }
    }
};

struct NormParams {
    const void *x, *residual, *weight;
    void *out, *residual_out;
    int64_t n, x_stride, residual_stride, out_stride, residual_out_stride;  // out_stride: bytes for compressed rows
    int32_t dim, weight_dtype;
    float eps;
};

// VE weights in fp32, by vectors where the address allows it; zeros behind the row's end.
template <typename T, int VE>
__device__ __forceinline__ void load_weight(const void *p, int dtype, int col, int dim, float *w)
{
    if (col >= dim) {
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = 0.0f;
    } else if (dtype == LEGION_F32 && (uintptr_t)p % 16 == 0) {   // col is a multiple of VE
        Vec<float, VE> v;
        v.load(static_cast<const float *>(p) + col);
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = v.get(i);
    } else if (dtype != LEGION_F32 && (uintptr_t)p % 16 == 0) {
        Vec<T, VE> v;
        v.load(static_cast<const T *>(p) + col);
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = v.get(i);
    } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) w[i] = load_any(p, dtype, col + i);
    }
}

template <int VE>
__device__ __forceinline__ void store_codes(uint8_t *p, const uint32_t *c)
{
    if (VE == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(c[0], c[1 % ((VE + 3) / 4)]);
    else if (VE == 4) *reinterpret_cast<uint32_t *>(p) = c[0];
    else if (VE == 2) *reinterpret_cast<uint16_t *>(p) = (uint16_t)c[0];
    else *p = (uint8_t)c[0];
}

template <typename T, int VE, int U, int GROUP, int CODEC, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_kernel(NormParams p)
{
    __shared__ float smem[128];
    RowReduce<GROUP> reduce(smem);
    const int width = GROUP == 0 ? blockDim.x : GROUP;
    const int t = GROUP == 0 ? threadIdx.x : threadIdx.x & (GROUP - 1);
    const int per_cta = GROUP == 0 ? 1 : 128 / (GROUP == 0 ? 1 : GROUP);
    const int mate = GROUP == 0 ? 0 : threadIdx.x / (GROUP == 0 ? 1 : GROUP);
    Vec<T, VE> a[U], r[U];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = (t + u * width) * VE;
            a[u].zero();
            r[u].zero();
            if (row < p.n && col < p.dim) {
                a[u].load(static_cast<const T *>(p.x) + row * p.x_stride + col);
                if (p.residual != nullptr) r[u].load(static_cast<const T *>(p.residual) + row * p.residual_stride + col);
            }
        }
    };
    constexpr bool kAhead = U * VE <= 16 || GROUP == 32 || sizeof(T) == 2;   // wider threads of a CTA have no registers for it
    const int64_t step = (int64_t)gridDim.x * per_cta;
    if (kAhead) fetch((int64_t)blockIdx.x * per_cta + mate);
    float w[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u) load_weight<T, VE>(p.weight, p.weight_dtype, (t + u * width) * VE, p.dim, w[u]);
    const float top = CODEC == LEGION_CODEC_INT8 ? 127.0f : 448.0f;
    // the rows of a CTA's groups end together, so that every lane takes part in the reductions
    for (int64_t row0 = (int64_t)blockIdx.x * per_cta; row0 < p.n; row0 += step) {
        const int64_t row = row0 + mate;
        const bool in = row < p.n;
        if (!kAhead) fetch(row);
        float h[U][VE];
        float sum = 0.0f, most = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                h[u][i] = a[u].get(i);
                if (p.residual != nullptr) h[u][i] += r[u].get(i);
            }
        if (kAhead && row0 + step < p.n) fetch(row + step);  // the next row is on its way while this one is worked on
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = (t + u * width) * VE;
#pragma unroll
            for (int i = 0; i < VE; ++i) sum = fmaf(h[u][i], h[u][i], sum);
            if (p.residual_out != nullptr && in && col < p.dim) {
                Vec<T, VE> o;
                o.set(h[u]);
                o.store(static_cast<T *>(p.residual_out) + row * p.residual_out_stride + col);
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                h[u][i] *= w[u][i];
                if (CODEC != LEGION_CODEC_RAW && col < p.dim) most = max_nan(most, fabsf(h[u][i]));
            }
        }
        reduce.two(sum, most, true);
        const float s = 1.0f / sqrtf(sum / (float)p.dim + p.eps);
        if (CODEC == LEGION_CODEC_RAW) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int col = (t + u * width) * VE;
                if (!in || col >= p.dim) continue;
#pragma unroll
                for (int i = 0; i < VE; ++i) h[u][i] *= s;
                Vec<T, VE> o;
                o.set(h[u]);
                o.store(static_cast<T *>(p.out) + row * p.out_stride + col);
            }
            continue;
        }
        most *= s;
        const bool plain_max = __float_as_uint(most) < 0x7F800000u;
        if (GROUP == 0 ? !plain_max : __any_sync(kFull, !plain_max)) {
            // not all values are numbers: the scale is that of those that are
            float num = 0.0f, unused = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    if ((t + u * width) * VE < p.dim) num = fmaxf(num, fabsf(h[u][i] * s));
            reduce.two(unused, num, true);
            if (!plain_max) most = num;
        }
        const float inv = most > 0.0f ? __fdiv_rn(top, most) : 0.0f, scale = __fdiv_rn(most, top);
        const bool plain = plain_max && __float_as_uint(inv) < 0x7F800000u;
        if (!in) continue;
        uint8_t *dst = static_cast<uint8_t *>(p.out) + row * p.out_stride;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = (t + u * width) * VE;
            if (col >= p.dim) continue;
            uint32_t c[(VE + 3) / 4];
#pragma unroll
            for (int q = 0; q < (VE + 3) / 4; ++q) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = 4 * q + i < VE ? h[u][(4 * q + i) % VE] * s : 0.0f;
                const float4 f = make_float4(v[0], v[1], v[2], v[3]);
                c[q] = plain ? encode4<CODEC, false>(f, inv) : encode4<CODEC, true>(f, inv);
            }
            store_codes<VE>(dst + col, c);
        }
        const int tail = (int)((code_row_bytes(p.dim) - p.dim) >> 2);
        if (t < tail) reinterpret_cast<uint32_t *>(dst + p.dim)[t] = t == 0 ? __float_as_uint(scale) : 0u;
    }
}

// Long rows of an odd number of elements, where all operands' rows lie alike: vectors are those of memory, not of the row.  A row begins `shift` elements into its first vector; whole vectors are moved as such, the two at the ends
// element by element.  Which weight meets which element of a vector then changes from row to row: weights lie in shared
// memory, column j at [j % VE][j / VE], where the lanes of an access hit different banks whatever the shift.
// Measured, with residual: 8192 rows of 4097 bf16 109 us, 291 element by element; 4000 of 4097 fp32 75 us, 250.  Rows that a warp holds are
// better off with elements (20000 of 603 fp16: 45 us like this, 35), and so are rows on 4-byte boundaries with vectors of four bytes (8192 of
// 4098 bf16: 109 us like this, 82).
template <typename T, int U>
struct Framed {
    static constexpr int VE = 16 / (int)sizeof(T);
    int t, width, dim, pitch;
    __device__ __forceinline__ int first(int u, int shift) const { return (t + u * width) * VE - shift; }   // column of the vector's first element
    __device__ __forceinline__ int at(int u, int i, int shift) const   // of element i's column in a table laid out as above
    {
        const int v = t + u * width, q = i - shift;
        return q < 0 ? (q + VE) * pitch + v - 1 : q * pitch + v;
    }
    __device__ __forceinline__ bool has(int u, int i, int shift) const { return (unsigned)(first(u, shift) + i) < (unsigned)dim; }
    __device__ __forceinline__ void load(const T *row, int shift, Vec<T, VE> *v) const
    {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = first(u, shift);
            v[u].zero();
            if (c >= 0 && c + VE <= dim) {
                v[u].load(row + c);
            } else if (c + VE > 0 && c < dim) {
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    if (has(u, i, shift)) v[u].e[i] = row[c + i];
            }
        }
    }
    __device__ __forceinline__ void store(T *row, int shift, int u, const float *x) const
    {
        const int c = first(u, shift);
        Vec<T, VE> v;
        v.set(x);
        if (c >= 0 && c + VE <= dim) {
            v.store(row + c);
        } else if (c + VE > 0 && c < dim) {
#pragma unroll
            for (int i = 0; i < VE; ++i)
                if (has(u, i, shift)) row[c + i] = v.e[i];
        }
    }
};
constexpr int kFramedThreads = 544;   // 16384 elements, four vectors of eight or eight of four a thread, and the ends
// words of such a table
__host__ __device__ __forceinline__ int framed_pitch(int dim, int ve) { return dim / ve + 2; }

template <typename T, int U>
__global__ void __launch_bounds__(kFramedThreads) norm_framed_kernel(NormParams p)
{
    constexpr int VE = 16 / (int)sizeof(T);
    extern __shared__ float table[];
    __shared__ float smem[128];
    RowReduce<0> reduce(smem);
    const Framed<T, U> f{ (int)threadIdx.x, (int)blockDim.x, p.dim, framed_pitch(p.dim, VE) };
    for (int j = threadIdx.x; j < p.dim; j += blockDim.x) table[(j % VE) * f.pitch + j / VE] = load_any(p.weight, p.weight_dtype, j);
    __syncthreads();
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
        const int shift = (int)((uintptr_t)x / sizeof(T) % VE);
        Vec<T, VE> a[U], r[U];
        f.load(x, shift, a);
        if (p.residual != nullptr) f.load(static_cast<const T *>(p.residual) + row * p.residual_stride, shift, r);
        float h[U][VE];
        float sum = 0.0f, unused = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                h[u][i] = a[u].get(i);
                if (p.residual != nullptr) h[u][i] += r[u].get(i);
                sum = fmaf(h[u][i], h[u][i], sum);
            }
            if (p.residual_out != nullptr) f.store(static_cast<T *>(p.residual_out) + row * p.residual_out_stride, shift, u, h[u]);
        }
        reduce.two(sum, unused, false);
        const float s = 1.0f / sqrtf(sum / (float)p.dim + p.eps);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < VE; ++i)
                if (f.has(u, i, shift)) h[u][i] = h[u][i] * table[f.at(u, i, shift)] * s;
            f.store(static_cast<T *>(p.out) + row * p.out_stride, shift, u, h[u]);
        }
    }
}

constexpr int kStreamStages = 8;
constexpr int kStreamSmem = 216 * 1024;   // of an SM, for rows on their way

struct NormGradParams {
    const void *grad_out, *x, *grad_residual, *weight;
    void *grad_x;
    float *part;   // [CTA][dim]: the CTA's rows' share of the weight's gradient
    int64_t n, grad_stride, x_stride, grad_residual_stride, grad_x_stride;
    int32_t dim, weight_dtype;
    float eps;
    uint32_t tries;   // of a wait
};

// One CTA an SM is asked for where a thread has 32 columns: without that the compiler gives such a thread of fp32 32 registers and 3 KB of
// spills (2000 rows of 12000 with a residual: 536 us, 113 with 128 registers).
template <typename T, int VE, int U, int GROUP, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 512 && U * VE == 32 ? 1 : 0) norm_grad_kernel(NormGradParams p)
{
    __shared__ float smem[128];
    __shared__ float cross[GROUP == 0 ? 1 : 128 * U * VE];
    RowReduce<GROUP> reduce(smem);
    cudaTriggerProgrammaticLaunchCompletion();
    const int width = GROUP == 0 ? blockDim.x : GROUP;
    const int t = GROUP == 0 ? threadIdx.x : threadIdx.x & (GROUP - 1);
    const int per_cta = GROUP == 0 ? 1 : 128 / (GROUP == 0 ? 1 : GROUP);
    const int mate = GROUP == 0 ? 0 : threadIdx.x / (GROUP == 0 ? 1 : GROUP);
    Vec<T, VE> next_h[U], next_dy[U], next_r[U];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = (t + u * width) * VE;
            next_h[u].zero();
            next_dy[u].zero();
            next_r[u].zero();
            if (row < p.n && col < p.dim) {
                next_h[u].load(static_cast<const T *>(p.x) + row * p.x_stride + col);
                next_dy[u].load(static_cast<const T *>(p.grad_out) + row * p.grad_stride + col);
                if (p.grad_residual != nullptr) next_r[u].load(static_cast<const T *>(p.grad_residual) + row * p.grad_residual_stride + col);
            }
        }
    };
    // wider threads have no registers for it (12371 rows of 602 fp32: 51 us with it, 32 without, 28 since two elements share an instruction)
    constexpr bool kAhead = U * VE * (int)sizeof(T) <= 64 && MAXT <= 256;
    const int64_t step = (int64_t)gridDim.x * per_cta;
    if (kAhead) fetch((int64_t)blockIdx.x * per_cta + mate);
    // the thread's elements in pairs, whatever vectors they came by (a thread of one element has half a pair)
    constexpr int E = U * VE, P = (E + 1) / 2;
    float x[2 * P];
    x[2 * P - 1] = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) load_weight<T, VE>(p.weight, p.weight_dtype, (t + u * width) * VE, p.dim, x + u * VE);
    Two w[P], dw[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
        w[j] = Two::of(x[2 * j], x[2 * j + 1]);
        dw[j] = Two::of(0.0f, 0.0f);
    }
    auto pair = [&](const Vec<T, VE> *v, int j) { return Two::of(v[2 * j / VE].get(2 * j % VE), 2 * j + 1 < E ? v[(2 * j + 1) % E / VE].get((2 * j + 1) % VE) : 0.0f); };
    const float per_dim = 1.0f / (float)p.dim;
    for (int64_t row0 = (int64_t)blockIdx.x * per_cta; row0 < p.n; row0 += step) {
        const int64_t row = row0 + mate;
        const bool in = row < p.n;
        if (!kAhead) fetch(row);
        Vec<T, VE> h[U], dy[U], r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            h[u] = next_h[u];
            dy[u] = next_dy[u];
            r[u] = next_r[u];
        }
        if (kAhead && row0 + step < p.n) fetch(row + step);  // the next row is on its way while this one is worked on
        Two square2 = Two::of(0.0f, 0.0f), dot2 = square2;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const Two a = pair(h, j);
            square2 = fma(a, a, square2);
            dot2 = fma(pair(dy, j) * w[j], a, dot2);
        }
        float square = square2.sum(), dot = dot2.sum();
        reduce.two(square, dot, false);
        const float s = inverse_root(fmaf(square, per_dim, p.eps));
        const float k = s * (s * (dot * per_dim));
        const Two s2 = Two::of(s, s), k2 = Two::of(-k, -k);
        float dx[2 * P];
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const Two normed = pair(h, j) * s2, g = pair(dy, j);
            const Two d = fma(normed, k2, fma(g * w[j], s2, pair(r, j)));
            dx[2 * j] = d.low();
            dx[2 * j + 1] = d.high();
            if (in) dw[j] = fma(g, normed, dw[j]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = (t + u * width) * VE;
            if (!in || col >= p.dim) continue;
            Vec<T, VE> o;
            o.set(dx + u * VE);
            o.store(static_cast<T *>(p.grad_x) + row * p.grad_x_stride + col);
        }
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
        x[2 * j] = dw[j].low();
        x[2 * j + 1] = dw[j].high();
    }
    float *part = p.part + (int64_t)blockIdx.x * p.dim;
    if (GROUP == 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < VE; ++i)
                if ((t + u * width) * VE < p.dim) part[(t + u * width) * VE + i] = x[u * VE + i];
        return;
    }
    // the groups of a CTA add theirs in group order
    constexpr int kCols = (GROUP == 0 ? 1 : GROUP) * U * VE;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < VE; ++i) cross[(threadIdx.x / (GROUP == 0 ? 1 : GROUP)) * kCols + (t + u * GROUP) * VE + i] = x[u * VE + i];
    __syncthreads();
    for (int col = threadIdx.x; col < p.dim; col += 128) {
        float sum = 0.0f;
        for (int g = 0; g < per_cta; ++g) sum += cross[g * kCols + col];
        part[col] = sum;
    }
}

// Sums of N values each over the threads of a CTA, for N of 2 or 4 and at most 32 / N warps: halves of the lanes take over half of the values as
// the lanes are added up, so that N values cost little more than one.  One barrier.
template <int N>
__device__ __forceinline__ void sums_of_cta(float *v, float *smem, int &flip)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int d = 16;
#pragma unroll
    for (int n = N; n > 1; n /= 2, d /= 2) {
        const bool upper = lane & d;
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
            const float give = upper ? v[i] : v[i + n / 2], keep = upper ? v[i + n / 2] : v[i];
            v[i] = keep + __shfl_xor_sync(kFull, give, d);
        }
    }
#pragma unroll
    for (; d > 0; d /= 2) v[0] += __shfl_xor_sync(kFull, v[0], d);
    // the lane's value: the bits of the lane from the highest on
    constexpr int kLanes = 32 / N;
    float *s = smem + flip * 32;
    flip ^= 1;
    const int warps = blockDim.x >> 5;
    if (lane % kLanes == 0) s[lane + warp] = v[0];
    __syncthreads();
    float x = lane % kLanes < warps ? s[lane] : 0.0f;
#pragma unroll
    for (int e = kLanes / 2; e > 0; e /= 2) x += __shfl_xor_sync(kFull, x, e);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __shfl_sync(kFull, x, i * kLanes);
}

// The same for long rows on 16-byte boundaries, where there are many: one thread has the copy engine bring whole rows into shared memory,
// `stages` rows ahead, so that what is on its way does not depend on registers.  A stage is free again when the threads
// have met in the row's reduction: by then all of them have read their part of it.  R rows meet in one reduction (stages: a multiple of R):
// what bounds a CTA is that meeting, and the instructions (hence pairs of fp32).
// Measured, 16384 rows of 2048 bf16 with residual (268 MB): 49 us a call, 5.5 TB/s; one row a meeting 53.5; single fp32 and the reduction of one row at a
// time 60; the next row in registers 64, without it 72.
template <typename T, int U, int R, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) norm_grad_stream_kernel(NormGradParams p, int stages)
{
    constexpr int VE = 16 / (int)sizeof(T);
    // a CTA of many threads has no registers for a row and reads it from its stage again, which is free a row later then (with the row in
    // spilled registers, 4000 rows of 12000 bf16 took 360 us, like this 61)
    constexpr bool kAgain = MAXT > 256;
    static_assert(R == 1 || !kAgain, "the stage before is one row's");
    extern __shared__ __align__(128) uint8_t rows[];   // [stage][x, grad_out, grad_residual][row]
    __shared__ float smem[128];
    __shared__ uint64_t bars[kStreamStages];
    RowReduce<0> reduce(smem);
    int flip = 0;
    const int t = threadIdx.x, width = blockDim.x;
    const uint32_t row_bytes = (uint32_t)p.dim * sizeof(T);
    const int arrays = p.grad_residual != nullptr ? 3 : 2;
    auto bring = [&](int64_t row, int stage) {   // one thread
        const uint32_t bar = shared_addr(&bars[stage]), dst = shared_addr(rows) + stage * arrays * row_bytes;
        expect_bytes(bar, arrays * row_bytes);
        bulk_copy(dst, static_cast<const T *>(p.x) + row * p.x_stride, row_bytes, bar);
        bulk_copy(dst + row_bytes, static_cast<const T *>(p.grad_out) + row * p.grad_stride, row_bytes, bar);
        if (arrays == 3) bulk_copy(dst + 2 * row_bytes, static_cast<const T *>(p.grad_residual) + row * p.grad_residual_stride, row_bytes, bar);
    };
    const int64_t step = gridDim.x;
    cudaTriggerProgrammaticLaunchCompletion();
    if (t == 0) {
        for (int s = 0; s < stages; ++s) init_barrier(shared_addr(&bars[s]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int s = 0; s < stages; ++s)
            if (blockIdx.x + s * step < p.n) bring(blockIdx.x + s * step, s);
    }
    Two w[U][VE / 2], dw[U][VE / 2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[VE];
        load_weight<T, VE>(p.weight, p.weight_dtype, (t + u * width) * VE, p.dim, x);
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            w[u][i] = Two::of(x[2 * i], x[2 * i + 1]);
            dw[u][i] = Two::of(0.0f, 0.0f);
        }
    }
    const float per_dim = 1.0f / (float)p.dim;
    __syncthreads();
    int stage = 0;
    uint32_t phase = 0, tries = p.tries;
    for (int64_t row = blockIdx.x; row < p.n; row += R * step) {
        Vec<T, VE> h[R][U], dy[R][U], r[R][U];
        const uint8_t *src[R];
        float sums[2 * R];   // of the rows' squares, then of dy w h
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const bool in = row + q * step < p.n;
            if (in && !wait_barrier(shared_addr(&bars[stage + q]), phase, tries)) tries = 0;   // given up: the rest is not waited for, the error is kept
            src[q] = rows + (size_t)(stage + q) * arrays * row_bytes;
            Two square = Two::of(0.0f, 0.0f), dot = square;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int col = (t + u * width) * VE;
                h[q][u].zero();
                dy[q][u].zero();
                r[q][u].zero();
                if (in && col < p.dim) {
                    h[q][u].load(reinterpret_cast<const T *>(src[q]) + col);
                    dy[q][u].load(reinterpret_cast<const T *>(src[q] + row_bytes) + col);
                    if (!kAgain && arrays == 3) r[q][u].load(reinterpret_cast<const T *>(src[q] + 2 * row_bytes) + col);
                }
#pragma unroll
                for (int i = 0; i < VE / 2; ++i) {
                    const Two a = Two::of(h[q][u].get(2 * i), h[q][u].get(2 * i + 1));
                    square = fma(a, a, square);
                    dot = fma(Two::of(dy[q][u].get(2 * i), dy[q][u].get(2 * i + 1)) * w[u][i], a, dot);
                }
            }
            sums[q] = square.sum();
            sums[R + q] = dot.sum();
        }
        if (MAXT <= 256) sums_of_cta<2 * R>(sums, smem, flip);
        else reduce.two(sums[0], sums[R], false);
        if (t == 0 && tries != 0) {
            if (kAgain) {   // the row before is done with
                if (row >= step && row + (stages - 1) * step < p.n) bring(row + (stages - 1) * step, stage == 0 ? stages - 1 : stage - 1);
            } else {
#pragma unroll
                for (int q = 0; q < R; ++q)
                    if (row + (stages + q) * step < p.n) bring(row + (stages + q) * step, stage + q);
            }
        }
        stage += R;
        if (stage == stages) {
            stage = 0;
            phase ^= 1;
        }
#pragma unroll
        for (int q = 0; q < R; ++q) {
            const float s = inverse_root(fmaf(sums[q], per_dim, p.eps));
            const float k = s * (s * (sums[R + q] * per_dim));
            const Two s2 = Two::of(s, s), k2 = Two::of(-k, -k);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int col = (t + u * width) * VE;
                if (col >= p.dim || row + q * step >= p.n) continue;
                if (kAgain) {
                    h[q][u].load(reinterpret_cast<const T *>(src[q]) + col);
                    dy[q][u].load(reinterpret_cast<const T *>(src[q] + row_bytes) + col);
                    if (arrays == 3) r[q][u].load(reinterpret_cast<const T *>(src[q] + 2 * row_bytes) + col);
                }
                float dx[VE];
#pragma unroll
                for (int i = 0; i < VE / 2; ++i) {
                    const Two normed = Two::of(h[q][u].get(2 * i), h[q][u].get(2 * i + 1)) * s2, g = Two::of(dy[q][u].get(2 * i), dy[q][u].get(2 * i + 1));
                    const Two d = fma(normed, k2, fma(g * w[u][i], s2, Two::of(r[q][u].get(2 * i), r[q][u].get(2 * i + 1))));
                    dx[2 * i] = d.low();
                    dx[2 * i + 1] = d.high();
                    dw[u][i] = fma(g, normed, dw[u][i]);
                }
                Vec<T, VE> o;
                o.set(dx);
                o.store(static_cast<T *>(p.grad_x) + (row + q * step) * p.grad_x_stride + col);
            }
        }
    }
    float *part = p.part + (int64_t)blockIdx.x * p.dim;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int col = (t + u * width) * VE;
        if (col >= p.dim) continue;
        float x[VE];
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            x[2 * i] = dw[u][i].low();
            x[2 * i + 1] = dw[u][i].high();
        }
        Vec<float, VE> o;
        o.set(x);
        o.store(part + col);
    }
    // one thread's wait may have been given up where another's was not: all of them decide together
    if (__syncthreads_or(tries == 0) && t == 0) {
        raise_operator_error();
        // the copies that are under way land before the CTA's memory goes: they take microseconds, this waits a millisecond
        for (const long long t0 = clock64(); clock64() - t0 < 2000000;) { }
    }
}

// Columns of the CTAs' shares added: 16 columns a CTA, 64 threads a column, one fixed order.
__global__ void __launch_bounds__(1024) norm_weight_grad_kernel(const float *__restrict__ part, int parts, int dim, void *out, int dtype)
{
    __shared__ float s[64][17];
    const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
    const int col = blockIdx.x * 16 + x;
    cudaGridDependencySynchronize();
    float sum = 0.0f;
    if (col < dim)
#pragma unroll 10
        for (int g = y; g < parts; g += 64) sum += part[(int64_t)g * dim + col];
    s[y][x] = sum;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (warp >= 16) return;
    sum = s[lane][warp] + s[lane + 32][warp];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
    if (lane == 0 && blockIdx.x * 16 + warp < dim) store_any(out, dtype, blockIdx.x * 16 + warp, sum);
}

// ---- host side -----------------------------------------------------------------------------------------------------

constexpr int kGradCtas = 4 * kSms;  // most CTAs of the gradient: their shares of the weight's gradient lie in scratch

// How a row of `vecs` vectors is held: by 8 lanes, by a warp (up to 32 elements a lane where there are many rows: nobody waits at a
// barrier then), or by a CTA.
struct RowShape {
    int group, u, threads, per_cta;
};
static RowShape row_shape(int vecs, int ve, int64_t n)
{
    if (vecs <= 8) return { 8, 1, 128, 16 };
    for (int w = 1; w <= 16 && w * ve <= 32 && (w == 1 || n >= 8 * kSms); w *= 2)
        if (vecs <= 32 * w) return { 32, w, 128, 4 };
    int u = 1;  // few rows: as many threads as there are vectors; many: CTAs of about 256 threads, so that several are on an SM
    if (n >= 2 * kSms)
        while (u < 4 && (vecs + u - 1) / u > 256) u *= 2;
    while ((vecs + u - 1) / u > 512) u *= 2;
    return { 0, u, ((vecs + u - 1) / u + 31) / 32 * 32, 1 };
}

// CTAs of a kernel that loops over rows: as many as are on the chip at one time (at most `per_sm` a SM), so that none starts late.
static unsigned resident(int64_t need, const void *kernel, int threads, int per_sm, int smem = 0)
{
    if (need <= kSms) return (unsigned)need;
    int fit = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, threads, smem) != cudaSuccess || fit < 1) fit = 1;
    if (fit > per_sm) fit = per_sm;
    return (unsigned)(need < (int64_t)fit * kSms ? need : (int64_t)fit * kSms);
}

template <typename T, int U>
static int go_framed(cudaStream_t s, const NormParams &p, int threads)
{
    constexpr int VE = 16 / (int)sizeof(T);
    const void *kernel = (const void *)norm_framed_kernel<T, U>;
    const int smem = 4 * VE * framed_pitch(p.dim, VE);
    static bool allowed[64];
    const int rc = allow_smem(kernel, 4 * VE * framed_pitch(LEGION_NORM_MAX_DIM, VE), allowed);
    if (rc != LEGION_OK) return rc;
    norm_framed_kernel<T, U><<<resident(p.n, kernel, threads, 16, smem), threads, smem, s>>>(p);
    LG_LAUNCH_CHECK();
    return LEGION_OK;
}

template <typename T>
static int launch_framed(cudaStream_t s, const NormParams &p)
{
    constexpr int VE = 16 / (int)sizeof(T);
    const int vecs = p.dim / VE + 2;
    int u = 1;
    while (u * VE < 32 && (vecs + u - 1) / u > 256) u *= 2;
    const int threads = ((vecs + u - 1) / u + 31) / 32 * 32;
    if (u == 1) return go_framed<T, 1>(s, p, threads);
    if (u == 2) return go_framed<T, 2>(s, p, threads);
    if constexpr (VE == 8) return go_framed<T, 4>(s, p, threads);
    else return u == 4 ? go_framed<T, 4>(s, p, threads) : go_framed<T, 8>(s, p, threads);
}

// Whether all rows of the operands lie alike in 16-byte vectors.
static bool lie_alike(int dtype, std::initializer_list<std::pair<const void *, int64_t>> rows)
{
    const auto &first = *rows.begin();
    for (const auto &r : rows)
        if (r.first != nullptr && (((uintptr_t)r.first ^ (uintptr_t)first.first) % 16 != 0 || (r.second - first.second) % (16 / dtype_bytes(dtype)) != 0))
            return false;
    return true;
}

template <typename T, int VE, int CODEC>
static int launch_norm(cudaStream_t s, const NormParams &p)
{
    const RowShape r = row_shape(p.dim / VE, VE, p.n);
    const int64_t need = (p.n + r.per_cta - 1) / r.per_cta;
#define LG_NORM(U, GROUP, MAXT)                                                                                                     \
    norm_kernel<T, VE, U, GROUP, CODEC, MAXT><<<resident(need, (const void *)norm_kernel<T, VE, U, GROUP, CODEC, MAXT>, r.threads, 16), \
                                                r.threads, 0, s>>>(p)
// a CTA of at most 256 threads may have twice the registers of a thread of one of 512
#define LG_NORM_CTA(U) do { if (r.threads <= 256) LG_NORM(U, 0, 256); else LG_NORM(U, 0, 512); } while (0)
    if (r.group == 8) LG_NORM(1, 8, 128);
    else if (r.group == 32) {
        if (r.u == 1) LG_NORM(1, 32, 128);
        else if (r.u == 2) LG_NORM(2, 32, 128);
        else if (r.u == 4) LG_NORM(4, 32, 128);
        else if (r.u == 8) { if constexpr (VE <= 4) LG_NORM(8, 32, 128); }
        else { if constexpr (VE <= 2) LG_NORM(16, 32, 128); }
    }
    else if (r.u == 1) LG_NORM_CTA(1);
    else if (r.u == 2) LG_NORM_CTA(2);
    else if (r.u == 4) LG_NORM_CTA(4);
    else if (r.u == 8) { if constexpr (VE <= 4) LG_NORM(8, 0, 512); }
    else if (r.u == 16) { if constexpr (VE <= 2) LG_NORM(16, 0, 512); }
    else { if constexpr (VE == 1) LG_NORM(32, 0, 512); }
#undef LG_NORM_CTA
#undef LG_NORM
    LG_LAUNCH_CHECK();
    return LEGION_OK;
}

template <typename T, int CODEC>
static int launch_norm_ve(cudaStream_t s, const NormParams &p, int ve)
{
    switch (ve) {
    case 8:
        if constexpr (sizeof(T) == 2) return launch_norm<T, 8, CODEC>(s, p);
    case 4: return launch_norm<T, 4, CODEC>(s, p);
    case 2: return launch_norm<T, 2, CODEC>(s, p);
    default: return launch_norm<T, 1, CODEC>(s, p);
    }
}

template <typename T>
static int launch_norm_codec(cudaStream_t s, const NormParams &p, int codec, int ve)
{
    if (codec == LEGION_CODEC_RAW) return launch_norm_ve<T, LEGION_CODEC_RAW>(s, p, ve);
    if (codec == LEGION_CODEC_INT8) return launch_norm_ve<T, LEGION_CODEC_INT8>(s, p, ve);
    return launch_norm_ve<T, LEGION_CODEC_E4M3>(s, p, ve);
}

template <typename T, int U, int R, int MAXT>
static int launch_norm_grad_stream(cudaStream_t s, const NormGradParams &p, int threads, int *parts)
{
    const void *kernel = (const void *)norm_grad_stream_kernel<T, U, R, MAXT>;
    static bool allowed[64];
    const int rc = allow_smem(kernel, kStreamSmem, allowed);
    if (rc != LEGION_OK) return rc;
    const int stage = (p.grad_residual != nullptr ? 3 : 2) * p.dim * (int)sizeof(T);
    // CTAs by their registers; each SM's shared memory is shared out among them, two stages a CTA at least
    int fit = 0;
    LG_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, threads, 0));
    if (fit > kGradCtas / kSms) fit = kGradCtas / kSms;
    while (fit > 1 && kStreamSmem / fit < 2 * R * stage) --fit;
    int stages = kStreamSmem / (fit < 1 ? 1 : fit) / stage;
    if (stages > kStreamStages) stages = kStreamStages;
    stages -= stages % R;
    const int64_t most = (int64_t)(fit < 1 ? 1 : fit) * kSms;
    *parts = (int)(p.n < most ? p.n : most);
    norm_grad_stream_kernel<T, U, R, MAXT><<<*parts, threads, stages * stage, s>>>(p, stages);
    LG_LAUNCH_CHECK();
    return LEGION_OK;
}

template <typename T, int VE>
static int launch_norm_grad(cudaStream_t s, const NormGradParams &p, int *parts)
{
    if constexpr (VE * sizeof(T) == 16) {
        const int64_t bytes = (int64_t)p.dim * sizeof(T), stage = (p.grad_residual != nullptr ? 3 : 2) * bytes;
        const int vecs = p.dim / VE;
        // (20000 rows of 2048 bytes: 35.5 us like this, 34 by a warp each; 16384 of 4096: 49 and 64; 4000 of 16 KB: 54 and 88; 300 of 16 KB: 14.5
        // and 18; 500 of 4096: the same)
        if (bytes >= 4096 && p.n >= kSms && 2 * stage <= kStreamSmem) {
            int u = 1;
            while (u < 4 && (vecs + u - 1) / u > 256) u *= 2;
            const int threads = ((vecs + u - 1) / u + 31) / 32 * 32;
            if (threads <= 256) {
                // two rows of at most 8 KB each: four stages always fit
                if (u == 1) return launch_norm_grad_stream<T, 1, 2, 256>(s, p, threads, parts);
                if (u == 2) return launch_norm_grad_stream<T, 2, 2, 256>(s, p, threads, parts);
                return launch_norm_grad_stream<T, 4, 1, 256>(s, p, threads, parts);
            }
            if (threads <= 512) return launch_norm_grad_stream<T, 4, 1, 512>(s, p, threads, parts);
        }
    }
    const RowShape r = row_shape(p.dim / VE, VE, p.n);
    const int64_t need = (p.n + r.per_cta - 1) / r.per_cta;
#define LG_NORM(U, GROUP, MAXT)                                                                                                    \
    norm_grad_kernel<T, VE, U, GROUP, MAXT><<<*parts = resident(need, (const void *)norm_grad_kernel<T, VE, U, GROUP, MAXT>, r.threads, \
                                                                kGradCtas / kSms), r.threads, 0, s>>>(p)
// a CTA of at most 256 threads may have twice the registers of a thread of one of 512
#define LG_NORM_CTA(U) do { if (r.threads <= 256) LG_NORM(U, 0, 256); else LG_NORM(U, 0, 512); } while (0)
    if (r.group == 8) LG_NORM(1, 8, 128);
    else if (r.group == 32) {
        if (r.u == 1) LG_NORM(1, 32, 128);
        else if (r.u == 2) LG_NORM(2, 32, 128);
        else if (r.u == 4) LG_NORM(4, 32, 128);
        else if (r.u == 8) { if constexpr (VE <= 4) LG_NORM(8, 32, 128); }
        else { if constexpr (VE <= 2) LG_NORM(16, 32, 128); }
    }
    else if (r.u == 1) LG_NORM_CTA(1);
    else if (r.u == 2) LG_NORM_CTA(2);
    else if (r.u == 4) LG_NORM_CTA(4);
    else if (r.u == 8) { if constexpr (VE <= 4) LG_NORM(8, 0, 512); }
    else if (r.u == 16) { if constexpr (VE <= 2) LG_NORM(16, 0, 512); }
    else { if constexpr (VE == 1) LG_NORM(32, 0, 512); }
#undef LG_NORM_CTA
#undef LG_NORM
    LG_LAUNCH_CHECK();
    return LEGION_OK;
}

template <typename T>
static int launch_norm_grad_ve(cudaStream_t s, const NormGradParams &p, int ve, int *parts)
{
    switch (ve) {
    case 8:
        if constexpr (sizeof(T) == 2) return launch_norm_grad<T, 8>(s, p, parts);
    case 4: return launch_norm_grad<T, 4>(s, p, parts);
    case 2: return launch_norm_grad<T, 2>(s, p, parts);
    default: return launch_norm_grad<T, 1>(s, p, parts);
    }
}

}  // namespace legion

using namespace legion;

// a row operand of the call's type: NULL only where it may be
#define LG_OPERAND(p, stride, dim, dtype, what)                                                          \
    LG_ARG((uintptr_t)(p) % dtype_bytes(dtype) == 0, what " must start on a multiple of its element's size"); \
    LG_ARG((p) == nullptr || ((stride) >= (dim) && (stride) <= (1ll << 40)), what ": a row's stride must be at least its length")

// Rows in the place of other rows: one by one, or each would be written over others that are not read yet.
static bool same_stride(const void *a, int64_t a_stride, const void *b, int64_t b_stride) { return a == nullptr || a != b || a_stride == b_stride; }

extern "C" int legion_rms_norm(int32_t dev_id, const void *x, int32_t dtype, int64_t x_stride, const void *residual,
                               int64_t residual_stride, const void *weight, int32_t weight_dtype, float eps, int64_t n_rows, int32_t dim,
                               int32_t codec, void *out, int64_t out_stride, void *residual_out, int64_t residual_out_stride, void *stream)
{
    LG_ARG(dtype_known(dtype), "dtype must be LEGION_F32, LEGION_F16 or LEGION_BF16");
    LG_ARG(weight_dtype == dtype || weight_dtype == LEGION_F32, "weight must be fp32 or of the rows' type");
    LG_ARG(codec >= LEGION_CODEC_RAW && codec <= LEGION_CODEC_E4M3, "codec must be RAW, INT8 or E4M3");
    LG_ARG(dim > 0 && dim <= LEGION_NORM_MAX_DIM, "dim out of range");
    LG_ARG(codec == LEGION_CODEC_RAW || dim % 4 == 0, "compressed rows need dim % 4 == 0");
    LG_ARG(n_rows >= 0 && n_rows < (1ll << 31), "n_rows out of range");
    LG_ARG(eps >= 0.0f, "eps must not be negative");
    LG_ARG(n_rows == 0 || (x != nullptr && out != nullptr && weight != nullptr), "NULL pointer");
    LG_ARG((uintptr_t)weight % dtype_bytes(weight_dtype) == 0, "weight must start on a multiple of its element's size");
    LG_OPERAND(x, x_stride, dim, dtype, "x");
    LG_OPERAND(residual, residual_stride, dim, dtype, "residual");
    LG_OPERAND(residual_out, residual_out_stride, dim, dtype, "residual_out");
    if (codec == LEGION_CODEC_RAW) {
        LG_OPERAND(out, out_stride, dim, dtype, "out");
    } else {
        LG_ARG((uintptr_t)out % 16 == 0 && out_stride % 16 == 0 && out_stride >= code_row_bytes(dim),
               "compressed rows start on multiples of 16 bytes and are (dim + 4) rounded up to 16 bytes long");
    }
    LG_ARG(n_rows == 0 || out != residual_out, "out and residual_out must be two buffers");
    LG_ARG(n_rows == 0 || codec == LEGION_CODEC_RAW || (out != x && out != residual), "compressed rows cannot take the place of x or residual");
    LG_ARG(n_rows <= 1 || (same_stride(out, out_stride, x, x_stride) && same_stride(out, out_stride, residual, residual_stride) &&
                           same_stride(residual_out, residual_out_stride, x, x_stride) &&
                           same_stride(residual_out, residual_out_stride, residual, residual_stride)),
           "an output in an input's place must have its stride");
    if (n_rows == 0) return LEGION_OK;
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    NormParams p{ x, residual, weight, out, residual_out, n_rows, x_stride, residual_stride, out_stride, residual_out_stride, dim,
                  weight_dtype, eps };
    int ve = common_vector(dtype == LEGION_F32 ? 4 : 8, { dim, x_stride, aligned_elements(x, dtype) });
    if (residual != nullptr) ve = common_vector(ve, { residual_stride, aligned_elements(residual, dtype) });
    if (residual_out != nullptr) ve = common_vector(ve, { residual_out_stride, aligned_elements(residual_out, dtype) });
    if (codec == LEGION_CODEC_RAW) ve = common_vector(ve, { out_stride, aligned_elements(out, dtype) });
    cudaStream_t s = (cudaStream_t)stream;
    if (codec == LEGION_CODEC_RAW && ve == 1 && dim > 1024 && n_rows >= 2 * kSms &&
        lie_alike(dtype, { { x, x_stride }, { residual, residual_stride }, { out, out_stride }, { residual_out, residual_out_stride } })) {
        if (dtype == LEGION_F32) return launch_framed<float>(s, p);
        if (dtype == LEGION_F16) return launch_framed<__half>(s, p);
        return launch_framed<__nv_bfloat16>(s, p);
    }
    if (dtype == LEGION_F32) return launch_norm_codec<float>(s, p, codec, ve);
    if (dtype == LEGION_F16) return launch_norm_codec<__half>(s, p, codec, ve);
    return launch_norm_codec<__nv_bfloat16>(s, p, codec, ve);
}

static int64_t norm_grad_scratch(int64_t n_rows, int32_t dim) { return (n_rows < kGradCtas ? n_rows : kGradCtas) * (int64_t)dim * 4; }

extern "C" int legion_rms_norm_grad_workspace(int64_t n_rows, int32_t dim, int64_t *bytes)
{
    LG_ARG(bytes != nullptr, "bytes is NULL");
    LG_ARG(dim > 0 && dim <= LEGION_NORM_MAX_DIM, "dim out of range");
    LG_ARG(n_rows >= 0 && n_rows < (1ll << 31), "n_rows out of range");
    *bytes = norm_grad_scratch(n_rows, dim);
    return LEGION_OK;
}

extern "C" int legion_rms_norm_grad(int32_t dev_id, const void *grad_out, int64_t grad_stride, const void *x, int64_t x_stride,
                                    int32_t dtype, const void *grad_residual, int64_t grad_residual_stride, const void *weight,
                                    int32_t weight_dtype, float eps, int64_t n_rows, int32_t dim, void *grad_x, int64_t grad_x_stride,
                                    void *grad_weight, int32_t grad_weight_dtype, void *workspace, int64_t workspace_bytes, void *stream)
{
    LG_ARG(dtype_known(dtype), "dtype must be LEGION_F32, LEGION_F16 or LEGION_BF16");
    LG_ARG(weight_dtype == dtype || weight_dtype == LEGION_F32, "weight must be fp32 or of the rows' type");
    LG_ARG(grad_weight_dtype == dtype || grad_weight_dtype == LEGION_F32, "grad_weight must be fp32 or of the rows' type");
    LG_ARG(dim > 0 && dim <= LEGION_NORM_MAX_DIM, "dim out of range");
    LG_ARG(n_rows >= 0 && n_rows < (1ll << 31), "n_rows out of range");
    LG_ARG(eps >= 0.0f, "eps must not be negative");
    LG_ARG(grad_weight != nullptr && weight != nullptr, "NULL pointer");
    LG_ARG(n_rows == 0 || (x != nullptr && grad_out != nullptr && grad_x != nullptr), "NULL pointer");
    LG_ARG((uintptr_t)weight % dtype_bytes(weight_dtype) == 0, "weight must start on a multiple of its element's size");
    LG_ARG((uintptr_t)grad_weight % dtype_bytes(grad_weight_dtype) == 0, "grad_weight must start on a multiple of its element's size");
    LG_OPERAND(x, x_stride, dim, dtype, "x");
    LG_OPERAND(grad_out, grad_stride, dim, dtype, "grad_out");
    LG_OPERAND(grad_x, grad_x_stride, dim, dtype, "grad_x");
    LG_OPERAND(grad_residual, grad_residual_stride, dim, dtype, "grad_residual");
    LG_ARG(n_rows <= 1 || (same_stride(grad_x, grad_x_stride, grad_out, grad_stride) && same_stride(grad_x, grad_x_stride, x, x_stride) &&
                           same_stride(grad_x, grad_x_stride, grad_residual, grad_residual_stride)),
           "grad_x in an input's place must have its stride");
    LG_ARG(grad_weight != weight, "grad_weight must not be the weight");
    LG_ARG(n_rows == 0 || (workspace != nullptr && (uintptr_t)workspace % 16 == 0), "workspace is NULL or not on a multiple of 16 bytes");
    LG_ARG(workspace_bytes >= norm_grad_scratch(n_rows, dim), "workspace is smaller than the call asks for");
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    cudaStream_t s = (cudaStream_t)stream;
    if (n_rows == 0) {
        LG_CUDA(cudaMemsetAsync(grad_weight, 0, (size_t)dim * dtype_bytes(grad_weight_dtype), s));
        return LEGION_OK;
    }
    NormGradParams p{ grad_out, x, grad_residual, weight, grad_x, (float *)workspace, n_rows, grad_stride, x_stride, grad_residual_stride,
                      grad_x_stride, dim, weight_dtype, eps, operator_wait_tries() };
    int ve = common_vector(dtype == LEGION_F32 ? 4 : 8, { dim, x_stride, aligned_elements(x, dtype), grad_stride, aligned_elements(grad_out, dtype),
                                                          grad_x_stride, aligned_elements(grad_x, dtype) });
    if (grad_residual != nullptr) ve = common_vector(ve, { grad_residual_stride, aligned_elements(grad_residual, dtype) });
    int parts = 0, rc;
    if (dtype == LEGION_F32) rc = launch_norm_grad_ve<float>(s, p, ve, &parts);
    else if (dtype == LEGION_F16) rc = launch_norm_grad_ve<__half>(s, p, ve, &parts);
    else rc = launch_norm_grad_ve<__nv_bfloat16>(s, p, ve, &parts);
    if (rc != LEGION_OK) return rc;
    // as a dependent of the launch before it, which it may overlap up to its cudaGridDependencySynchronize
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(dim + 15) / 16);
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    LG_CUDA(cudaLaunchKernelEx(&cfg, norm_weight_grad_kernel, (const float *)workspace, parts, (int)dim, grad_weight, (int)grad_weight_dtype));
    return LEGION_OK;
}
