// Learned rows: lookup by id with a scale, and the gradient by sorted ids.
//
//   out[i]  = scale * table[ids[i]]                       (an id outside the table: a row of zeros)
//   grad[v] = scale * sum over i with ids[i] = v of g[i]  (whole table, or only the rows of the ids that occur)
//
// The gradient sorts (id, position) pairs (stable), cuts the sorted list into stretches of equal length and lets a group
// of threads sum the rows of a stretch in list order.  A stretch writes the sums of the ids that lie wholly inside it;
// what an id that crosses a boundary has in a stretch goes to scratch, and a second launch adds these pieces in
// list order.  So an id that comes once and one that comes ten thousand times cost the same per row, each
// gradient row is read once, and the result does not depend on the order in which the CTAs run: no atomics on floats.
#include "typed.cuh"

namespace legion {

static constexpr unsigned kFull = 0xFFFFFFFFu;

struct Ids {
    const void *p;
    int32_t wide;      // 64-bit ids
    int64_t n_nodes;
    // n_nodes stands for every id outside [0, n_nodes)
    __device__ __forceinline__ uint32_t key(int64_t i) const
    {
        const int64_t v = wide ? static_cast<const int64_t *>(p)[i] : (int64_t)static_cast<const int32_t *>(p)[i];
        return (uint64_t)v < (uint64_t)n_nodes ? (uint32_t)v : (uint32_t)n_nodes;
    }
};

// ---- lookup --------------------------------------------------------------------------------------------------------

// The rows as one flat run of vectors, R vectors of 256 threads each per CTA.
template <typename TI, typename TO, int VE, int R>
__global__ void __launch_bounds__(256)
lookup_kernel(Ids ids, const TI *__restrict__ table, int64_t table_stride, TO *__restrict__ out, int64_t out_stride,
              int64_t total, FastDiv per_row, float scale)
{
    const int64_t first = (int64_t)blockIdx.x * (256 * R);
    const int64_t row0 = first / per_row.d;
    const uint32_t at0 = (uint32_t)(first - row0 * per_row.d) + threadIdx.x;
    Vec<TI, VE> v[R];
    uint32_t row[R], col[R], key[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t at = at0 + r * 256;
        row[r] = per_row.div(at);
        col[r] = (at - row[r] * per_row.d) * VE;
        key[r] = (uint32_t)ids.n_nodes;
        if (first + r * 256 + threadIdx.x < total) key[r] = ids.key(row0 + row[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        v[r].zero();
        if (key[r] < (uint32_t)ids.n_nodes) v[r].load(table + (int64_t)key[r] * table_stride + col[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (first + r * 256 + threadIdx.x >= total) break;
        float x[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) x[i] = v[r].get(i) * scale;
        Vec<TO, VE> o;
        o.set(x);
        o.store_stream(out + (row0 + row[r]) * out_stride + col[r]);
    }
}

template <typename TI, typename TO, int VE>
static void launch_lookup(cudaStream_t s, const Ids &ids, const void *table, int64_t table_stride, void *out, int64_t out_stride,
                          int64_t n, int32_t dim, float scale)
{
    const int64_t total = n * (dim / VE);
    const FastDiv per_row((uint32_t)(dim / VE));
    if (total <= (int64_t)kSms * 4 * 256)  // fewer vectors than a quarter of the chip's threads: one each
        lookup_kernel<TI, TO, VE, 1><<<(unsigned)((total + 255) / 256), 256, 0, s>>>(
            ids, (const TI *)table, table_stride, (TO *)out, out_stride, total, per_row, scale);
    else
        lookup_kernel<TI, TO, VE, 4><<<(unsigned)((total + 1023) / 1024), 256, 0, s>>>(
            ids, (const TI *)table, table_stride, (TO *)out, out_stride, total, per_row, scale);
}

template <typename TI, typename TO>
static void launch_lookup_ve(int ve, cudaStream_t s, const Ids &ids, const void *table, int64_t ts, void *out, int64_t os, int64_t n,
                             int32_t dim, float scale)
{
    switch (ve) {
    case 8:
        if constexpr (sizeof(TI) == 2 || sizeof(TO) == 2) { launch_lookup<TI, TO, 8>(s, ids, table, ts, out, os, n, dim, scale); break; }
    case 4: launch_lookup<TI, TO, 4>(s, ids, table, ts, out, os, n, dim, scale); break;
    case 2: launch_lookup<TI, TO, 2>(s, ids, table, ts, out, os, n, dim, scale); break;
    default: launch_lookup<TI, TO, 1>(s, ids, table, ts, out, os, n, dim, scale); break;
    }
}

template <typename TI>
static void launch_lookup_to(int out_dtype, int ve, cudaStream_t s, const Ids &ids, const void *table, int64_t ts, void *out, int64_t os,
                             int64_t n, int32_t dim, float scale)
{
    if (out_dtype == LEGION_F32) launch_lookup_ve<TI, float>(ve, s, ids, table, ts, out, os, n, dim, scale);
    else if (out_dtype == LEGION_F16) launch_lookup_ve<TI, __half>(ve, s, ids, table, ts, out, os, n, dim, scale);
    else launch_lookup_ve<TI, __nv_bfloat16>(ve, s, ids, table, ts, out, os, n, dim, scale);
}

// ---- sort ----------------------------------------------------------------------------------------------------------

constexpr int kRankMax = 8192;   // lists up to here are sorted by counting, in one launch
constexpr int kDigits = 256;

// The place of entry i in the sorted list is the number of entries that come before it: those with a smaller key, and
// those with the same key and a smaller position.  A CTA has 64 entries and a quarter of the list per 64 threads.
// n^2 comparisons, but one launch and no dependence: 8192 entries are 2^26 comparisons over 148 SMs.
__global__ void __launch_bounds__(256) rank_sort_kernel(Ids ids, int n, uint32_t *keys, int32_t *pos)
{
    __shared__ uint32_t tile[1024];
    __shared__ int part[256];
    const int t = threadIdx.x & 63, q = threadIdx.x >> 6;
    const int i = blockIdx.x * 64 + t;
    const uint32_t mine = i < n ? ids.key(i) : 0;
    int before = 0;
    for (int j0 = 0; j0 < n; j0 += 1024) {
        __syncthreads();
        for (int j = threadIdx.x; j < 1024; j += 256) tile[j] = j0 + j < n ? ids.key(j0 + j) : 0xFFFFFFFFu;
        __syncthreads();
        const int lo = j0 + q * 256;
        const uint4 *four = reinterpret_cast<const uint4 *>(tile + q * 256);
        if (lo + 256 <= (int)blockIdx.x * 64) {        // all of them stand before entry i
#pragma unroll 8
            for (int j = 0; j < 64; ++j) {
                const uint4 k = four[j];
                before += (k.x <= mine) + (k.y <= mine) + (k.z <= mine) + (k.w <= mine);
            }
        } else if (lo >= (int)blockIdx.x * 64 + 64) {  // behind it
#pragma unroll 8
            for (int j = 0; j < 64; ++j) {
                const uint4 k = four[j];
                before += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
            }
        } else {
            for (int j = 0; j < 256; ++j) {
                const uint32_t k = tile[q * 256 + j];
                before += (k < mine) || (k == mine && lo + j < i);
            }
        }
    }
    part[threadIdx.x] = before;
    __syncthreads();
    if (q == 0 && i < n) {
        const int at = part[t] + part[t + 64] + part[t + 128] + part[t + 192];
        keys[at] = mine;
        pos[at] = i;
    }
}

// Longer lists: least significant digit first, 8 bits a pass, every CTA one contiguous part of the list.
struct SortPass {
    Ids ids;                  // first pass: the ids themselves
    const uint32_t *keys_in;  // later ones: the pairs
    const int32_t *pos_in;
    uint32_t *keys_out;
    int32_t *pos_out;
    int32_t *counts;          // [CTA][digit]
    int64_t n, part;          // entries, entries per CTA
    int32_t shift;
    __device__ __forceinline__ uint32_t key(int64_t i) const { return keys_in != nullptr ? keys_in[i] : ids.key(i); }
};

__global__ void __launch_bounds__(1024) sort_count_kernel(SortPass p)
{
    __shared__ int32_t hist[kDigits];
    if (threadIdx.x < kDigits) hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t lo = blockIdx.x * p.part, hi = min(p.n, lo + p.part);
    for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) atomicAdd(&hist[(p.key(i) >> p.shift) & (kDigits - 1)], 1);
    __syncthreads();
    if (threadIdx.x < kDigits) p.counts[blockIdx.x * kDigits + threadIdx.x] = hist[threadIdx.x];
}

__global__ void __launch_bounds__(1024) sort_scatter_kernel(SortPass p)
{
    __shared__ int32_t whist[32][kDigits];  // per warp: entries of a digit, then where its first one goes
    __shared__ int32_t base[kDigits];
    __shared__ int32_t warp_sum[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int d = threadIdx.x & (kDigits - 1), g = threadIdx.x >> 8;
    // entries of smaller digits, and of the same digit in the parts before this one
    int total = 0, before = 0;
#pragma unroll 8
    for (int c = g; c < (int)gridDim.x; c += 4) {
        const int v = p.counts[c * kDigits + d];
        total += v;
        before += c < (int)blockIdx.x ? v : 0;
    }
    whist[g][d] = total;
    whist[4 + g][d] = before;
    __syncthreads();
    int incl = 0, mine = 0;
    if (threadIdx.x < kDigits) {
        mine = whist[0][d] + whist[1][d] + whist[2][d] + whist[3][d];
        before = whist[4][d] + whist[5][d] + whist[6][d] + whist[7][d];
        incl = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(kFull, incl, s);
            if (lane >= s) incl += v;
        }
        if (lane == 31) warp_sum[warp] = incl;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
        for (int w = 0; w < warp; ++w) incl += warp_sum[w];
        base[d] = incl - mine + before;
    }
    const int64_t lo = blockIdx.x * p.part, hi = min(p.n, lo + p.part);
    for (int64_t i0 = lo; i0 < hi; i0 += 1024) {
        __syncthreads();
        for (int k = threadIdx.x; k < 32 * kDigits; k += 1024) (&whist[0][0])[k] = 0;
        __syncthreads();
        const int64_t i = i0 + threadIdx.x;
        const bool in = i < hi;
        const uint32_t key = in ? p.key(i) : 0u;
        const int32_t at = in ? (p.pos_in != nullptr ? p.pos_in[i] : (int32_t)i) : 0;
        const int digit = in ? (int)((key >> p.shift) & (kDigits - 1)) : kDigits;  // no entry: a digit of its own
        const unsigned same = __match_any_sync(kFull, digit);
        const int rank = __popc(same & ((1u << lane) - 1u));
        if (in && rank == 0) whist[warp][digit] = __popc(same);
        __syncthreads();
        if (threadIdx.x < kDigits) {
            int run = base[d];
#pragma unroll 8
            for (int w = 0; w < 32; ++w) {
                const int v = whist[w][d];
                whist[w][d] = run;
                run += v;
            }
            base[d] = run;
        }
        __syncthreads();
        if (in) {
            const int to = whist[warp][digit] + rank;
            p.keys_out[to] = key;
            p.pos_out[to] = at;
        }
    }
}

// ---- sums over the sorted list -------------------------------------------------------------------------------------

struct Sorted {
    const uint32_t *keys;
    const int32_t *pos;
    int64_t n;
    uint32_t n_nodes;     // the key of what is left out; such entries are the last ones
    int32_t stretch;      // entries that a group of threads sums
    int64_t stretches;
};

// heads[c] = entries of stretch c that are the first of their id
__global__ void __launch_bounds__(256) head_count_kernel(Sorted l, int32_t *heads)
{
    const int64_t c = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (c >= l.stretches) return;
    int count = 0;
    for (int64_t i = c * l.stretch + lane; i < min(l.n, (c + 1) * l.stretch); i += 32) {
        const uint32_t k = l.keys[i];
        count += k < l.n_nodes && (i == 0 || l.keys[i - 1] != k);
    }
    count = __reduce_add_sync(kFull, count);
    if (lane == 0) heads[c] = count;
}

// heads[c] = first entries before stretch c; heads[stretches] and count[0] = all of them.  One CTA.
__global__ void __launch_bounds__(1024) head_scan_kernel(int32_t *heads, int64_t stretches, int32_t *count)
{
    __shared__ int32_t warp_sum[32];
    __shared__ int32_t carry;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) carry = 0;
    for (int64_t c0 = 0; c0 < stretches; c0 += 1024) {
        __syncthreads();
        const int64_t c = c0 + threadIdx.x;
        const int mine = c < stretches ? heads[c] : 0;
        int incl = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(kFull, incl, s);
            if (lane >= s) incl += v;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        const int before = carry + __reduce_add_sync(kFull, lane < warp ? warp_sum[lane] : 0);
        if (c < stretches) heads[c] = before + incl - mine;
        __syncthreads();
        if (threadIdx.x == 1023) carry = before + incl;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        heads[stretches] = carry;
        count[0] = carry;
    }
}

struct GradOut {
    void *rows;           // gradient of the table, or of the rows that occur
    int64_t stride;
    int32_t dtype;
    int32_t accumulate;
    const int32_t *heads; // rows that occur: first entries before every stretch; whole table: nullptr
    void *unique;         // rows that occur: their ids
    int32_t wide;
    float scale;
    int32_t dim;
    float *head_part, *tail_part;  // [stretch][dim]: what an id that crosses a boundary has in a stretch

    template <int VE>
    __device__ __forceinline__ void put(int64_t row, int col, const float *acc) const
    {
        float x[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) x[i] = acc[i] * scale;
        const int64_t at = row * stride + col;
        if (dtype == LEGION_F32) put_as<VE>(static_cast<float *>(rows) + at, x);
        else if (dtype == LEGION_F16) put_as<VE>(static_cast<__half *>(rows) + at, x);
        else put_as<VE>(static_cast<__nv_bfloat16 *>(rows) + at, x);
    }
    template <int VE, typename T>
    __device__ __forceinline__ void put_as(T *p, float *x) const
    {
        Vec<T, VE> v;
        if (accumulate) {  // the sum so far and the new part are added in fp32 and rounded once
            v.load(p);
#pragma unroll
            for (int i = 0; i < VE; ++i) x[i] += v.get(i);
        }
        v.set(x);
        v.store(p);
    }
};

// 2^log_group threads have a stretch, one vector of VE columns each.  What bounds it is HBM: the rows of the gradient are read
// once, `kAhead` of them in flight per thread, whatever ids they belong to; only the additions go one after the other.
template <typename T, int VE>
__global__ void __launch_bounds__(256)
grad_sum_kernel(Sorted l, const T *__restrict__ grad, int64_t grad_stride, GradOut o, int log_group)
{
    constexpr int kAhead = 8;
    const int group = threadIdx.x >> log_group;
    const int col = ((int)blockIdx.y * 256 + (threadIdx.x & ((1 << log_group) - 1))) * VE;
    const int64_t c = ((int64_t)blockIdx.x << (8 - log_group)) + group;
    if (c >= l.stretches || col >= o.dim) return;
    const int64_t lo = c * l.stretch, hi = min(l.n, lo + l.stretch);
    const uint32_t prev = lo > 0 ? l.keys[lo - 1] : 0xFFFFFFFFu;
    uint32_t cur = l.keys[lo];
    if (cur >= l.n_nodes) return;
    bool open = prev == cur;                   // the id began in a stretch before
    int32_t seg = o.heads != nullptr ? o.heads[c] - (open ? 1 : 0) : 0;
    float acc[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
    auto flush = [&]() {
        if (open) {
            float *p = o.head_part + c * o.dim + col;
#pragma unroll
            for (int i = 0; i < VE; ++i) p[i] = acc[i];
        } else {
            o.put<VE>(o.heads != nullptr ? seg : (int64_t)cur, col, acc);
        }
    };
    auto name = [&]() {
        if (o.unique != nullptr && col == 0 && !open) {
            if (o.wide) static_cast<int64_t *>(o.unique)[seg] = cur;
            else static_cast<int32_t *>(o.unique)[seg] = (int32_t)cur;
        }
    };
    name();
    for (int64_t i0 = lo; i0 < hi; i0 += kAhead) {
        uint32_t key[kAhead];
        Vec<T, VE> v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            key[j] = i0 + j < hi ? l.keys[i0 + j] : l.n_nodes;
            if (key[j] < l.n_nodes) v[j].load_stream(grad + (int64_t)l.pos[i0 + j] * grad_stride + col);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (key[j] >= l.n_nodes) continue;  // behind the last entry
            if (key[j] != cur) {
                flush();
                cur = key[j];
                open = false;
                ++seg;
                name();
#pragma unroll
                for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) acc[i] += v[j].get(i);
        }
    }
    if (hi < l.n && l.keys[hi] == cur) {
        float *p = o.tail_part + c * o.dim + col;
#pragma unroll
        for (int i = 0; i < VE; ++i) p[i] = acc[i];
    } else {
        flush();
    }
}

// The ids that cross boundaries: the CTA of the stretch where such an id begins adds its pieces, eight threads a column, each
// every eighth piece, then their eight sums: one fixed order.
__global__ void __launch_bounds__(256) grad_join_kernel(Sorted l, GradOut o)
{
    const int64_t c = blockIdx.x, lo = c * l.stretch, hi = lo + l.stretch;
    if (hi >= l.n) return;
    const uint32_t k = l.keys[hi - 1];
    if (k >= l.n_nodes || l.keys[hi] != k || (lo > 0 && l.keys[lo - 1] == k)) return;
    int64_t a = hi, b = l.n;   // first entry behind the id
    while (a < b) {
        const int64_t m = (a + b) / 2;
        if (l.keys[m] <= k) a = m + 1;
        else b = m;
    }
    const int64_t last = (a - 1) / l.stretch;
    const int64_t row = o.heads != nullptr ? o.heads[c + 1] - 1 : (int64_t)k;
    __shared__ float part[8][32];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int col0 = blockIdx.y * 32; col0 < o.dim; col0 += gridDim.y * 32) {
        const int col = col0 + x;
        float acc = 0.0f;
        if (col < o.dim)
#pragma unroll 4
            for (int64_t s = c + y; s <= last; s += 8) acc += (s == last ? o.head_part : o.tail_part)[s * o.dim + col];
        part[y][x] = acc;
        __syncthreads();
        if (y == 0 && col < o.dim) {
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) sum += part[w][x];
            o.put<1>(row, col, &sum);
        }
        __syncthreads();
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------

static int32_t stretch_of(int64_t n) { return n <= 65536 ? 32 : (n <= 524288 ? 64 : 128); }

struct GradScratch {
    uint32_t *keys[2];
    int32_t *pos[2], *counts, *heads;
    float *head_part, *tail_part;
    int64_t bytes;
    GradScratch(uint8_t *base, int64_t n, int64_t dim)
    {
        bytes = 0;
        auto take = [&](int64_t b) {
            uint8_t *p = base + bytes;
            bytes += (b + 255) / 256 * 256;
            return p;
        };
        const int64_t stretches = (n + stretch_of(n) - 1) / stretch_of(n);
        for (int k = 0; k < 2; ++k) {
            keys[k] = (uint32_t *)take(4 * n);
            pos[k] = (int32_t *)take(4 * n);
        }
        counts = (int32_t *)take((int64_t)kSms * kDigits * 4);
        heads = (int32_t *)take(4 * (stretches + 1));
        head_part = (float *)take(stretches > 1 ? 4 * stretches * dim : 0);
        tail_part = (float *)take(stretches > 1 ? 4 * stretches * dim : 0);
    }
};

static int sort_ids(cudaStream_t s, const Ids &ids, int64_t n, const GradScratch &w, Sorted *l)
{
    l->n = n;
    l->n_nodes = (uint32_t)ids.n_nodes;
    l->stretch = stretch_of(n);
    l->stretches = (n + l->stretch - 1) / l->stretch;
    if (n <= kRankMax) {
        rank_sort_kernel<<<(unsigned)((n + 63) / 64), 256, 0, s>>>(ids, (int)n, w.keys[0], w.pos[0]);
        l->keys = w.keys[0];
        l->pos = w.pos[0];
        LG_LAUNCH_CHECK();
        return LEGION_OK;
    }
    int bits = 0;
    while ((ids.n_nodes >> bits) != 0) ++bits;  // n_nodes itself is a key
    SortPass p;
    p.ids = ids;
    p.counts = w.counts;
    p.n = n;
    const int64_t ctas = (n + 1023) / 1024 < kSms ? (n + 1023) / 1024 : kSms;
    p.part = (n + ctas - 1) / ctas;
    int to = 0;
    for (p.shift = 0; p.shift < bits; p.shift += 8, to ^= 1) {
        p.keys_in = p.shift == 0 ? nullptr : w.keys[to ^ 1];
        p.pos_in = p.shift == 0 ? nullptr : w.pos[to ^ 1];
        p.keys_out = w.keys[to];
        p.pos_out = w.pos[to];
        sort_count_kernel<<<(unsigned)ctas, 1024, 0, s>>>(p);
        sort_scatter_kernel<<<(unsigned)ctas, 1024, 0, s>>>(p);
    }
    l->keys = w.keys[to ^ 1];
    l->pos = w.pos[to ^ 1];
    LG_LAUNCH_CHECK();
    return LEGION_OK;
}

template <typename T>
static void launch_sum(int ve, cudaStream_t s, const Sorted &l, const void *grad, int64_t stride, const GradOut &o)
{
    const int vecs = o.dim / ve;
    int log_group = 0;
    while (log_group < 8 && (1 << log_group) < vecs) ++log_group;
    const int64_t per = 256 >> log_group;
    const dim3 grid((unsigned)((l.stretches + per - 1) / per), (unsigned)((vecs + 255) / 256));
    switch (ve) {
    case 8:
        if constexpr (sizeof(T) == 2) { grad_sum_kernel<T, 8><<<grid, 256, 0, s>>>(l, (const T *)grad, stride, o, log_group); break; }
    case 4: grad_sum_kernel<T, 4><<<grid, 256, 0, s>>>(l, (const T *)grad, stride, o, log_group); break;
    case 2: grad_sum_kernel<T, 2><<<grid, 256, 0, s>>>(l, (const T *)grad, stride, o, log_group); break;
    default: grad_sum_kernel<T, 1><<<grid, 256, 0, s>>>(l, (const T *)grad, stride, o, log_group); break;
    }
}

static int run_grad(cudaStream_t s, const Ids &ids, int64_t n, const void *grad, int32_t grad_dtype, int64_t grad_stride, GradOut o,
                    const GradScratch &w, int32_t *count)
{
    Sorted l;
    int rc = sort_ids(s, ids, n, w, &l);
    if (rc != LEGION_OK) return rc;
    o.head_part = w.head_part;
    o.tail_part = w.tail_part;
    if (count != nullptr) {
        head_count_kernel<<<(unsigned)((l.stretches + 7) / 8), 256, 0, s>>>(l, w.heads);
        head_scan_kernel<<<1, 1024, 0, s>>>(w.heads, l.stretches, count);
        o.heads = w.heads;
    }
    // what a vector may have: the loads of the gradient are at most 16 bytes, and every address is a multiple of it
    const int ve = common_vector(grad_dtype == LEGION_F32 ? 4 : 8,
                                 { o.dim, grad_stride, aligned_elements(grad, grad_dtype), o.stride, aligned_elements(o.rows, o.dtype) });
    if (grad_dtype == LEGION_F32) launch_sum<float>(ve, s, l, grad, grad_stride, o);
    else if (grad_dtype == LEGION_F16) launch_sum<__half>(ve, s, l, grad, grad_stride, o);
    else launch_sum<__nv_bfloat16>(ve, s, l, grad, grad_stride, o);
    if (l.stretches > 1)
        grad_join_kernel<<<dim3((unsigned)l.stretches, (unsigned)(o.dim < 512 ? 1 : (o.dim / 512 > 16 ? 16 : o.dim / 512))), 256, 0, s>>>(l, o);
    LG_LAUNCH_CHECK();
    return LEGION_OK;
}

}  // namespace legion

using namespace legion;

#define LG_ROWS(p, dtype, dim, stride, n, what)                                                                                 \
    LG_ARG(dtype_known(dtype), what ": dtype must be LEGION_F32, LEGION_F16 or LEGION_BF16");                                   \
    LG_ARG((n) == 0 || (p) != nullptr, what " is NULL");                                                                        \
    LG_ARG((stride) >= (dim) && (stride) <= (1ll << 40), what ": a row's stride must be at least its length");                  \
    LG_ARG((uintptr_t)(p) % dtype_bytes(dtype) == 0, what " must start on a multiple of its element's size")

static int check_ids(const void *ids, int32_t id_bytes, int64_t n_ids, int64_t n_nodes, int32_t dim)
{
    LG_ARG(n_ids >= 0 && n_ids <= LEGION_MAX_IDS, "n_ids out of range");
    LG_ARG(n_ids == 0 || ids != nullptr, "ids is NULL");
    LG_ARG(id_bytes == 4 || id_bytes == 8, "ids must be 4 or 8 bytes wide");
    LG_ARG((uintptr_t)ids % id_bytes == 0, "ids must start on a multiple of their width");
    LG_ARG(n_nodes > 0 && n_nodes < (1ll << 31), "n_nodes must fit int32");
    LG_ARG(dim > 0 && dim <= LEGION_MAX_DIM, "dim out of range");
    return LEGION_OK;
}

extern "C" int legion_embedding_lookup(int32_t dev_id, const void *table, int32_t table_dtype, int64_t table_stride, int64_t n_nodes,
                                       const void *ids, int32_t id_bytes, int64_t n_ids, int32_t dim, float scale, void *out,
                                       int32_t out_dtype, int64_t out_stride, void *stream)
{
    int rc = check_ids(ids, id_bytes, n_ids, n_nodes, dim);
    if (rc != LEGION_OK) return rc;
    LG_ROWS(table, table_dtype, dim, table_stride, n_nodes, "table");
    LG_ROWS(out, out_dtype, dim, out_stride, n_ids, "out");
    if (n_ids == 0) return LEGION_OK;
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    const Ids list{ ids, id_bytes == 8, n_nodes };
    const int ve = common_vector(table_dtype == LEGION_F32 && out_dtype == LEGION_F32 ? 4 : 8,
                                 { dim, table_stride, out_stride, aligned_elements(table, table_dtype), aligned_elements(out, out_dtype) });
    cudaStream_t s = (cudaStream_t)stream;
    if (table_dtype == LEGION_F32) launch_lookup_to<float>(out_dtype, ve, s, list, table, table_stride, out, out_stride, n_ids, dim, scale);
    else if (table_dtype == LEGION_F16) launch_lookup_to<__half>(out_dtype, ve, s, list, table, table_stride, out, out_stride, n_ids, dim, scale);
    else launch_lookup_to<__nv_bfloat16>(out_dtype, ve, s, list, table, table_stride, out, out_stride, n_ids, dim, scale);
    LG_LAUNCH_CHECK();
    return LEGION_OK;
}

extern "C" int legion_embedding_grad_workspace(int64_t n_ids, int32_t dim, int64_t n_nodes, int64_t *bytes)
{
    LG_ARG(bytes != nullptr, "bytes is NULL");
    LG_ARG(n_ids >= 0 && n_ids <= LEGION_MAX_IDS, "n_ids out of range");
    LG_ARG(n_nodes > 0 && n_nodes < (1ll << 31), "n_nodes must fit int32");
    LG_ARG(dim > 0 && dim <= LEGION_MAX_DIM, "dim out of range");
    *bytes = GradScratch(nullptr, n_ids, dim).bytes;
    return LEGION_OK;
}

static int check_workspace(const void *workspace, int64_t bytes, int64_t need)
{
    LG_ARG(workspace != nullptr || need == 0, "workspace is NULL");
    LG_ARG((uintptr_t)workspace % 16 == 0, "workspace must start on a multiple of 16 bytes");
    LG_ARG(bytes >= need, "workspace is smaller than the call asks for");
    return LEGION_OK;
}

extern "C" int legion_embedding_grad(int32_t dev_id, const void *ids, int32_t id_bytes, int64_t n_ids, const void *grad_out,
                                     int32_t grad_dtype, int64_t grad_stride, int32_t dim, float scale, void *grad_table,
                                     int32_t table_dtype, int64_t table_stride, int64_t n_nodes, int32_t accumulate, void *workspace,
                                     int64_t workspace_bytes, void *stream)
{
    int rc = check_ids(ids, id_bytes, n_ids, n_nodes, dim);
    if (rc != LEGION_OK) return rc;
    LG_ROWS(grad_out, grad_dtype, dim, grad_stride, n_ids, "grad_out");
    LG_ROWS(grad_table, table_dtype, dim, table_stride, n_nodes, "grad_table");
    const GradScratch w((uint8_t *)workspace, n_ids, dim);
    if (n_ids > 0 && (rc = check_workspace(workspace, workspace_bytes, w.bytes)) != LEGION_OK) return rc;
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    cudaStream_t s = (cudaStream_t)stream;
    const size_t width = (size_t)dim * dtype_bytes(table_dtype);
    if (!accumulate) {
        if (table_stride == dim) LG_CUDA(cudaMemsetAsync(grad_table, 0, width * (size_t)n_nodes, s));
        else LG_CUDA(cudaMemset2DAsync(grad_table, (size_t)table_stride * dtype_bytes(table_dtype), 0, width, (size_t)n_nodes, s));
    }
    if (n_ids == 0) return LEGION_OK;
    GradOut o{};
    o.rows = grad_table;
    o.stride = table_stride;
    o.dtype = table_dtype;
    o.accumulate = accumulate != 0;
    o.scale = scale;
    o.dim = dim;
    return run_grad(s, Ids{ ids, id_bytes == 8, n_nodes }, n_ids, grad_out, grad_dtype, grad_stride, o, w, nullptr);
}

extern "C" int legion_embedding_grad_rows(int32_t dev_id, const void *ids, int32_t id_bytes, int64_t n_ids, const void *grad_out,
                                          int32_t grad_dtype, int64_t grad_stride, int32_t dim, float scale, int64_t n_nodes,
                                          void *unique_ids, float *grad_rows, int64_t rows_stride, int32_t *count, void *workspace,
                                          int64_t workspace_bytes, void *stream)
{
    int rc = check_ids(ids, id_bytes, n_ids, n_nodes, dim);
    if (rc != LEGION_OK) return rc;
    LG_ROWS(grad_out, grad_dtype, dim, grad_stride, n_ids, "grad_out");
    LG_ROWS(grad_rows, LEGION_F32, dim, rows_stride, n_ids, "grad_rows");
    LG_ARG(count != nullptr && (uintptr_t)count % 4 == 0, "count is NULL");
    LG_ARG(n_ids == 0 || (unique_ids != nullptr && (uintptr_t)unique_ids % id_bytes == 0), "unique_ids is NULL");
    const GradScratch w((uint8_t *)workspace, n_ids, dim);
    if (n_ids > 0 && (rc = check_workspace(workspace, workspace_bytes, w.bytes)) != LEGION_OK) return rc;
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    cudaStream_t s = (cudaStream_t)stream;
    if (n_ids == 0) {
        LG_CUDA(cudaMemsetAsync(count, 0, 4, s));
        return LEGION_OK;
    }
    GradOut o{};
    o.rows = grad_rows;
    o.stride = rows_stride;
    o.dtype = LEGION_F32;
    o.unique = unique_ids;
    o.wide = id_bytes == 8;
    o.scale = scale;
    o.dim = dim;
    return run_grad(s, Ids{ ids, id_bytes == 8, n_nodes }, n_ids, grad_out, grad_dtype, grad_stride, o, w, count);
}
