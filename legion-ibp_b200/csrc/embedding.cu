// Learned rows: lookup by id with a scale, and the gradient by sorted ids.
//
//   out[i]  = scale * table[ids[i]]                       (an id outside the table: a row of zeros)
//   grad[v] = scale * sum over i with ids[i] = v of g[i]  (whole table, or only the rows of the ids that occur)
//
// The gradient sorts (id, position) pairs (stable), cuts the sorted list into stretches of equal length and lets a group
// of threads sum the rows of a stretch in list order.  A stretch writes the sums of the ids that lie wholly inside it;
// what an id that crosses a boundary has in a stretch goes to scratch, and a second launch adds these pieces in
// list order.  So a stretch takes the same time whatever ids it has, each gradient row is read once, and the result does not depend
// on the order in which the CTAs run: no atomics on floats.  What an id of many stretches costs beyond that is the joining of its pieces by
// one CTA per 128 vectors (16,384 rows of 2048 bf16 into 32,000: 90 us of different ids, 164 of one).
#include "typed.cuh"

#include <cmath>

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

// The rows as one flat run of vectors, R vectors of 256 threads each per CTA.  Bound by HBM: 200,000 rows of 400 bytes out of 980 MB
// 32.8 us, where the rows touch 464 bytes of 64-byte bursts each on average (27 us at the rate of a copy); 30,000 rows of 4096 bytes 35 us.
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

// Rows whose vectors are only 2 or 4 bytes wide (odd lengths): a warp has up to 256 vectors of one row, so that the place of a vector costs
// no division: what bounds such rows is the instructions.  100,000 rows of 333 fp16: 76 us as a flat
// run, 43 like this.
template <typename TI, typename TO, int VE>
__global__ void __launch_bounds__(256)
lookup_rows_kernel(Ids ids, const TI *__restrict__ table, int64_t table_stride, TO *__restrict__ out, int64_t out_stride, int64_t n, int vecs,
                   int per_warp, float scale)
{
    constexpr int U = 8;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= n) return;
    const uint32_t key = ids.key(row);
    const int first = blockIdx.y * per_warp + (threadIdx.x & 31), end = min(vecs, (int)(blockIdx.y + 1) * per_warp);
    const TI *src = table + (int64_t)key * table_stride;
    Vec<TI, VE> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        v[u].zero();
        if (first + u * 32 < end && key < (uint32_t)ids.n_nodes) v[u].load(src + (first + u * 32) * VE);
    }
    TO *dst = out + row * out_stride;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (first + u * 32 >= end) break;
        float x[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) x[i] = v[u].get(i) * scale;
        Vec<TO, VE> o;
        o.set(x);
        o.store(dst + (first + u * 32) * VE);
    }
}

template <typename TI, typename TO, int VE>
static void launch_lookup(cudaStream_t s, const Ids &ids, const void *table, int64_t table_stride, void *out, int64_t out_stride,
                          int64_t n, int32_t dim, float scale)
{
    const int64_t total = n * (dim / VE);
    const FastDiv per_row((uint32_t)(dim / VE));
    if constexpr (VE * sizeof(TI) <= 4 && VE * sizeof(TO) <= 4) {
        const int vecs = dim / VE, chunks = (vecs + 255) / 256, per_warp = ((vecs + chunks - 1) / chunks + 31) / 32 * 32;
        if (vecs >= 32) {
            lookup_rows_kernel<TI, TO, VE><<<dim3((unsigned)((n + 7) / 8), (unsigned)((vecs + per_warp - 1) / per_warp)), 256, 0, s>>>(
                ids, (const TI *)table, table_stride, (TO *)out, out_stride, n, vecs, per_warp, scale);
            return;
        }
    }
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

constexpr int kDigits = 256;
constexpr int kClusterThreads = 1024;
constexpr int kClusterItems = 4;                             // entries that a thread has at most
constexpr int kClusterPart = kClusterItems * kClusterThreads; // entries that a CTA has at most
constexpr int64_t kClusterList = 20480;   // longest list that a cluster sorts (16384 ids: 30 us a call, 31 by the passes below; 32768: 33 and 32)
constexpr int kHistPitch = kDigits + 1;                      // the 32 counts of a digit lie in 32 banks

// The rows of the gradient that no id names are zeros: a launch of its own writes them, all rows (those that are named are written again by
// the sums), and the sort inside a cluster runs beside it.
struct ZeroFill {
    uint8_t *p;            // nullptr: nothing to fill
    int64_t rows, width, pitch;  // bytes of a row, bytes from row to row
};

// `threads` threads write `bytes` zero bytes from p on (both multiples of two).
__device__ __forceinline__ void zero_run(uint8_t *p, int64_t bytes, int64_t at, int64_t threads)
{
    int64_t head = (16 - ((uintptr_t)p & 15)) & 15;
    if (head > bytes) head = bytes;
    const int64_t vecs = (bytes - head) / 16, tail = bytes - head - vecs * 16;
    if (at * 2 < head) reinterpret_cast<uint16_t *>(p)[at] = 0;
    uint4 *v = reinterpret_cast<uint4 *>(p + head);
    for (int64_t i = at; i < vecs; i += threads) __stcs(v + i, make_uint4(0, 0, 0, 0));
    if (at * 2 < tail) reinterpret_cast<uint16_t *>(p + head + vecs * 16)[at] = 0;
}
__device__ __forceinline__ void zero_fill(const ZeroFill &z, int64_t at, int64_t threads)
{
    if (z.pitch == z.width) {
        zero_run(z.p, z.rows * z.width, at, threads);
    } else {
        for (int64_t r = at >> 5; r < z.rows; r += threads >> 5) zero_run(z.p + r * z.pitch, z.width, at & 31, 32);
    }
}

// Lanes of the warp whose digit is this lane's, by one vote a bit (a match instruction takes a step per different digit).
__device__ __forceinline__ unsigned same_digit(int digit, bool in)
{
    unsigned same = __ballot_sync(kFull, in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const unsigned ones = __ballot_sync(kFull, (digit >> b) & 1);
        same &= (digit >> b) & 1 ? ones : ~ones;
    }
    return same;
}

// Bound by HBM's writes: 7 TB/s with four CTAs on every SM (112 CTAs of the sort's own launch wrote 4.8).
__global__ void __launch_bounds__(256) zero_fill_kernel(ZeroFill z)
{
    cudaTriggerProgrammaticLaunchCompletion();
    zero_fill(z, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

// Rows of a lookup whose ids are outside the table, a warp a row, behind a lookup by a scale that does not leave zeros as they are (choosing
// the scale vector by vector in the lookup itself took registers from loads: 30,000 rows of 4096 bytes 37.1 us for 35.8).
__global__ void __launch_bounds__(256) zero_outside_kernel(Ids ids, int64_t n, uint8_t *out, int64_t width, int64_t pitch)
{
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row < n && ids.key(row) == (uint32_t)ids.n_nodes) zero_run(out + row * pitch, width, threadIdx.x & 31, 32);
}

struct ClusterSort {
    Ids ids;
    int32_t n, part;      // entries; entries per CTA, a multiple of kClusterThreads
    FastDiv per_part;
    int32_t bits;
    uint2 *pairs;         // sorted: (key, position)
    int32_t *heads;       // rows that occur: first entries before every stretch (GradOut), or nullptr
    int32_t *count;
    int32_t stretch;      // a multiple of 32
};

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of the same shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(const void *p, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ int32_t load_cta(uint32_t a)
{
    int32_t v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void store_cta(uint32_t a, uint2 v)
{
    asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(a), "r"(v.x), "r"(v.y) : "memory");
}

__host__ __device__ constexpr int64_t cluster_sort_smem(int64_t part) { return part * 16 + 4 * (32 * kHistPitch + 2 * kDigits + 80); }

// Stable sort by least significant digit, eight bits a pass, inside the shared memory of one cluster: no launch and no global memory
// between the passes.  A warp has 32 * items entries one behind the other and ranks them in list order; counts of
// the CTAs' digits are read out of each other's shared memory, entries are written straight to the CTA that has their place.
// What bounds it is latency (two cluster barriers a pass), so the entries are spread over up to 16 CTAs even when one could hold them.
// It does not wait for the launch before it, the zero rows, until its own work is done: what follows it may write over them.
__global__ void __launch_bounds__(kClusterThreads, 1) cluster_sort_kernel(ClusterSort p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t size = cluster_size();
    cudaTriggerProgrammaticLaunchCompletion();
    const uint32_t me = cluster_rank();
    uint2 *buf[2] = { reinterpret_cast<uint2 *>(smem), reinterpret_cast<uint2 *>(smem) + p.part };
    int32_t *hist = reinterpret_cast<int32_t *>(buf[1] + p.part);  // [warp][digit]
    int32_t *total = hist + 32 * kHistPitch;                       // entries of each digit in this CTA; read by the others
    int32_t *base = total + kDigits;                               // where the CTA's first entry of a digit goes
    int32_t *scan = base + kDigits;                                // 32 words and a word that the others read
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int first = (int)me * p.part, mine = max(0, min(p.part, p.n - first));
    const int items = p.part / kClusterThreads;
    const int at0 = warp * 32 * items + lane;                      // the lane's first entry; the next ones are 32 apart
    for (int i = threadIdx.x; i < mine; i += kClusterThreads) buf[0][i] = make_uint2(p.ids.key(first + i), (uint32_t)(first + i));
    int cur = 0;
    for (int shift = 0; shift < p.bits; shift += 8, cur ^= 1) {
        for (int i = threadIdx.x; i < 32 * kHistPitch; i += kClusterThreads) hist[i] = 0;
        __syncthreads();
        uint16_t rank[kClusterItems];  // among the warp's entries of the same digit
#pragma unroll
        for (int j = 0; j < kClusterItems; ++j) {
            if (j < items) {
                const int i = at0 + j * 32;
                const bool in = i < mine;
                const int digit = in ? (int)((buf[cur][i].x >> shift) & (kDigits - 1)) : 0;
                const unsigned same = same_digit(digit, in);
                const int before = hist[warp * kHistPitch + digit];
                __syncwarp();
                const int among = __popc(same & ((1u << lane) - 1u));
                if (in && among == 0) hist[warp * kHistPitch + digit] = before + __popc(same);
                __syncwarp();
                rank[j] = (uint16_t)(before + among);
            }
        }
        __syncthreads();
        {   // counts of the warps -> entries of the digit in the warps before; four threads a digit, eight warps each
            const int d = threadIdx.x >> 2, q = threadIdx.x & 3;
            int v[8], sum = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = hist[(q * 8 + k) * kHistPitch + d];
                sum += v[k];
            }
            int incl = sum;
            int o = __shfl_up_sync(kFull, incl, 1, 4);
            if (q >= 1) incl += o;
            o = __shfl_up_sync(kFull, incl, 2, 4);
            if (q >= 2) incl += o;
            int run = incl - sum;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                hist[(q * 8 + k) * kHistPitch + d] = run;
                run += v[k];
            }
            if (q == 3) total[d] = incl;
        }
        cluster_sync();
        {   // entries of smaller digits anywhere, and of the same digit in the CTAs before; four threads a digit
            const int d = threadIdx.x >> 2, q = threadIdx.x & 3;
            int all = 0, before = 0;
            for (uint32_t c = q; c < size; c += 4) {
                const int v = load_cta(in_cta(total + d, c));
                all += v;
                before += c < me ? v : 0;
            }
            all += __shfl_xor_sync(kFull, all, 1);
            all += __shfl_xor_sync(kFull, all, 2);
            before += __shfl_xor_sync(kFull, before, 1);
            before += __shfl_xor_sync(kFull, before, 2);
            int incl = q == 0 ? all : 0;   // sum over the digits up to d
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const int o = __shfl_up_sync(kFull, incl, s);
                if (lane >= s) incl += o;
            }
            if (lane == 31) scan[warp] = incl;
            __syncthreads();
            const int warps_before = __reduce_add_sync(kFull, lane < warp ? scan[lane] : 0);
            if (q == 0) base[d] = warps_before + incl - all + before;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kClusterItems; ++j) {
            const int i = at0 + j * 32;
            if (j < items && i < mine) {
                const uint2 e = buf[cur][i];
                const int digit = (int)((e.x >> shift) & (kDigits - 1));
                const uint32_t to = (uint32_t)(base[digit] + hist[warp * kHistPitch + digit] + rank[j]);
                const uint32_t cta = p.per_part.div(to);
                store_cta(in_cta(buf[cur ^ 1] + (to - cta * (uint32_t)p.part), cta), e);
            }
        }
        cluster_sync();
    }
    const uint2 *sorted = buf[cur];
    for (int i = threadIdx.x; i < mine; i += kClusterThreads) p.pairs[first + i] = sorted[i];
    if (p.heads != nullptr) {
        // first entries of 32 entries each: at most kClusterPart / 32 counts, one thread each
        const int pieces = p.part / 32;
        int32_t *count = hist;
        for (int k = warp; k < pieces; k += 32) {
            const int i = k * 32 + lane;
            bool head = i < mine && sorted[i].x < (uint32_t)p.ids.n_nodes;
            if (head && first + i > 0)
                head = sorted[i].x != (i > 0 ? sorted[i - 1].x : (uint32_t)load_cta(in_cta(&sorted[p.part - 1].x, me - 1)));
            const unsigned all = __ballot_sync(kFull, head);
            if (lane == 0) count[k] = __popc(all);
        }
        __syncthreads();
        const int c = threadIdx.x < pieces ? count[threadIdx.x] : 0;
        int incl = c;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(kFull, incl, s);
            if (lane >= s) incl += o;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        const int of_cta = __reduce_add_sync(kFull, scan[lane]);
        const int excl = __reduce_add_sync(kFull, lane < warp ? scan[lane] : 0) + incl - c;
        if (threadIdx.x == 0) scan[32] = of_cta;
        cluster_sync();
        const int before = __reduce_add_sync(kFull, (uint32_t)lane < me ? load_cta(in_cta(scan + 32, lane)) : 0);
        const int i = threadIdx.x * 32;
        if (threadIdx.x < pieces && i < mine && (first + i) % p.stretch == 0) p.heads[(first + i) / p.stretch] = before + excl;
        if (threadIdx.x == 0 && me == size - 1) {
            p.count[0] = before + of_cta;
        }
    }
    cudaGridDependencySynchronize();
    cluster_sync();  // no CTA's memory goes while another one may read it
}

// Longer lists: the same passes over global memory, every CTA one contiguous part of the list.  A pass counts the parts' digits
// and then moves the entries.  Counts are kept for every part and for groups of kGroup parts (whole numbers: the order of the atomics
// changes nothing): a CTA reads those of its group and of the other groups, 25 rows in place of 148 (every CTA reading all
// counts took 14000 of a move's 20000 clocks; counting the next pass's digits by atomics while entries move took 6 us, a launch for
// it 3.5).  What bounds a pass is the chain of latencies in it; the launches are dependents that start while the one before ends.
constexpr int kPassMax = 4;
constexpr int kGroup = 12, kGroups = (kSms + kGroup - 1) / kGroup;
constexpr int kCountRows = kSms + kGroups;   // the parts', then the groups'
__device__ __forceinline__ void count_digit(int32_t *counts, uint32_t part, int digit, int v)
{
    atomicAdd(&counts[part * kDigits + digit], v);
    atomicAdd(&counts[(kSms + part / kGroup) * kDigits + digit], v);
}
struct SortPass {
    Ids ids;                  // first pass: the ids themselves
    const uint2 *in;          // later ones: the pairs
    uint2 *out;
    int32_t *counts;          // [kCountRows][digit] of this pass
    int64_t n;
    int32_t part;             // entries per CTA
    int32_t shift;
    __device__ __forceinline__ uint2 pair(int64_t i) const { return in != nullptr ? in[i] : make_uint2(ids.key(i), (uint32_t)i); }
};

// Counts of all passes and the ticket behind them: zeros.
__global__ void __launch_bounds__(1024) sort_zero_kernel(int32_t *counts, int words)
{
    cudaTriggerProgrammaticLaunchCompletion();
    for (int i = blockIdx.x * 1024 + threadIdx.x; i < words; i += gridDim.x * 1024) counts[i] = 0;
}

__global__ void __launch_bounds__(1024) sort_count_kernel(SortPass p)
{
    __shared__ int32_t hist[kDigits];
    if (threadIdx.x < kDigits) hist[threadIdx.x] = 0;
    cudaTriggerProgrammaticLaunchCompletion();
    if (p.in != nullptr) cudaGridDependencySynchronize();   // the ids are there already
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * p.part, hi = min(p.n, lo + p.part);
    for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) {
        const uint32_t key = p.in != nullptr ? p.in[i].x : p.ids.key(i);
        atomicAdd(&hist[(key >> p.shift) & (kDigits - 1)], 1);
    }
    __syncthreads();
    if (p.in == nullptr) cudaGridDependencySynchronize();
    if (threadIdx.x < kDigits && hist[threadIdx.x] != 0) count_digit(p.counts, blockIdx.x, threadIdx.x, hist[threadIdx.x]);
}

__global__ void __launch_bounds__(1024) sort_scatter_kernel(SortPass p)
{
    __shared__ int32_t whist[32][kHistPitch];  // per warp: entries of a digit, then where its first one goes
    __shared__ int32_t base[kDigits];
    __shared__ int32_t scan[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int k = threadIdx.x; k < 32 * kHistPitch; k += 1024) (&whist[0][0])[k] = 0;
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    const int64_t lo = (int64_t)blockIdx.x * p.part, hi = min(p.n, lo + p.part);
    uint2 e = lo + threadIdx.x < hi ? p.pair(lo + threadIdx.x) : make_uint2(0, 0);
    {   // entries of smaller digits, and of the same digit in the parts before this one; warp w has digits 8 w to 8 w + 7, a quarter
        // of the counts per eight lanes
        const int d = warp * 8 + (lane & 7), q = lane >> 3, group = blockIdx.x / kGroup, in_group = blockIdx.x - group * kGroup;
        int all = 0, before = 0;
#pragma unroll
        for (int j = 0; j < (kGroups + 3) / 4; ++j) {
            const int c = 4 * j + q;
            const int v = c < kGroups ? p.counts[(kSms + c) * kDigits + d] : 0;
            all += v;
            before += c < group ? v : 0;
        }
#pragma unroll
        for (int j = 0; j < kGroup / 4; ++j) {
            const int c = 4 * j + q;
            if (c < in_group) before += p.counts[(group * kGroup + c) * kDigits + d];
        }
        all += __shfl_xor_sync(kFull, all, 8);
        all += __shfl_xor_sync(kFull, all, 16);
        before += __shfl_xor_sync(kFull, before, 8);
        before += __shfl_xor_sync(kFull, before, 16);
        int incl = all;   // over the warp's digits up to this one
#pragma unroll
        for (int s = 1; s < 8; s <<= 1) {
            const int o = __shfl_up_sync(kFull, incl, s, 8);
            if ((lane & 7) >= s) incl += o;
        }
        if (lane == 7) scan[warp] = incl;
        __syncthreads();
        const int warps_before = __reduce_add_sync(kFull, lane < warp ? scan[lane] : 0);
        if (lane < 8) base[d] = warps_before + incl - all + before;
    }
    for (int64_t i0 = lo; i0 < hi; i0 += 1024) {
        const int64_t i = i0 + threadIdx.x;
        const bool in = i < hi;
        const int digit = in ? (int)((e.x >> p.shift) & (kDigits - 1)) : 0;
        const unsigned same = same_digit(digit, in);
        const int rank = __popc(same & ((1u << lane) - 1u));
        if (in && rank == 0) whist[warp][digit] = __popc(same);
        __syncthreads();
        {   // four threads a digit, eight warps each
            const int d = threadIdx.x >> 2, q = threadIdx.x & 3;
            int v[8], sum = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = whist[q * 8 + k][d];
                sum += v[k];
            }
            int incl = sum;
            int o = __shfl_up_sync(kFull, incl, 1, 4);
            if (q >= 1) incl += o;
            o = __shfl_up_sync(kFull, incl, 2, 4);
            if (q >= 2) incl += o;
            int run = base[d] + incl - sum;
            __syncwarp();
            if (q == 3) base[d] += incl;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                whist[q * 8 + k][d] = run;
                run += v[k];
            }
        }
        __syncthreads();
        if (in) p.out[whist[warp][digit] + rank] = e;
        if (i0 + 1024 < hi) {
            if (i + 1024 < hi) e = p.pair(i + 1024);
            __syncthreads();
            for (int k = threadIdx.x; k < 32 * kHistPitch; k += 1024) (&whist[0][0])[k] = 0;
            __syncthreads();
        }
    }
}

// ---- sums over the sorted list -------------------------------------------------------------------------------------

struct Sorted {
    const uint2 *pairs;   // (key, position)
    int64_t n;
    uint32_t n_nodes;     // the key of what is left out; such entries are the last ones
    int32_t stretch;      // entries that a group of threads sums
    int64_t stretches;
    __device__ __forceinline__ uint32_t key(int64_t i) const { return pairs[i].x; }
};

// First entries of their id before every stretch: `local` counts from the start of the stretch's part on, `base` is the part's (nullptr:
// local counts from the list's start); count[0] = all of them.
struct Heads {
    int32_t *local, *base, *count;
    FastDiv per_part;   // stretches
    __device__ __forceinline__ int32_t before(int64_t stretch) const
    {
        return local[stretch] + (base != nullptr ? base[per_part.div((uint32_t)stretch)] : 0);
    }
};

// Every CTA has a part of the list; the last one to end turns the parts' numbers into sums.
__global__ void __launch_bounds__(1024) head_kernel(Sorted l, Heads h, int32_t *ticket)
{
    __shared__ int32_t scan[32];
    __shared__ bool last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t part = (int64_t)h.per_part.d * l.stretch, lo = min(l.n, blockIdx.x * part), hi = min(l.n, lo + part);
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    int carry = 0;
    for (int64_t i0 = lo; i0 < hi; i0 += 1024) {
        const int64_t i = i0 + threadIdx.x;
        bool head = false;
        if (i < hi) {
            const uint32_t k = l.key(i);
            head = k < l.n_nodes && (i == 0 || l.key(i - 1) != k);
        }
        const unsigned first = __ballot_sync(kFull, head);
        __syncthreads();
        if (lane == 0) scan[warp] = __popc(first);
        __syncthreads();
        const int before = carry + __reduce_add_sync(kFull, lane < warp ? scan[lane] : 0);
        if (lane == 0 && i < hi && i % l.stretch == 0) h.local[i / l.stretch] = before;   // stretches are whole warps
        carry += __reduce_add_sync(kFull, scan[lane]);
    }
    if (threadIdx.x == 0) {
        h.base[blockIdx.x] = carry;
        __threadfence();
        last = atomicAdd(ticket, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last || warp != 0) return;
    __threadfence();
    int sum = 0;
    for (int c0 = 0; c0 < (int)gridDim.x; c0 += 32) {
        const int mine = c0 + lane < (int)gridDim.x ? __ldcg(&h.base[c0 + lane]) : 0;
        int incl = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(kFull, incl, s);
            if (lane >= s) incl += o;
        }
        if (c0 + lane < (int)gridDim.x) h.base[c0 + lane] = sum + incl - mine;
        sum += __shfl_sync(kFull, incl, 31);
    }
    if (lane == 0) h.count[0] = sum;
}

struct GradOut {
    void *rows;           // gradient of the table, or of the rows that occur
    int64_t stride;
    int32_t dtype;
    int32_t accumulate;
    Heads heads;          // rows that occur: first entries before every stretch; whole table: local is nullptr
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

constexpr int kSumThreads = 128;

template <int VE>
__device__ __forceinline__ void store_part(float *p, const float *x)
{
    Vec<float, VE> v;
    v.set(x);
    v.store(p);
}
template <int VE>
__device__ __forceinline__ void load_part(const float *p, float *x)
{
    Vec<float, VE> v;
    v.load(p);
#pragma unroll
    for (int i = 0; i < VE; ++i) x[i] = v.get(i);
}

// 2^log_group threads have a stretch, one vector of VE columns each.  What bounds it is HBM: the rows of the gradient are read
// once, `kAhead` of them on their way while the `kAhead` before them are added, whatever ids they belong to; only the additions
// go one after the other.  150,000 rows of 512 bytes: 26 us, 5.8 TB/s in and out; 16,384 rows of 4 KB into rows of 8 KB: 32 us.  (Eight rows
// ahead take the registers of half the CTAs: 102 us for a call of 89.)
template <typename T, int VE>
__global__ void __launch_bounds__(kSumThreads, 5)
grad_sum_kernel(Sorted l, const T *__restrict__ grad, int64_t grad_stride, GradOut o, int log_group)
{
    constexpr int kAhead = 4;
    const int group = threadIdx.x >> log_group;
    const int col = ((int)blockIdx.y * kSumThreads + (threadIdx.x & ((1 << log_group) - 1))) * VE;
    const int64_t c = (int64_t)blockIdx.x * (kSumThreads >> log_group) + group;
    if (c >= l.stretches || col >= o.dim) return;
    const int64_t lo = c * l.stretch, hi = min(l.n, lo + l.stretch);
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
    uint32_t key[kAhead];
    Vec<T, VE> next[kAhead];
    auto fetch = [&](int64_t i0, uint32_t *k, Vec<T, VE> *v) {
        uint2 e[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) e[j] = i0 + j < hi ? l.pairs[i0 + j] : make_uint2(l.n_nodes, 0);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            k[j] = e[j].x;
            if (k[j] < l.n_nodes) v[j].load_stream(grad + (int64_t)e[j].y * grad_stride + col);
        }
    };
    const uint32_t prev = lo > 0 ? l.key(lo - 1) : 0xFFFFFFFFu, behind = hi < l.n ? l.key(hi) : 0xFFFFFFFFu;
    const int32_t heads = o.heads.local != nullptr ? o.heads.before(c) : 0;
    fetch(lo, key, next);
    uint32_t cur = key[0];
    if (cur >= l.n_nodes) return;
    bool open = prev == cur;                   // the id began in a stretch before
    int32_t seg = heads - (open ? 1 : 0);
    float acc[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
    auto flush = [&]() {
        if (open) store_part<VE>(o.head_part + c * o.dim + col, acc);
        else o.put<VE>(o.heads.local != nullptr ? seg : (int64_t)cur, col, acc);
    };
    auto name = [&]() {
        if (o.unique != nullptr && col == 0 && !open) {
            if (o.wide) static_cast<int64_t *>(o.unique)[seg] = cur;
            else static_cast<int32_t *>(o.unique)[seg] = (int32_t)cur;
        }
    };
    name();
    for (int64_t i0 = lo; i0 < hi; i0 += kAhead) {
        uint32_t k[kAhead];
        Vec<T, VE> v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            k[j] = key[j];
            v[j] = next[j];
        }
        fetch(i0 + kAhead, key, next);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (k[j] >= l.n_nodes) continue;  // behind the last entry
            if (k[j] != cur) {
                flush();
                cur = k[j];
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
    if (behind == cur) store_part<VE>(o.tail_part + c * o.dim + col, acc);
    else flush();
}

// The ids that cross boundaries: the threads of the stretch where such an id begins add its pieces in list order.  An id of more than
// kLong pieces is left to the whole CTA: four threads a column, each every fourth piece, then their four sums.
constexpr int kLong = 24;
template <int VE>
__global__ void __launch_bounds__(kSumThreads) grad_join_kernel(Sorted l, GradOut o, int log_group)
{
    __shared__ int32_t longs;
    __shared__ int64_t long_first[kSumThreads], long_last[kSumThreads];
    constexpr int kParts = kSumThreads / 32;
    __shared__ float part[kParts][32 * VE];
    const int groups = kSumThreads >> log_group;
    const int in_group = threadIdx.x & ((1 << log_group) - 1);
    const int col = ((int)blockIdx.y * kSumThreads + in_group) * VE;
    const int64_t c = (int64_t)blockIdx.x * groups + (threadIdx.x >> log_group), lo = c * l.stretch, hi = lo + l.stretch;
    if (threadIdx.x == 0) longs = 0;
    cudaGridDependencySynchronize();
    __syncthreads();
    if (c < l.stretches && hi < l.n) {
        const uint32_t k = l.key(hi - 1), behind = l.key(hi), before = lo > 0 ? l.key(lo - 1) : 0xFFFFFFFFu;
        if (k < l.n_nodes && behind == k && before != k) {
            // the last stretch that begins with the id: c + 1 does; steps that double, then halve
            int64_t last = c + 1, step = 1;
            while (last + step < l.stretches && l.key((last + step) * l.stretch) == k) {
                last += step;
                step *= 2;
            }
            for (; step >= 1; step /= 2)
                if (last + step < l.stretches && l.key((last + step) * l.stretch) == k) last += step;
            const int64_t row = o.heads.local != nullptr ? o.heads.before(c + 1) - 1 : (int64_t)k;
            if (last - c >= kLong) {
                if (in_group == 0) {
                    const int at = atomicAdd(&longs, 1);   // in which order they are taken changes nothing
                    long_first[at] = c;
                    long_last[at] = last;
                }
            } else if (col < o.dim) {
                float acc[VE], v[VE];
                load_part<VE>(o.tail_part + c * o.dim + col, acc);
#pragma unroll 4
                for (int64_t s = c + 1; s <= last; ++s) {
                    load_part<VE>((s == last ? o.head_part : o.tail_part) + s * o.dim + col, v);
#pragma unroll
                    for (int i = 0; i < VE; ++i) acc[i] += v[i];
                }
                o.put<VE>(row, col, acc);
            }
        }
    }
    __syncthreads();
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int q = 0; q < longs; ++q) {
        const int64_t first = long_first[q], last = long_last[q];
        const int64_t row = o.heads.local != nullptr ? o.heads.before(first + 1) - 1 : (int64_t)l.key((first + 1) * l.stretch);
        const int end = min(o.dim, ((int)blockIdx.y + 1) * kSumThreads * VE);
        for (int col0 = (int)blockIdx.y * kSumThreads * VE; col0 < end; col0 += 32 * VE) {
            const int at = col0 + x * VE;
            float acc[VE], v[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
            if (at < end)
#pragma unroll 8
                for (int64_t s = first + y; s <= last; s += kParts) {
                    load_part<VE>((s == last ? o.head_part : o.tail_part) + s * o.dim + at, v);
#pragma unroll
                    for (int i = 0; i < VE; ++i) acc[i] += v[i];
                }
#pragma unroll
            for (int i = 0; i < VE; ++i) part[y][x * VE + i] = acc[i];
            __syncthreads();
            if (y == 0 && at < end) {
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    acc[i] = 0.0f;
#pragma unroll
                    for (int w = 0; w < kParts; ++w) acc[i] += part[w][x * VE + i];
                }
                o.put<VE>(row, at, acc);
            }
            __syncthreads();
        }
    }
}

// ---- short lists -----------------------------------------------------------------------------------------------------

constexpr int kDirectMax = 1024;   // lists up to here are not sorted
constexpr int kDirectThreads = 128;
constexpr int kFillRows = 32768;   // rows whose presence a CTA notes at a time

// Which positions of the list are the first of their id (a bit each), and how many there are.  One CTA, a thread a position.
__global__ void __launch_bounds__(kDirectMax) direct_first_kernel(Ids ids, int n, uint32_t *first, int32_t *count)
{
    __shared__ uint32_t key[kDirectMax];
    __shared__ int32_t found[32];
    const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
    const uint32_t mine = i < n ? ids.key(i) : (uint32_t)ids.n_nodes;
    key[i] = mine;
    __syncthreads();
    bool is_first = mine < (uint32_t)ids.n_nodes;
    const uint4 *four = reinterpret_cast<const uint4 *>(key);
    const int whole = (warp * 32) / 4;   // the positions before this warp's
    bool seen = false;
#pragma unroll 8
    for (int j = 0; j < whole; ++j) {
        const uint4 k = four[j];
        seen |= k.x == mine || k.y == mine || k.z == mine || k.w == mine;
    }
    const unsigned same = __match_any_sync(kFull, mine);
    is_first = is_first && !seen && (same & ((1u << lane) - 1u)) == 0;
    const unsigned all = __ballot_sync(kFull, is_first);
    if (lane == 0) {
        first[warp] = all;
        found[warp] = __popc(all);
    }
    __syncthreads();
    if (warp == 0) {
        const int sum = __reduce_add_sync(kFull, found[lane]);
        if (lane == 0) count[0] = sum;
    }
}

// The whole gradient of a list of at most kDirectMax ids without sorting it.  The CTAs of a position read all ids; the position that is
// the first of its id has the positions of that id in order, and its CTAs add their rows.  Rows of the table that no id names are
// zeroed by the CTAs behind them, which read all ids too.  n^2 comparisons, but one launch (two for the rows that occur, whose places
// need the first positions of all ids).  333 rows of 602 fp16 into 5003: 8.2 us a call, bound by the chain of ids, positions, rows; 22 us
// by way of the sort above.  The rows of one id are added one after the other, eight on their way: 1000 rows of 512 fp32 of as good as different ids
// 5.7 us, of one id 70 (1025 of one, by way of the sort, 25).
struct Direct {
    Ids ids;
    int32_t n, blocks_y;     // CTAs per position
    const uint32_t *first;   // rows that occur: direct_first_kernel's bits
    ZeroFill fill;
    int32_t fill_word;       // bytes that are zeroed at a time: 16, 4 or 2; every row, start and pitch is a multiple
    FastDiv words;           // of them in a row
};

template <typename W>
__device__ __forceinline__ void zero_absent(const Direct &d, int64_t row0, int rows, const uint32_t *present)
{
    W zero = W();
    const uint32_t all = (uint32_t)rows * d.words.d;   // kFillRows rows have less than 2^32 words
    uint8_t *base = d.fill.p + row0 * d.fill.pitch;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < all; i += kDirectThreads) {
        const uint32_t r = d.words.div(i);
        if ((present[r >> 5] >> (r & 31) & 1u) == 0) reinterpret_cast<W *>(base + (int64_t)r * d.fill.pitch)[i - r * d.words.d] = zero;
    }
}

template <typename T, int VE>
__global__ void __launch_bounds__(kDirectThreads) direct_grad_kernel(Direct d, const T *__restrict__ grad, int64_t grad_stride, GradOut o)
{
    __shared__ uint32_t words[kFillRows / 32];   // fill: rows that occur; sums: the positions of the id, 16 bits each
    __shared__ int32_t counts[kDirectThreads / 32], smaller;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t none = (uint32_t)d.ids.n_nodes;
    const int position_ctas = d.n * d.blocks_y;
    if ((int)blockIdx.x >= position_ctas) {
        const int64_t me = blockIdx.x - position_ctas, ctas = gridDim.x - position_ctas;
        const int64_t end = d.fill.rows * (me + 1) / ctas;
        for (int64_t row0 = d.fill.rows * me / ctas; row0 < end; row0 += kFillRows) {
            const int rows = (int)min((int64_t)kFillRows, end - row0);
            __syncthreads();
            for (int i = threadIdx.x; i < (rows + 31) / 32; i += kDirectThreads) words[i] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < d.n; i += kDirectThreads) {
                const int64_t r = (int64_t)d.ids.key(i) - row0;
                if (r >= 0 && r < rows) atomicOr(&words[r >> 5], 1u << (r & 31));
            }
            __syncthreads();
            if (d.fill_word == 16) zero_absent<uint4>(d, row0, rows, words);
            else if (d.fill_word == 4) zero_absent<uint32_t>(d, row0, rows, words);
            else zero_absent<uint16_t>(d, row0, rows, words);
        }
        return;
    }
    const int me = blockIdx.x / d.blocks_y, block_y = blockIdx.x - me * d.blocks_y;
    const uint32_t mine = d.ids.key(me);
    if (mine >= none) return;
    uint16_t *list = reinterpret_cast<uint16_t *>(words);
    if (threadIdx.x == 0) smaller = 0;
    int found = 0;
    bool is_first = true;
    // a warp has a contiguous quarter of the list, so that the positions come in order
    const int part = ((d.n + kDirectThreads - 1) / kDirectThreads) * 32;
    uint32_t key[kDirectMax / kDirectThreads];
#pragma unroll
    for (int q = 0; q < kDirectMax / kDirectThreads; ++q) {
        const int i = warp * part + q * 32 + lane;
        key[q] = q * 32 < part && i < d.n ? d.ids.key(i) : none;
    }
    int below = 0;
#pragma unroll
    for (int q = 0; q < kDirectMax / kDirectThreads; ++q) {
        const int i0 = warp * part + q * 32;
        const unsigned same = __ballot_sync(kFull, key[q] == mine);
        found += __popc(same);
        if (same != 0 && i0 + __ffs((int)same) - 1 < me) is_first = false;
        if (d.first != nullptr && q * 32 < part && i0 < d.n) below += __popc(d.first[i0 >> 5] & __ballot_sync(kFull, key[q] < mine));
    }
    if (lane == 0) counts[warp] = found;
    if (__syncthreads_or(!is_first)) return;
    if (lane == 0 && below != 0) atomicAdd(&smaller, below);
    int total = 0, at = 0;
#pragma unroll
    for (int w = 0; w < kDirectThreads / 32; ++w) {
        at += w < warp ? counts[w] : 0;
        total += counts[w];
    }
#pragma unroll
    for (int q = 0; q < kDirectMax / kDirectThreads; ++q) {
        const unsigned same = __ballot_sync(kFull, key[q] == mine);
        if (key[q] == mine) list[at + __popc(same & ((1u << lane) - 1u))] = (uint16_t)(warp * part + q * 32 + lane);
        at += __popc(same);
    }
    __syncthreads();
    const int col = (block_y * kDirectThreads + (int)threadIdx.x) * VE;
    const int64_t row = d.first != nullptr ? smaller : (int64_t)mine;
    if (d.first != nullptr && col == 0) {
        if (o.wide) static_cast<int64_t *>(o.unique)[row] = mine;
        else static_cast<int32_t *>(o.unique)[row] = (int32_t)mine;
    }
    if (col >= o.dim) return;
    constexpr int kAhead = 8;
    float acc[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[i] = 0.0f;
    for (int j0 = 0; j0 < total; j0 += kAhead) {
        Vec<T, VE> v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (j0 + j < total) v[j].load_stream(grad + (int64_t)list[j0 + j] * grad_stride + col);
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (j0 + j < total) {
#pragma unroll
                for (int i = 0; i < VE; ++i) acc[i] += v[j].get(i);
            }
    }
    o.put<VE>(row, col, acc);
}

// ---- host side -----------------------------------------------------------------------------------------------------

static int32_t stretch_of(int64_t n) { return n <= (1 << 20) ? 32 : (n <= (1 << 22) ? 64 : 128); }

// The layout is the same for all lists; those that are not sorted use `heads` alone.
struct GradScratch {
    uint2 *pairs[2];
    int32_t *counts, *heads;
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
        for (int k = 0; k < 2; ++k) pairs[k] = (uint2 *)take(8 * n);
        counts = (int32_t *)take(((int64_t)kPassMax * kCountRows * kDigits + 1 + kSms) * 4);   // and a ticket, and the parts' first entries
        heads = (int32_t *)take(n <= kDirectMax ? kDirectMax / 8 : 4 * (stretches + 1));
        head_part = (float *)take(stretches > 1 ? 4 * stretches * dim : 0);
        tail_part = (float *)take(stretches > 1 ? 4 * stretches * dim : 0);
    }
};

// Most CTAs of a cluster of the sort on the current device: 16 where a group of SMs has that many free, 8 anywhere.
static int widest_cluster()
{
    static int found[64];   // per device, 0: not asked yet
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 8;
    if (found[dev] == 0) {
        int most = 8;
        if (cudaFuncSetAttribute(cluster_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cluster_sort_smem(kClusterPart)) == cudaSuccess &&
            cudaFuncSetAttribute(cluster_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = 16;
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(16);
            cfg.blockDim = dim3(kClusterThreads);
            cfg.dynamicSmemBytes = (size_t)cluster_sort_smem(kClusterPart);
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int clusters = 0;
            if (cudaOccupancyMaxActiveClusters(&clusters, cluster_sort_kernel, &cfg) == cudaSuccess && clusters >= 1) most = 16;
        }
        cudaGetLastError();  // what was refused here is no error of the call
        found[dev] = most;
    }
    return found[dev];
}

// A launch in clusters of `cluster` CTAs (0: none), `after_own`: as a dependent of this file's launch before it, which it may overlap
// up to its cudaGridDependencySynchronize.
template <typename... A, typename... B>
static cudaError_t launch(cudaStream_t s, void (*kernel)(A...), unsigned grid_x, unsigned grid_y, unsigned threads, int64_t smem, unsigned cluster,
                          bool after_own, B... args)
{
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid_x, grid_y);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cfg.attrs = attr;
    if (cluster > 0) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    if (after_own) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    return cudaLaunchKernelEx(&cfg, kernel, A(args)...);
}

static int sort_ids(cudaStream_t s, const Ids &ids, int64_t n, const GradScratch &w, int32_t *count, const ZeroFill &fill, Sorted *l, Heads *heads)
{
    l->n = n;
    l->n_nodes = (uint32_t)ids.n_nodes;
    l->stretch = stretch_of(n);
    l->stretches = (n + l->stretch - 1) / l->stretch;
    int bits = 0;
    while ((ids.n_nodes >> bits) != 0) ++bits;  // n_nodes itself is a key
    const int widest = widest_cluster();
    if (n <= kClusterList && n <= (int64_t)widest * kClusterPart) {
        int ctas = 1;
        while (ctas < widest && (int64_t)ctas * kClusterThreads < n) ctas *= 2;
        const int64_t part = ((n + ctas - 1) / ctas + kClusterThreads - 1) / kClusterThreads * kClusterThreads;
        ClusterSort p{ ids, (int32_t)n, (int32_t)part, FastDiv((uint32_t)part), bits, w.pairs[0], count != nullptr ? w.heads : nullptr, count, l->stretch };
        if (fill.p != nullptr) {
            const int64_t need = (fill.rows * fill.width + 16383) / 16384;   // 16 KB a CTA or more
            LG_CUDA(launch(s, zero_fill_kernel, (unsigned)(need < 4 * kSms ? need : 4 * kSms), 1, 256, 0, 0, false, fill));
        }
        LG_CUDA(launch(s, cluster_sort_kernel, (unsigned)ctas, 1, kClusterThreads, cluster_sort_smem(part), (unsigned)ctas, fill.p != nullptr, p));
        l->pairs = w.pairs[0];
        if (count != nullptr) *heads = Heads{ w.heads, nullptr, count, FastDiv(1) };
        return LEGION_OK;
    }
    if (fill.p != nullptr) {
        if (fill.pitch == fill.width) LG_CUDA(cudaMemsetAsync(fill.p, 0, (size_t)(fill.rows * fill.width), s));
        else LG_CUDA(cudaMemset2DAsync(fill.p, (size_t)fill.pitch, 0, (size_t)fill.width, (size_t)fill.rows, s));
    }
    const int part = (int)((n + kSms - 1) / kSms);
    SortPass p{ ids, nullptr, nullptr, w.counts, n, part, 0 };
    const int passes = (bits + 7) / 8, words = passes * kCountRows * kDigits;
    int32_t *ticket = w.counts + words;
    LG_CUDA(launch(s, sort_zero_kernel, 64, 1, 1024, 0, 0, false, w.counts, words + 1));
    for (int q = 0; q < passes; ++q) {
        p.in = q == 0 ? nullptr : w.pairs[(q & 1) ^ 1];
        p.out = w.pairs[q & 1];
        p.counts = w.counts + q * kCountRows * kDigits;
        p.shift = q * 8;
        LG_CUDA(launch(s, sort_count_kernel, kSms, 1, 1024, 0, 0, true, p));
        LG_CUDA(launch(s, sort_scatter_kernel, kSms, 1, 1024, 0, 0, true, p));
    }
    l->pairs = w.pairs[(passes & 1) ^ 1];
    if (count != nullptr) {
        const uint32_t per_part = (uint32_t)((l->stretches + kSms - 1) / kSms);
        *heads = Heads{ w.heads, ticket + 1, count, FastDiv(per_part) };
        LG_CUDA(launch(s, head_kernel, (unsigned)((l->stretches + per_part - 1) / per_part), 1, 1024, 0, 0, true, *l, *heads, ticket));
    }
    return LEGION_OK;
}

template <typename T, int VE>
static int launch_sum(cudaStream_t s, const Sorted &l, const void *grad, int64_t stride, const GradOut &o)
{
    const int vecs = o.dim / VE;
    int log_group = 0;
    while ((1 << log_group) < kSumThreads && (1 << log_group) < vecs) ++log_group;
    const int64_t per = kSumThreads >> log_group;
    const dim3 grid((unsigned)((l.stretches + per - 1) / per), (unsigned)((vecs + kSumThreads - 1) / kSumThreads));
    LG_CUDA(launch(s, grad_sum_kernel<T, VE>, grid.x, grid.y, kSumThreads, 0, 0, true, l, (const T *)grad, stride, o, log_group));
    LG_CUDA(launch(s, grad_join_kernel<VE>, grid.x, grid.y, kSumThreads, 0, 0, true, l, o, log_group));
    return LEGION_OK;
}

template <typename T, int VE>
static void launch_direct(cudaStream_t s, Direct d, const void *grad, int64_t stride, const GradOut &o)
{
    d.blocks_y = (o.dim / VE + kDirectThreads - 1) / kDirectThreads;
    // a CTA that fills has 8 KB or more to write
    int64_t fillers = d.fill.p != nullptr ? (d.fill.rows * d.fill.width + (8 << 10) - 1) / (8 << 10) : 0;
    if (fillers > d.fill.rows) fillers = d.fill.rows;
    if (fillers > 16 * kSms) fillers = 16 * kSms;
    direct_grad_kernel<T, VE><<<(unsigned)(d.n * d.blocks_y + fillers), kDirectThreads, 0, s>>>(d, (const T *)grad, stride, o);
}

template <typename T>
static void launch_direct_ve(int ve, cudaStream_t s, const Direct &d, const void *grad, int64_t stride, const GradOut &o)
{
    switch (ve) {
    case 8:
        if constexpr (sizeof(T) == 2) { launch_direct<T, 8>(s, d, grad, stride, o); break; }
    case 4: launch_direct<T, 4>(s, d, grad, stride, o); break;
    case 2: launch_direct<T, 2>(s, d, grad, stride, o); break;
    default: launch_direct<T, 1>(s, d, grad, stride, o); break;
    }
}

template <typename T>
static int launch_sum_ve(int ve, cudaStream_t s, const Sorted &l, const void *grad, int64_t stride, const GradOut &o)
{
    switch (ve) {
    case 8:
        if constexpr (sizeof(T) == 2) return launch_sum<T, 8>(s, l, grad, stride, o);
    case 4: return launch_sum<T, 4>(s, l, grad, stride, o);
    case 2: return launch_sum<T, 2>(s, l, grad, stride, o);
    default: return launch_sum<T, 1>(s, l, grad, stride, o);
    }
}

static int run_grad(cudaStream_t s, const Ids &ids, int64_t n, const void *grad, int32_t grad_dtype, int64_t grad_stride, GradOut o,
                    const GradScratch &w, int32_t *count, const ZeroFill &fill)
{
    // what a vector may have: the loads of the gradient are at most 16 bytes, and every address is a multiple of it
    const int ve = common_vector(grad_dtype == LEGION_F32 ? 4 : 8,
                                 { o.dim, grad_stride, aligned_elements(grad, grad_dtype), o.stride, aligned_elements(o.rows, o.dtype) });
    if (n <= kDirectMax) {
        int word = 16;
        while (word > 2 && (fill.width % word != 0 || fill.pitch % word != 0 || (uintptr_t)fill.p % word != 0)) word = word == 16 ? 4 : 2;
        uint32_t *first = count != nullptr ? (uint32_t *)w.heads : nullptr;
        const Direct d{ ids, (int32_t)n, 1, first, fill, word, FastDiv((uint32_t)(fill.p != nullptr ? fill.width / word : 1)) };
        if (count != nullptr) direct_first_kernel<<<1, kDirectMax, 0, s>>>(ids, (int)n, first, count);
        if (grad_dtype == LEGION_F32) launch_direct_ve<float>(ve, s, d, grad, grad_stride, o);
        else if (grad_dtype == LEGION_F16) launch_direct_ve<__half>(ve, s, d, grad, grad_stride, o);
        else launch_direct_ve<__nv_bfloat16>(ve, s, d, grad, grad_stride, o);
        LG_LAUNCH_CHECK();
        return LEGION_OK;
    }
    Sorted l;
    Heads heads{ nullptr, nullptr, nullptr, FastDiv(1) };
    int rc = sort_ids(s, ids, n, w, count, fill, &l, &heads);
    if (rc != LEGION_OK) return rc;
    o.head_part = w.head_part;
    o.tail_part = w.tail_part;
    o.heads = heads;
    if (grad_dtype == LEGION_F32) return launch_sum_ve<float>(ve, s, l, grad, grad_stride, o);
    if (grad_dtype == LEGION_F16) return launch_sum_ve<__half>(ve, s, l, grad, grad_stride, o);
    return launch_sum_ve<__nv_bfloat16>(ve, s, l, grad, grad_stride, o);
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
    LG_ARG(n_ids == 0 || out != table, "out must not be the table");
    if (n_ids * dim > (1ll << 40)) {
        set_error("legion_embedding_lookup: %lld rows of %d elements are above the limit of 2^40 elements", (long long)n_ids, dim);
        return LEGION_E_LIMIT;
    }
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
    if (!std::isfinite(scale) || std::signbit(scale)) {
        const int64_t bytes = dtype_bytes(out_dtype);
        zero_outside_kernel<<<(unsigned)((n_ids + 7) / 8), 256, 0, s>>>(list, n_ids, (uint8_t *)out, dim * bytes, out_stride * bytes);
        LG_LAUNCH_CHECK();
    }
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
    LG_ARG(n_ids == 0 || grad_table != grad_out, "grad_table must not be grad_out");
    const GradScratch w((uint8_t *)workspace, n_ids, dim);
    if (n_ids > 0 && (rc = check_workspace(workspace, workspace_bytes, w.bytes)) != LEGION_OK) return rc;
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    cudaStream_t s = (cudaStream_t)stream;
    const int64_t width = (int64_t)dim * dtype_bytes(table_dtype), pitch = table_stride * dtype_bytes(table_dtype);
    if (n_ids == 0) {
        if (!accumulate) LG_CUDA(cudaMemset2DAsync(grad_table, (size_t)pitch, 0, (size_t)width, (size_t)n_nodes, s));
        return LEGION_OK;
    }
    const ZeroFill fill{ accumulate ? nullptr : (uint8_t *)grad_table, n_nodes, width, pitch };
    GradOut o{ nullptr, 0, 0, 0, Heads{ nullptr, nullptr, nullptr, FastDiv(1) }, nullptr, 0, 0.0f, 0, nullptr, nullptr };
    o.rows = grad_table;
    o.stride = table_stride;
    o.dtype = table_dtype;
    o.accumulate = accumulate != 0;
    o.scale = scale;
    o.dim = dim;
    return run_grad(s, Ids{ ids, id_bytes == 8, n_nodes }, n_ids, grad_out, grad_dtype, grad_stride, o, w, nullptr, fill);
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
    LG_ARG(n_ids == 0 || (unique_ids != nullptr && (uintptr_t)unique_ids % id_bytes == 0), "unique_ids is NULL or not on a multiple of the ids' width");
    LG_ARG(n_ids == 0 || (unique_ids != ids && (const void *)grad_rows != grad_out), "unique_ids and grad_rows must not be the inputs");
    const GradScratch w((uint8_t *)workspace, n_ids, dim);
    if (n_ids > 0 && (rc = check_workspace(workspace, workspace_bytes, w.bytes)) != LEGION_OK) return rc;
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    cudaStream_t s = (cudaStream_t)stream;
    if (n_ids == 0) {
        LG_CUDA(cudaMemsetAsync(count, 0, 4, s));
        return LEGION_OK;
    }
    GradOut o{ nullptr, 0, 0, 0, Heads{ nullptr, nullptr, nullptr, FastDiv(1) }, nullptr, 0, 0.0f, 0, nullptr, nullptr };
    o.rows = grad_rows;
    o.stride = rows_stride;
    o.dtype = LEGION_F32;
    o.unique = unique_ids;
    o.wide = id_bytes == 8;
    o.scale = scale;
    o.dim = dim;
    return run_grad(s, Ids{ ids, id_bytes == 8, n_nodes }, n_ids, grad_out, grad_dtype, grad_stride, o, w, count, ZeroFill{});
}
