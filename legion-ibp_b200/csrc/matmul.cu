// Products of compressed rows: out[i][j] = sa[i] * sb[j] * sum_k a[i][k] * b[j][k], codes int8 or e4m3, one fp32 scale per row
// behind the codes.  Nothing is decoded: the codes go to the tensor cores as they lie in memory, the two scales
// meet the sum in the epilogue.
#include "async.cuh"
#include "codec.cuh"
#include "typed.cuh"

#include <cuda.h>
#include <type_traits>

namespace legion {

static constexpr unsigned kFull = 0xFFFFFFFFu;

__device__ int32_t g_operator_error = 0;

// ---- PTX ---------------------------------------------------------------------------------------------------------

__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// PAIR: the barrier may be the other CTA's.
template <int PAIR>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y)
{
    if (PAIR == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                     "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    else asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}

// Whether any of the 128 threads of warps 0 to 3 says so; a barrier among them.
__device__ __forceinline__ bool any_of_128(bool mine)
{
    uint32_t any;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(any) : "r"((uint32_t)mine) : "memory");
    return any != 0;
}

// Shared-memory matrix descriptor of a K-major operand in the 128-byte swizzle: rows of 128 bytes, groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr)
{
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor: D type (1 fp32, 2 int32) at bit 4, A and B types (int8: 1, e4m3: 0) at 7 and 10, N / 8 at 17, M / 16 at 24.
template <int CODEC, int M, int N>
__device__ __forceinline__ constexpr uint32_t instruction_desc()
{
    return (CODEC == LEGION_CODEC_INT8 ? (2u << 4 | 1u << 7 | 1u << 10) : 1u << 4) | (uint32_t)(N / 8) << 17 | (uint32_t)(M / 16) << 24;
}
#define LG_MMA(GROUP, KIND)                                                                                                                  \
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n}" ::"r"(d), \
                 "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory")
template <int CODEC, int PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add)
{
    if (CODEC == LEGION_CODEC_INT8 && PAIR == 1) LG_MMA("1", "i8");
    else if (CODEC == LEGION_CODEC_INT8) LG_MMA("2", "i8");
    else if (PAIR == 1) LG_MMA("1", "f8f6f4");
    else LG_MMA("2", "f8f6f4");
}
#undef LG_MMA
// The barrier (PAIR: of both CTAs) is arrived at when the products issued so far are done.
template <int PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar)
{
    if (PAIR == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool one_lane()
{
    uint32_t mine;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(mine));
    return mine != 0;
}
// Address of a shared variable in the pair's first CTA.
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(addr));
    return a;
}
__device__ __forceinline__ void pair_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the warp's 32 lanes; tmem_wait before the registers are read.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
                 "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// A tile of shared memory to global memory by TMA, in the calling thread's group of copies.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int x, int y)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// ---- tensor-core kernel ----------------------------------------------------------------------------------------------

struct MatmulParams {
    const uint8_t *p_rows, *q_rows;   // the operand whose rows are TMEM lanes (tiles of 128), and the other
    int64_t p_stride, q_stride;
    int32_t p_n, q_n, k;
    void *out;
    int64_t out_stride;
    int32_t out_dtype;
    int32_t word;     // the widest word of 16, 8, 4 or 2 bytes that the output's rows start on multiples of
    int32_t stages, stage_bytes, q_at;   // of shared memory; where a stage's rows of Q begin
    int32_t step_p;   // rows of P per CTA and tile: kTileP, or fewer (a multiple of 8) where that gives every SM a tile
    uint32_t tries;   // of a wait
};

constexpr int kTileP = 128;
constexpr int kTileK = 128;   // bytes of a row per stage: one swizzle line
constexpr int kStagesMax = 32;
// Blocks of kTileK codes per stage: what a stage costs beside its products (the wait, the commit, the loop: 230 clocks) is more than the
// products of a narrow tile.
__host__ __device__ constexpr int blocks_per_stage(int bq, int pair) { return bq / pair >= 128 ? 1 : 2; }
__host__ __device__ constexpr int tmem_columns(int bq) { return 2 * bq < 32 ? 32 : 2 * bq; }
constexpr int kOutBytes = 32 * 128;   // of a warp's 32 rows, 128 bytes each, on their way out
__host__ __device__ constexpr int out_buffers(int bq, int pair) { return bq / pair >= 256 ? 1 : 2; }
constexpr int kSmem = 227 * 1024;
// What the stages do not take: alignment, the output's buffers, the scales, the barriers.
__host__ __device__ constexpr int smem_beside_stages(int bq, int pair) { return 1024 + 4 * out_buffers(bq, pair) * kOutBytes + 2 * bq * 4 + 16 * kStagesMax + 64; }

// Tiles in groups of kGroupP along P, so that the tiles that run together share rows of both operands in L2.
constexpr int kGroupP = 16;
__device__ __forceinline__ void tile_at(int64_t t, int tiles_p, int tiles_q, int &p, int &q)
{
    const int64_t per_group = (int64_t)kGroupP * tiles_q;
    const int g = (int)(t / per_group);
    const int rest = (int)(t - g * per_group);
    const int height = min(kGroupP, tiles_p - g * kGroupP);
    q = rest / height;
    p = g * kGroupP + rest - q * height;
}

// 32 (or, a tile of 16 columns, 16) sums of a lane's row as fp32.
template <int CODEC, int N>
__device__ __forceinline__ void load_sums(uint32_t acc, float *v)
{
    uint32_t r[N];
    if (N == 32) tmem_load32(acc, r);
    else tmem_load16(acc, r);
    tmem_wait();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = CODEC == LEGION_CODEC_INT8 ? (float)(int32_t)r[i] : __uint_as_float(r[i]);
}

// A sum times the scales of its row and of its weight row, rounded the same way wherever it is worked out.  The scales' product is not formed: it leaves
// fp32's range where the result does not.  The sum meets the row's scale first: sums are below 2^35, so a scale of at most 2^92 does not
// overflow with one, and an integer times a subnormal number is exact or normal.  With a larger scale of the row the weight's comes first: if that
// overflows, so does the result.
__device__ __forceinline__ bool near(float scale) { return fabsf(scale) <= 4951760157141521099596496896.0f; }   // 2^92; not a NaN
__device__ __forceinline__ float scaled(float sum, float row, float weight)
{
    const bool row_first = near(row);
    return sum * (row_first ? row : weight) * (row_first ? weight : row);
}

// N sums of a lane: ONE_ROW: of one row and N weight rows, otherwise of one weight row and N rows.  The warp votes on whether there is a choice (one made
// for each sum took 4 to 6% of products of 128 to 512 codes).
template <int N, bool ONE_ROW>
__device__ __forceinline__ void scale_all(float *v, float one, const float *other)
{
    if (__any_sync(kFull, !near(ONE_ROW ? one : other[threadIdx.x % N]))) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = ONE_ROW ? scaled(v[i], one, other[i]) : scaled(v[i], other[i], one);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = ONE_ROW ? v[i] * one * other[i] : v[i] * other[i] * one;
    }
}

__device__ __forceinline__ void store_one(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_one(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void store_one(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// `rows` rows of `cols` values of type T from shared memory (WIDTH values a row, SWIZZLED: 128 bytes with their 16-byte pieces in the
// order of the TMA swizzle) to rows `stride` apart, by words of type W: consecutive lanes write consecutive words.
template <typename W, typename T, int WIDTH, bool SWIZZLED>
__device__ __forceinline__ void write_rows(T *dst, int64_t stride, const uint8_t *src, int rows, int cols)
{
    if constexpr (sizeof(W) >= sizeof(T)) {
        constexpr int kPer = (int)(sizeof(W) / sizeof(T)), kWords = WIDTH / kPer, kBytes = WIDTH * (int)sizeof(T);
#pragma unroll 8
        for (int i = threadIdx.x & 31; i < rows * kWords; i += 32) {
            const int r = i / kWords, w = i % kWords, at = w * (int)sizeof(W);
            const uint8_t *s = src + r * kBytes + (SWIZZLED ? ((at / 16) ^ (r & 7)) * 16 + at % 16 : at);
            T *d = dst + r * stride + w * kPer;
            if ((w + 1) * kPer <= cols) {
                *reinterpret_cast<W *>(d) = *reinterpret_cast<const W *>(s);
            } else {
                for (int j = 0; j < kPer && w * kPer + j < cols; ++j) d[j] = reinterpret_cast<const T *>(s)[j];
            }
        }
    }
}

// A warp's 32 rows of a tile, scaled, rounded and on their way: 128 bytes of each row at a time.
template <int CODEC, typename T, int BQ, int BUFFERS>
__device__ __forceinline__ void store_tile(uint32_t acc, float ps, const float *qs, uint8_t *buffer, const CUtensorMap *map, int q0, int p0,
                                           const MatmulParams &m, uint32_t &copies)
{
    constexpr int kCols = 128 / (int)sizeof(T), kPer16 = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
    if (p0 >= m.p_n) return;
#pragma unroll 1
    for (int c = 0; c < BQ && q0 + c < m.q_n; c += kCols) {
        uint8_t *row = buffer + (copies++ % BUFFERS) * kOutBytes + lane * 128;
        // the copy that read this buffer last is done with it
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(BUFFERS - 1) : "memory");
        __syncwarp();
#pragma unroll
        for (int half = 0; half < kCols; half += 32) {
            float v[32];
            load_sums<CODEC, 32>(acc + c + half, v);
            scale_all<32, true>(v, ps, qs + c + half);
#pragma unroll
            for (int i = 0; i < 32; i += kPer16) {
                Vec<T, kPer16> o;
                o.set(v + i);
                o.store(reinterpret_cast<T *>(row + (((half + i) / kPer16) ^ (lane & 7)) * 16));
            }
        }
        const int cols = min(kCols, m.q_n - q0 - c);
        if (m.word == 16 && cols % kPer16 == 0) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tma_store_2d(map, shared_addr(row), q0 + c, p0);
        } else {
            // Rows that TMA cannot address, or that end inside 16 bytes (TMA leaves out what lies behind a row's end by whole 16 bytes only and zeroes
            // the rest): the lanes write along them, in words that the rows start on.
            __syncwarp();
            const int rows = min(32, m.p_n - p0);
            T *dst = static_cast<T *>(m.out) + (int64_t)p0 * m.out_stride + q0 + c;
            const uint8_t *src = row - lane * 128;
            if (m.word >= 8) write_rows<uint2, T, kCols, true>(dst, m.out_stride, src, rows, cols);
            else if (m.word == 4) write_rows<uint32_t, T, kCols, true>(dst, m.out_stride, src, rows, cols);
            else write_rows<uint16_t, T, kCols, true>(dst, m.out_stride, src, rows, cols);
            if (m.word == 16 && lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");   // of no copies: the wait above counts a group a buffer
            __syncwarp();
        }
    }
}

// The same for P_OUT_COLUMNS: 32 x 32 sums change places in shared memory, so that the lanes write along the rows of the output (2-byte
// stores took 66 clocks each: 4000 clocks for 64 rows).
template <int CODEC, typename T, int BQ>
__device__ __forceinline__ void store_turned(uint32_t acc, float ps, const float *qs, uint8_t *buffer, int q0, int p0, int valid, const MatmulParams &m)
{
    constexpr int N = BQ < 32 ? BQ : 32;
    const int lane = threadIdx.x & 31;
    T *mine = reinterpret_cast<T *>(buffer);
#pragma unroll 1
    for (int c = 0; c < BQ && q0 + c < m.q_n; c += N) {
        float v[N];
        load_sums<CODEC, N>(acc + c, v);
        scale_all<N, false>(v, ps, qs + c);
        __syncwarp();   // the last turn's values have been read
#pragma unroll
        for (int i = 0; i < N; ++i) store_one(mine + i * 32 + lane, v[i]);
        __syncwarp();
        const int rows = min(N, m.q_n - q0 - c);
        T *dst = static_cast<T *>(m.out) + (int64_t)(q0 + c) * m.out_stride + p0;
        if (m.word == 16) write_rows<uint4, T, 32, false>(dst, m.out_stride, buffer, rows, valid);
        else if (m.word == 8) write_rows<uint2, T, 32, false>(dst, m.out_stride, buffer, rows, valid);
        else if (m.word == 4) write_rows<uint32_t, T, 32, false>(dst, m.out_stride, buffer, rows, valid);
        else write_rows<uint16_t, T, 32, false>(dst, m.out_stride, buffer, rows, valid);
    }
}

// One CTA per SM takes tiles of 128 x BQ in turn.  Warp 4 loads stages of both operands by TMA, warp 5 issues the products into one of
// two accumulators in TMEM, warps 0 to 3 scale and store the other one meanwhile.
// PAIR 2: two CTAs take tiles of 256 x BQ together: each loads its 128 rows of P and half of the rows of Q, the first one issues
// the products of both, each holds and stores the sums of its own rows of P.
// The output leaves by TMA: a warp writes 128 bytes of each of its 32 rows to shared memory (in the swizzle that the store
// undoes, so that lanes hit different banks); rows that TMA cannot address are written by the lanes along the rows (every lane along its
// own row, 510 x 7548 bf16 took 47 us).
// What bounds it: large products of rows on 128-byte boundaries the tensor cores (4096 x 16384 x 4096 int8: 171 us, 3.2 POP/s); rows that
// start on 16-byte boundaries, as compressed rows do, the copy engine, which takes 278 clocks for 128 of them where the products of
// a stage take 512 (214 us; 128 x 256 tiles of one CTA: 342 us); few rows the weights' bytes (16 rows: 18 us for 67 MB).
// P_OUT_COLUMNS: rows of P are columns of the output (P holds the weights), for few rows on the other side.  A tile then has step_p rows of P,
// as many as spread the weights over all SMs.  The products read 128 rows all the same: what lies behind the tile's rows in shared
// memory reaches nobody's sums but those of rows that are not stored.
template <int CODEC, int BQ, bool P_OUT_COLUMNS, int PAIR>
__global__ void __launch_bounds__(224, 1)
matmul_kernel(const __grid_constant__ CUtensorMap p_map, const __grid_constant__ CUtensorMap q_map,
              const __grid_constant__ CUtensorMap out_map, MatmulParams m)
{
    constexpr int kPairP = kTileP * PAIR;
    constexpr int kSub = blocks_per_stage(BQ, PAIR);
    const int S = m.stages, kStage = m.stage_bytes, q_at = m.q_at;
    const uint32_t sub_bytes = (uint32_t)kStage / kSub;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    constexpr int kOut = out_buffers(BQ, PAIR);
    uint8_t *out_smem = smem + S * kStage;                                                   // [warp][buffer]
    float *q_scale = reinterpret_cast<float *>(out_smem + 4 * kOut * kOutBytes);             // [2][BQ]
    uint64_t *bars = reinterpret_cast<uint64_t *>(q_scale + 2 * BQ);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kStagesMax + 4);
    volatile int32_t *gave_up = reinterpret_cast<volatile int32_t *>(tmem_slot + 1);
    const uint32_t full = shared_addr(bars), empty = full + 8 * S, acc_full = empty + 8 * S, acc_empty = acc_full + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t me = PAIR == 2 ? blockIdx.x & 1 : 0;   // which of the pair
    const int step_p = PAIR == 2 || !P_OUT_COLUMNS ? kPairP : m.step_p;
    const int tiles_p = (m.p_n + step_p - 1) / step_p, tiles_q = (m.q_n + BQ - 1) / BQ;
    const int64_t tiles = (int64_t)tiles_p * tiles_q;
    const int blocks_k = (m.k + kTileK - 1) / kTileK;

    // the producer's place: tile, block of its rows, stage, how often the stages have been gone through
    int64_t tile = blockIdx.x / PAIR;
    int block = 0, stage = 0, tp = 0, tq = 0;
    uint32_t round = 0;
    uint32_t full_of_first = full;
    auto produce = [&]() {   // the whole warp; one lane issues
        if (block == 0) tile_at(tile, tiles_p, tiles_q, tp, tq);
        if (one_lane()) {
            uint32_t dst = shared_addr(smem + stage * kStage);
            const uint32_t bar = full_of_first + 8 * stage;
            const int subs = min(kSub, blocks_k - block);
            if (warp == 4 && me == 0) expect_bytes(full + 8 * stage, (uint32_t)subs * sub_bytes * PAIR);   // what all bring
            for (int i = 0; i < subs; ++i, dst += sub_bytes) {
                if (warp == 4) tma_2d<PAIR>(dst, &p_map, bar, (block + i) * kTileK, tp * step_p + (int)me * kTileP);
                else tma_2d<PAIR>(dst + q_at, &q_map, bar, (block + i) * kTileK, tq * BQ + (int)me * (BQ / PAIR));
            }
        }
        __syncwarp();
        block += kSub;
        if (block >= blocks_k) {
            block = 0;
            tile += gridDim.x / PAIR;
        }
        if (++stage == S) {
            stage = 0;
            ++round;
        }
    };
    if (warp == 4) {
        if (lane < S) {
            init_barrier(full + 8 * lane, 1);
            init_barrier(empty + 8 * lane, 1);
        }
        if (lane < 2) {
            init_barrier(acc_full + 8 * lane, 1);
            init_barrier(acc_empty + 8 * lane, 4 * PAIR);   // the warps that store
        }
        if (lane == 0) *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        __syncwarp();
    }
    if (warp == 5) {
        if (PAIR == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(tmem_slot)), "r"(tmem_columns(BQ)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_addr(tmem_slot)), "r"(tmem_columns(BQ)) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (PAIR == 2) pair_sync();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 4 || warp == 6) {
        if (PAIR == 2) full_of_first = in_first_cta(full);
        uint32_t tries = m.tries;   // after a wait that was given up the others are not waited for: the loops end, the call has failed
        while (tile < tiles) {
            if (!wait_barrier(empty + 8 * stage, (round & 1) ^ 1, tries)) tries = 0;
            if (__any_sync(kFull, tries == 0)) break;
            produce();
        }
        // the last products have let go of every stage: nothing signals here any more
        for (int i = 0; i < S; ++i) {
            if (!wait_barrier(empty + 8 * stage, (round & 1) ^ 1, tries)) tries = 0;
            if (++stage == S) {
                stage = 0;
                ++round;
            }
        }
        if (tries == 0) *gave_up = 1;
    } else if (warp == 5) {
        if (me == 0) {
            // The whole warp walks through the stages and one lane of it issues: what the products are issued with stays uniform
            // (issued from a lane on a path of its own, four products took 650 clocks, more than the tensor cores need for 256 x 256).
            constexpr uint32_t idesc = instruction_desc<CODEC, kPairP, BQ>();
            const uint64_t first = operand_desc(shared_addr(smem));
            const uint32_t stage16 = (uint32_t)kStage >> 4, sub16 = sub_bytes >> 4, q16 = (uint32_t)q_at >> 4;   // descriptors count in 16 bytes
            int s = 0, turn = 0;
            uint32_t around = 0;
            bool over = false;   // a wait was given up: nothing more is issued
            for (int64_t t = blockIdx.x / PAIR; t < tiles; t += gridDim.x / PAIR, ++turn) {
                const int a = turn & 1;
                over = __any_sync(kFull, !wait_barrier(acc_empty + 8 * a, ((turn >> 1) & 1) ^ 1, m.tries));
                if (over) break;
                fence_after();
                const uint32_t acc = tmem + a * BQ;
                for (int kb = 0; kb < blocks_k; kb += kSub) {
                    over = __any_sync(kFull, !wait_barrier(full + 8 * s, around & 1, m.tries));
                    if (over) break;
                    const uint64_t dp = first + (uint32_t)s * stage16;
                    const int left = m.k - kb * kTileK;   // 32 codes a product; the last block has as many as the rows reach into
                    if (one_lane()) {
#pragma unroll
                        for (int i = 0; i < 4 * kSub; ++i) {
                            const uint64_t at = dp + (uint32_t)(i / 4) * sub16 + 2 * (i % 4);
                            if (i == 0 || left > 32 * i) mma<CODEC, PAIR>(acc, at, at + q16, idesc, i > 0 || kb != 0);
                        }
                        mma_commit<PAIR>(empty + 8 * s);
                        if (kb + kSub >= blocks_k) mma_commit<PAIR>(acc_full + 8 * a);
                    }
                    __syncwarp();
                    if (++s == S) {
                        s = 0;
                        ++around;
                    }
                }
                if (over) break;
            }
            if (over) *gave_up = 1;
        }
    } else {
        const uint32_t acc_empty_of_first = PAIR == 2 ? in_first_cta(acc_empty) : acc_empty;
        int turn = 0;
        uint32_t copies = 0;
        for (int64_t t = blockIdx.x / PAIR; t < tiles; t += gridDim.x / PAIR, ++turn) {
            int tp, tq;
            tile_at(t, tiles_p, tiles_q, tp, tq);
            const int a = turn & 1;
            const int p = tp * step_p + (int)me * kTileP + warp * 32 + lane;
            const bool mine = p < m.p_n && warp * 32 + lane + (int)me * kTileP < step_p;
            float *qs = q_scale + a * BQ;
            for (int i = threadIdx.x; i < BQ; i += 128) {
                const int q = tq * BQ + i;
                qs[i] = q < m.q_n ? *reinterpret_cast<const float *>(m.q_rows + (int64_t)q * m.q_stride + m.k) : 0.0f;
            }
            const float ps = mine ? *reinterpret_cast<const float *>(m.p_rows + (int64_t)p * m.p_stride + m.k) : 0.0f;
            if (!wait_barrier(acc_full + 8 * a, (turn >> 1) & 1, m.tries)) *gave_up = 1;
            if (any_of_128(*gave_up != 0)) break;   // all four warps go on, or none; also: the scales are there
            fence_after();
            const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + a * BQ;
            uint8_t *buffer = out_smem + warp * kOut * kOutBytes;
            if constexpr (P_OUT_COLUMNS) {
                const int p0 = p - lane, valid = min(step_p - warp * 32, m.p_n - p0);
                if (m.out_dtype == LEGION_F32) store_turned<CODEC, float, BQ>(acc, ps, qs, buffer, tq * BQ, p0, valid, m);
                else if (m.out_dtype == LEGION_F16) store_turned<CODEC, __half, BQ>(acc, ps, qs, buffer, tq * BQ, p0, valid, m);
                else store_turned<CODEC, __nv_bfloat16, BQ>(acc, ps, qs, buffer, tq * BQ, p0, valid, m);
            } else {
                if (m.out_dtype == LEGION_F32) store_tile<CODEC, float, BQ, kOut>(acc, ps, qs, buffer, &out_map, tq * BQ, p - lane, m, copies);
                else if (m.out_dtype == LEGION_F16) store_tile<CODEC, __half, BQ, kOut>(acc, ps, qs, buffer, &out_map, tq * BQ, p - lane, m, copies);
                else store_tile<CODEC, __nv_bfloat16, BQ, kOut>(acc, ps, qs, buffer, &out_map, tq * BQ, p - lane, m, copies);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR == 2) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(acc_empty_of_first + 8 * a) : "memory");
                else bar_arrive(acc_empty + 8 * a);
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (*gave_up) {   // the copies and products that are under way land before the CTA's memory goes: they take microseconds, this waits a millisecond
        for (const long long t0 = clock64(); clock64() - t0 < 2000000;) { }
        __syncwarp();
    }
    if (PAIR == 2) pair_sync();   // nothing of the other CTA still signals here, and the products that wrote its TMEM are done
    fence_after();
    if (threadIdx.x == 0 && *gave_up) atomicCAS(&g_operator_error, 0, LEGION_E_TIMEOUT);
    if (warp == 5) {
        if (PAIR == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_columns(BQ)));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_columns(BQ)));
    }
}

// ---- few rows: no tiles ------------------------------------------------------------------------------------------------

template <int CODEC>
__device__ __forceinline__ void dot16(const uint4 &a, const uint4 &b, typename std::conditional<CODEC == LEGION_CODEC_INT8, int, float>::type &acc)
{
    const uint32_t x[4] = { a.x, a.y, a.z, a.w }, y[4] = { b.x, b.y, b.z, b.w };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (CODEC == LEGION_CODEC_INT8) {
            acc = __dp4a((int)x[i], (int)y[i], acc);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const __half2_raw p = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x[i] >> (16 * h)), __NV_E4M3);
                const __half2_raw q = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(y[i] >> (16 * h)), __NV_E4M3);
                const float2 f = __half22float2(__half2(p)), g = __half22float2(__half2(q));
                acc = fmaf(f.x, g.x, acc);
                acc = fmaf(f.y, g.y, acc);
            }
        }
    }
}

// One row against weight rows that are read once: a warp has R weight rows.  Bound by the weights' bytes, and nearly by __dp4a, which
// runs once per 7 clocks and SM: 15.7 us by 16384 x 4096, where a plain read of the 67 MB takes 12.9.  (Two rows took 20 us, eight
// 40: they go to the tensor cores, which take 18 us for up to 16.)
template <int CODEC, int R>
__global__ void __launch_bounds__(256) matvec_kernel(MatmulParams m)
{
    typedef typename std::conditional<CODEC == LEGION_CODEC_INT8, int, float>::type acc_t;
    const int lane = threadIdx.x & 31;
    const int64_t n0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * R;
    if (n0 >= m.p_n) return;
    float ws[R];   // asked for before the codes
    const float xs = *reinterpret_cast<const float *>(m.q_rows + m.k);
#pragma unroll
    for (int r = 0; r < R; ++r) ws[r] = n0 + r < m.p_n ? *reinterpret_cast<const float *>(m.p_rows + (n0 + r) * m.p_stride + m.k) : 0.0f;
    acc_t acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0;
    const int chunks = m.k / 16;   // whole 16-byte pieces
#pragma unroll 4
    for (int c = lane; c < chunks; c += 32) {
        uint4 w[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            w[r] = make_uint4(0, 0, 0, 0);
            if (n0 + r < m.p_n) w[r] = __ldcs(reinterpret_cast<const uint4 *>(m.p_rows + (n0 + r) * m.p_stride) + c);
        }
        const uint4 x = *(reinterpret_cast<const uint4 *>(m.q_rows) + c);
#pragma unroll
        for (int r = 0; r < R; ++r) dot16<CODEC>(w[r], x, acc[r]);
    }
    if (lane < (m.k % 16) / 4) {   // words behind them, one a lane
        const uint32_t x = reinterpret_cast<const uint32_t *>(m.q_rows)[chunks * 4 + lane];
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (n0 + r < m.p_n)
                dot16<CODEC>(make_uint4(reinterpret_cast<const uint32_t *>(m.p_rows + (n0 + r) * m.p_stride)[chunks * 4 + lane], 0, 0, 0),
                             make_uint4(x, 0, 0, 0), acc[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        acc_t a = acc[r];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) a += __shfl_xor_sync(kFull, a, d);
        if (lane == r && n0 + r < m.p_n) store_any(m.out, m.out_dtype, n0 + r, scaled((float)a, xs, ws[r]));
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------------

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled()
{
    static EncodeTiled fn = nullptr;
    if (fn == nullptr) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiled)p;
    }
    return fn;
}

// k codes of n rows; what a box reaches beyond them (the scales among it) arrives as zeros
static int make_map(CUtensorMap *map, const void *rows, int64_t n, int64_t stride, int32_t k, int box_rows)
{
    EncodeTiled encode = encode_tiled();
    if (encode == nullptr) {
        set_error("legion_matmul_rows: the driver has no cuTensorMapEncodeTiled");
        return LEGION_E_CUDA;
    }
    const cuuint64_t dims[2] = { (cuuint64_t)k, (cuuint64_t)n }, strides[1] = { (cuuint64_t)stride };
    const cuuint32_t box[2] = { (cuuint32_t)kTileK, (cuuint32_t)box_rows }, one[2] = { 1, 1 };
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(rows), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("legion_matmul_rows: no tensor map for %lld rows of %d codes, %lld bytes apart (%d)", (long long)n, k, (long long)stride, (int)r);
        return LEGION_E_CUDA;
    }
    return LEGION_OK;
}

// boxes of 32 rows, 128 bytes of each; what lies outside of the output is not written, behind a row's end by whole 16 bytes (store_tile sees to the rest)
static int make_out_map(CUtensorMap *map, const MatmulParams &m)
{
    EncodeTiled encode = encode_tiled();
    const int bytes = dtype_bytes(m.out_dtype);
    const cuuint64_t dims[2] = { (cuuint64_t)m.q_n, (cuuint64_t)m.p_n }, strides[1] = { (cuuint64_t)(m.out_stride * bytes) };
    const cuuint32_t box[2] = { (cuuint32_t)(128 / bytes), 32 }, one[2] = { 1, 1 };
    const CUtensorMapDataType type = m.out_dtype == LEGION_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : m.out_dtype == LEGION_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult r = encode(map, type, 2, m.out, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("legion_matmul_rows: no tensor map for an output of %d x %d, rows %lld elements apart (%d)", m.p_n, m.q_n, (long long)m.out_stride, (int)r);
        return LEGION_E_CUDA;
    }
    return LEGION_OK;
}

template <int CODEC, int BQ, bool P_OUT_COLUMNS, int PAIR>
static int launch_tiles(cudaStream_t s, MatmulParams m)
{
    CUtensorMap p_map, q_map;
    int rc = make_map(&p_map, m.p_rows, m.p_n, m.p_stride, m.k, P_OUT_COLUMNS ? m.step_p : kTileP);
    if (rc == LEGION_OK) rc = make_map(&q_map, m.q_rows, m.q_n, m.q_stride, m.k, BQ / PAIR);
    if (rc != LEGION_OK) return rc;
    CUtensorMap out_map;
    memset(&out_map, 0, sizeof(out_map));
    m.word = 16;
    while (((uintptr_t)m.out | (uintptr_t)(m.out_stride * dtype_bytes(m.out_dtype))) % m.word != 0) m.word /= 2;
    if (m.word == 16 && !P_OUT_COLUMNS) rc = make_out_map(&out_map, m);
    if (rc != LEGION_OK) return rc;
    // As many stages as there is room for: what is on its way is what hides the latency of memory.
    m.q_at = m.step_p * kTileK;
    m.stage_bytes = blocks_per_stage(BQ, PAIR) * (m.q_at + BQ / PAIR * kTileK);
    m.stages = (kSmem - smem_beside_stages(BQ, PAIR)) / m.stage_bytes;
    if (m.stages > kStagesMax) m.stages = kStagesMax;
    const int step_p = P_OUT_COLUMNS ? m.step_p : kTileP * PAIR;
    const int64_t tiles = (int64_t)((m.p_n + step_p - 1) / step_p) * ((m.q_n + BQ - 1) / BQ);
    const int64_t groups = tiles < kSms / PAIR ? tiles : kSms / PAIR, a_tile = blocks_per_stage(BQ, PAIR) * kTileK,
                  steps = (tiles + groups - 1) / groups * ((m.k + a_tile - 1) / a_tile);
    if (m.stages > steps) m.stages = (int32_t)steps;
    const int smem = m.stages * m.stage_bytes + smem_beside_stages(BQ, PAIR);
    static bool allowed[64];
    rc = allow_smem((const void *)matmul_kernel<CODEC, BQ, P_OUT_COLUMNS, PAIR>, kSmem, allowed);
    if (rc != LEGION_OK) return rc;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = PAIR;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)groups * PAIR);
    cfg.blockDim = dim3(224);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = PAIR > 1 ? 1 : 0;
    LG_CUDA(cudaLaunchKernelEx(&cfg, matmul_kernel<CODEC, BQ, P_OUT_COLUMNS, PAIR>, p_map, q_map, out_map, m));
    return LEGION_OK;
}

// Few rows on the other side: the weights' bytes are what counts, so every SM gets the same number of them.
static int32_t weights_per_cta(int64_t n)
{
    const int64_t rows = ((n + kSms - 1) / kSms + 7) / 8 * 8;
    return rows < kTileP ? (int32_t)rows : kTileP;
}

template <int CODEC>
static int launch_matmul(cudaStream_t s, const uint8_t *rows, int64_t m, int64_t row_stride, const uint8_t *weights, int64_t n,
                         int64_t weight_stride, int32_t k, void *out, int32_t out_dtype, int64_t out_stride)
{
    const MatmulParams by_weight{ weights, rows, weight_stride, row_stride, (int32_t)n, (int32_t)m, k, out, out_stride, out_dtype, 0, 0, 0, 0, weights_per_cta(n), operator_wait_tries() };
    const MatmulParams by_row{ rows, weights, row_stride, weight_stride, (int32_t)m, (int32_t)n, k, out, out_stride, out_dtype, 0, 0, 0, 0, kTileP, operator_wait_tries() };
    if (m == 1) {
        matvec_kernel<CODEC, 2><<<(unsigned)((n + 15) / 16), 256, 0, s>>>(by_weight);
        LG_LAUNCH_CHECK();
        return LEGION_OK;
    }
    if (m <= 16) return launch_tiles<CODEC, 16, true, 1>(s, by_weight);
    if (m <= 32) return launch_tiles<CODEC, 32, true, 1>(s, by_weight);
    if (m <= 64) return launch_tiles<CODEC, 64, true, 1>(s, by_weight);
    if (m <= 128) return launch_tiles<CODEC, 128, true, 1>(s, by_weight);
    // wide tiles need the fewest bytes per product; narrower ones where they would leave SMs without work
    auto cost = [&](int bp, int bq, int at_once) {
        const int64_t tiles = ((m + bp - 1) / bp) * ((n + bq - 1) / bq);
        return (tiles + at_once - 1) / at_once * (bq + 96);
    };
    const int64_t c2 = cost(256, 256, kSms / 2), c256 = cost(128, 256, kSms), c128 = cost(128, 128, kSms), c64 = cost(128, 64, kSms);
    if (c2 <= c256 && c2 <= c128 && c2 <= c64) return launch_tiles<CODEC, 256, false, 2>(s, by_row);
    if (c256 <= c128 && c256 <= c64) return launch_tiles<CODEC, 256, false, 1>(s, by_row);
    if (c128 <= c64) return launch_tiles<CODEC, 128, false, 1>(s, by_row);
    return launch_tiles<CODEC, 64, false, 1>(s, by_row);
}

}  // namespace legion

using namespace legion;

extern "C" int legion_matmul_rows(int32_t dev_id, int32_t codec, const void *rows, int64_t m, int64_t row_stride, const void *weight_rows,
                                  int64_t n, int64_t weight_stride, int32_t feature_len, void *out, int32_t out_dtype, int64_t out_stride,
                                  void *stream)
{
    LG_ARG(codec == LEGION_CODEC_INT8 || codec == LEGION_CODEC_E4M3, "codec must be INT8 or E4M3");
    LG_ARG(feature_len > 0 && feature_len % 4 == 0, "compressed rows need feature_len % 4 == 0");
    if (feature_len > LEGION_MATMUL_MAX_DIM) {
        set_error("legion_matmul_rows: rows of %d codes are above the limit of %d", feature_len, LEGION_MATMUL_MAX_DIM);
        return LEGION_E_LIMIT;
    }
    LG_ARG(m >= 0 && m < (1ll << 31) - 256 && n >= 0 && n < (1ll << 31) - 256, "m or n out of range");
    LG_ARG(m == 0 || n == 0 || (rows != nullptr && weight_rows != nullptr && out != nullptr), "NULL pointer");
    LG_ARG((uintptr_t)rows % 16 == 0 && (uintptr_t)weight_rows % 16 == 0, "compressed rows must start on multiples of 16 bytes");
    LG_ARG(row_stride % 16 == 0 && row_stride >= code_row_bytes(feature_len) && row_stride < (1ll << 40) && weight_stride % 16 == 0 &&
               weight_stride >= code_row_bytes(feature_len) && weight_stride < (1ll << 40),
           "compressed rows are (feature_len + 4) rounded up to 16 bytes long, strides are multiples of 16 bytes");
    LG_ARG(dtype_known(out_dtype), "out: dtype must be LEGION_F32, LEGION_F16 or LEGION_BF16");
    LG_ARG(out_stride >= n && out_stride <= (1ll << 40) && (uintptr_t)out % dtype_bytes(out_dtype) == 0, "bad out stride or address");
    LG_ARG(m == 0 || n == 0 || (out != rows && out != weight_rows), "out must not be one of the operands");
    if (m == 0 || n == 0) return LEGION_OK;
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    cudaStream_t s = (cudaStream_t)stream;
    if (codec == LEGION_CODEC_INT8)
        return launch_matmul<LEGION_CODEC_INT8>(s, (const uint8_t *)rows, m, row_stride, (const uint8_t *)weight_rows, n, weight_stride,
                                                feature_len, out, out_dtype, out_stride);
    return launch_matmul<LEGION_CODEC_E4M3>(s, (const uint8_t *)rows, m, row_stride, (const uint8_t *)weight_rows, n, weight_stride,
                                            feature_len, out, out_dtype, out_stride);
}

extern "C" int legion_operator_error(int32_t dev_id, void *stream, int32_t *error, int32_t reset)
{
    LG_ARG(error != nullptr, "error is NULL");
    const OnDevice on(dev_id);
    LG_CUDA(on.err);
    *error = 0;
    cudaStream_t s = (cudaStream_t)stream;
    for (int k = 0; k < 2; ++k) {
        void *word = nullptr;
        int32_t found = 0;
        LG_CUDA(k == 0 ? cudaGetSymbolAddress(&word, g_operator_error) : norm_error_word(&word));
        LG_CUDA(cudaMemcpyAsync(&found, word, 4, cudaMemcpyDeviceToHost, s));
        LG_CUDA(cudaStreamSynchronize(s));
        if (reset && found != 0) {
            LG_CUDA(cudaMemsetAsync(word, 0, 4, s));
            LG_CUDA(cudaStreamSynchronize(s));
        }
        if (*error == 0) *error = found;
    }
    return LEGION_OK;
}
