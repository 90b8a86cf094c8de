// Products of 8-bit matrices with scales per row and per column, on the 5th-generation tensor cores:
//   out[i, j] = (sum_k a[i, k] b[j, k]) * row_scale[i] * col_scale[j] + bias[j],
// the sum exact in int32 (tcgen05.mma.kind::i8, accumulators in TMEM), the rest in fp32, rounded once to the output's type.
// Operands are tiled and swizzled in memory (int8.cuh), so a pipeline stage is two contiguous copies of at most 16 KiB each,
// and a matrix serves K-major or MN-major by a bit of the instruction descriptor.
//
// Two kernels:
//   product_pair_kernel  pairs of CTAs (cta_group::2) on 256 x 256 output tiles, persistent, two accumulators per CTA so that
//                        the epilogue of a tile runs under the next one's products.  Bound by the tensor pipe: 8192^3 in
//                        333 us (3.30 POP/s), 8192 x 4096 x 4096 in 85 us (3.24).
//   product_split_kernel 128 columns of the output (lanes of TMEM) x 16 to 128 rows per CTA; the CTAs of a cluster split the
//                        contraction and join their int32 sums through distributed shared memory (whole numbers: the
//                        order does not matter).  It takes two products in one launch (a layer's two gradients), and up
//                        to 32 tokens as they are, which it quantises itself.  Bound by latencies in a row: one token
//                        through 4096 x 4096 in 7.8 us, of which the weights' 17 MB take 2.6.
// Every mbarrier wait is bounded; a CTA whose wait gives up raises the library's status word (rexsc_int8_status), stores
// nothing more (nor does any CTA that would have joined its sums), waits, again with a limit, for its copies and products in
// flight, frees its TMEM and leaves.
#include <atomic>
#include <cuda.h>

#include "int8_quant.cuh"

namespace rexsc {

namespace {

__device__ int g_i8_status = 0; // != 0: a bounded wait gave up since rexsc_int8_status was last asked

constexpr uint32_t kWaitLimit = 1u << 22;
// The block whose waits give up without asking, so that tests see what a call does then; waits for what is in flight keep
// their limit.  In the split kernel no CTA waits for another one's copies or products, so it can be any block; in the pair
// kernel they do, so that there it is all blocks or none.
constexpr unsigned kNobody = ~0u, kEverybody = ~0u - 1;
std::atomic<unsigned> g_hasty{kNobody};
__device__ __forceinline__ uint32_t wait_limit(unsigned hasty)
{
    return hasty == kEverybody || hasty == blockIdx.x ? 0u : kWaitLimit;
}

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t limit = kWaitLimit)
{
    for (uint32_t i = 0; i < limit; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
    }
    atomicExch(&g_i8_status, 1);
    return false;
}
// by a whole warp, with one answer
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, uint32_t limit = kWaitLimit)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, limit));
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank)
{
    uint32_t out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
    return out;
}
// (orders nothing but TMEM reads, which tcgen05.wait::ld and the fence before it have finished)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t mapped)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(mapped) : "memory");
}
// (these by one lane of a converged warp, for the reason that product_step has)
__device__ __forceinline__ void mbar_expect_one(uint32_t bar, uint32_t bytes)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_in_one(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// A tile of a matrix of tiles (rows of 128 bytes) into this CTA's shared memory, its bytes counted by a barrier of either CTA of
// the pair: the leader's barrier then covers both CTAs' stages.  (Passing the word on by a remote arrive at cluster scope
// instead cost 900 to 1500 cycles a stage: 8192^3 in 946 us.)
__device__ __forceinline__ void copy_tile_pair(uint32_t dst, const CUtensorMap *map, int row, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(0), "r"(row) : "memory");
}
__device__ __forceinline__ void cluster_sync()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Shared-memory matrix descriptor, 128-byte swizzle.  Both ways of reading a tile share it: rows 128 bytes apart in groups of
// 8 that are 1024 bytes apart.  K-major the rows are the operand's rows and 32 products are 32 bytes further; MN-major the
// rows are the contraction and 32 products are 32 rows (4096 bytes) further.
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr)
{
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3fff);
    d |= (uint64_t)(kI8TileBytes >> 4) << 16; // next 128 along MN (not reached: one tile is as wide)
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// Four products (128 of the contraction) and a commit, by a converged warp of which one lane issues them: kept out of a
// one-lane branch, the descriptors stay in uniform registers.  (From such a branch a step took 472 cycles to issue whatever
// its size, 512 x 4096 x 4096 on the split kernel 33 us.)
template <int kCtas>
__device__ __forceinline__ void product_step(uint32_t tmem, uint64_t da, uint64_t db, uint32_t adv_a, uint32_t adv_b,
                                             uint32_t idesc, bool add)
{
#pragma unroll
    for (int q = 0; q < 4; q++) {
        if (kCtas == 2)
            asm volatile(
                "{\n\t.reg .pred p, e;\n\tsetp.ne.u32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
                "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                "l"(da + q * adv_a), "l"(db + q * adv_b), "r"(idesc), "r"((uint32_t)(add || q)) : "memory");
        else
            asm volatile(
                "{\n\t.reg .pred p, e;\n\tsetp.ne.u32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
                "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                "l"(da + q * adv_a), "l"(db + q * adv_b), "r"(idesc), "r"((uint32_t)(add || q)) : "memory");
    }
}
__device__ __forceinline__ void commit_one(uint32_t bar)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t bar, uint32_t ctas)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
                 "h"((uint16_t)ctas) : "memory");
}
// the warp's number as a value that is the same for all of it
__device__ __forceinline__ int warp_number() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }
// instruction descriptor: int32 sums, signed 8-bit operands, their major-ness, M and N
__host__ __device__ __forceinline__ uint32_t product_idesc(int m, int n, int a_mn, int b_mn)
{
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_load32(uint32_t addr, int (&v)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, int *v)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ---- output values --------------------------------------------------------------------------------------------
__device__ __forceinline__ float load_any(const void *p, int dtype, long long i)
{
    if (dtype == REXSC_F32) return static_cast<const float *>(p)[i];
    if (dtype == REXSC_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
template <typename T> __device__ __forceinline__ T round_to(float v);
template <> __device__ __forceinline__ float round_to<float>(float v) { return v; }
template <> __device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ uint32_t pack2(__half a, __half b)
{
    return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(b) << 16;
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 a, __nv_bfloat16 b)
{
    return (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16;
}
__device__ __forceinline__ float scaled(int sum, float row, float col, float bias)
{
    return fmaf(__fmul_rn(__int2float_rn(sum), row), col, bias);
}

struct PairArgs {
    CUtensorMap map_a, map_b;   // the operands as rows of 128 bytes
    I8Product p;
    long long tiles_i, tiles_j; // 256 x 256 output tiles
    int k_blocks;
    int store_bytes;            // bytes that every row of the output is aligned to: 32, 16, or fewer
    unsigned hasty;
};

constexpr int kPairStages = 6;
constexpr int kPairStageBytes = 2 * kI8TileBytes;
constexpr int kPairThreads = 192;     // producer, products, four warps for the epilogue
constexpr int kGroupTiles = 8;        // output tile rows that share the columns' operand while it is in L2
constexpr int kPairTurnFloats = 32 * 33; // a warp's 32 x 32 outputs on their way to whole rows
constexpr size_t kPairSmem = kPairStages * kPairStageBytes + 1024 + (2 * 256 * 2 + 4 * kPairTurnFloats) * sizeof(float) + 256;

// one lane's 32 neighbouring columns of a row, which begin on 16 or 32 bytes
template <typename T>
__device__ __forceinline__ void store_row(T *dst, const float (&v)[32], int store_bytes)
{
    if constexpr (sizeof(T) == 4) {
        if (store_bytes >= 32) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + i), "f"(v[i]),
                             "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3]), "f"(v[i + 4]), "f"(v[i + 5]), "f"(v[i + 6]),
                             "f"(v[i + 7]) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<float4 *>(dst + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
    } else {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = pack2(round_to<T>(v[2 * i]), round_to<T>(v[2 * i + 1]));
        if (store_bytes >= 32) {
#pragma unroll
            for (int i = 0; i < 16; i += 8)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 2 * i), "r"(w[i]),
                             "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]),
                             "r"(w[i + 7]) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<uint4 *>(dst + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        }
    }
}

// Output tile t of the persistent schedule: groups of kGroupTiles tile rows, column by column.
__device__ __forceinline__ void tile_of(long long t, const PairArgs &a, long long *ti, long long *tj)
{
    const long long per_group = kGroupTiles * a.tiles_j, g = t / per_group, rest = t - g * per_group;
    const long long left = a.tiles_i - g * kGroupTiles, rows = left < kGroupTiles ? left : kGroupTiles;
    *tj = rest / rows;
    *ti = g * kGroupTiles + (rest - *tj * rows);
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
product_pair_kernel(const __grid_constant__ PairArgs a)
{
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    float *col_s = reinterpret_cast<float *>(smem + kPairStages * kPairStageBytes); // [buffer][scale, bias][256]
    float *turn_s = col_s + 2 * 2 * 256;
    uint64_t *bars = reinterpret_cast<uint64_t *>(turn_s + 4 * kPairTurnFloats);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kPairStages + 5);
    const uint32_t bar0 = smem_addr(bars);
    auto full = [&](int s) { return bar0 + s * 8; };
    auto empty = [&](int s) { return bar0 + (kPairStages + s) * 8; };
    auto acc_full = [&](int b) { return bar0 + (2 * kPairStages + b) * 8; };
    auto acc_empty = [&](int b) { return bar0 + (2 * kPairStages + 2 + b) * 8; };
    const uint32_t drained = bar0 + (2 * kPairStages + 4) * 8;

    const int warp = warp_number(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const long long first = blockIdx.x >> 1, step = gridDim.x >> 1, tiles = a.tiles_i * a.tiles_j;
    const uint32_t limit = wait_limit(a.hasty);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; s++) {
            mbar_init(full(s), 1); // (the leader's counts both CTAs' bytes, the other's is not used)
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; b++) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), 8); // four warps of each CTA
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    wait_previous_launch();
    // (the next launch begins when this one ends: its blocks would crowd on the SMs that have no tile here, 1537 x 1111 x 2049
    //  in training 78 us so, 72 us as it is)

    // stage and its phase, advanced together: a division in these loops costs as much as a copy
    struct Ring {
        uint32_t at = 0, phase = 0;
        __device__ __forceinline__ void next()
        {
            if (++at == kPairStages) at = 0, phase ^= 1;
        }
    };
    if (warp == 0) {
        if (lane == 0) { // ---- copies
            const int step_a = (int)a.p.a.step_k * kI8Tile, step_b = (int)a.p.b.step_k * kI8Tile;
            const uint32_t smem0 = smem_addr(smem), leader_full = map_rank(full(0), 0);
            Ring r;
            uint32_t filled = 0; // stages that have been used
            bool ok = true;
            for (long long t = first; t < tiles && ok; t += step) {
                long long ti, tj;
                tile_of(t, a, &ti, &tj);
                // a block behind the last one is read in its place: its sums are not stored
                long long ia = ti * 2 + rank, ib = tj * 2 + rank;
                ia = ia < a.p.a.mn_tiles ? ia : a.p.a.mn_tiles - 1;
                ib = ib < a.p.b.mn_tiles ? ib : a.p.b.mn_tiles - 1;
                int row_a = (int)(ia * a.p.a.step_mn) * kI8Tile, row_b = (int)(ib * a.p.b.step_mn) * kI8Tile;
                for (int k = a.k_blocks; k > 0; k--) {
                    if (filled == kPairStages) {
                        if (!(ok = mbar_wait(empty(r.at), r.phase ^ 1, limit))) break;
                    } else {
                        filled++;
                    }
                    const uint32_t dst = smem0 + r.at * kPairStageBytes, bar = leader_full + r.at * 8;
                    if (rank == 0) mbar_expect(full(r.at), 2 * kPairStageBytes);
                    copy_tile_pair(dst, &a.map_a, row_a, bar);
                    copy_tile_pair(dst + kI8TileBytes, &a.map_b, row_b, bar);
                    row_a += step_a, row_b += step_b;
                    r.next();
                }
            }
            // nothing on its way to either CTA when they leave (at once, unless a wait gave up somewhere)
            for (uint32_t j = 0; rank == 0 && j < filled; j++) {
                const bool before = filled == kPairStages && j >= r.at; // last filled in the turn before this one
                mbar_wait(full(j), before ? r.phase ^ 1 : r.phase);
            }
        }
    } else if (warp == 1) {
        if (rank == 0) { // ---- products
            const uint32_t idesc = product_idesc(256, 256, a.p.a.mn_major, a.p.b.mn_major);
            const uint32_t adv_a = a.p.a.mn_major ? 4096 >> 4 : 32 >> 4, adv_b = a.p.b.mn_major ? 4096 >> 4 : 32 >> 4;
            const uint64_t desc0 = tile_desc(smem_addr(smem));
            Ring r;
            int turn = 0;
            bool ok = true;
            for (long long t = first; t < tiles && ok; t += step, turn++) {
                const int b = turn & 1;
                if (turn >= 2 && !(ok = mbar_wait_warp(acc_empty(b), (turn / 2 - 1) & 1, limit))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int k = 0; k < a.k_blocks; k++) {
                    if (!(ok = mbar_wait_warp(full(r.at), r.phase, limit))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t da = desc0 + r.at * (kPairStageBytes >> 4);
                    product_step<2>(tmem + b * 256, da, da + (kI8TileBytes >> 4), adv_a, adv_b, idesc, k > 0);
                    commit_pair(empty(r.at), 3);
                    r.next();
                }
                if (ok) commit_pair(acc_full(b), 3);
            }
            if (!ok) { // products in flight read both CTAs' stages and write their accumulators
                commit_pair(drained, 1);
                mbar_wait_warp(drained, 0);
            }
        }
    } else { // ---- epilogue: a lane per row of this CTA's 128
        const int quad = warp & 3, et = threadIdx.x - 64;
        const uint32_t leader_empty = map_rank(acc_empty(0), 0);
        T *out = static_cast<T *>(a.p.out);
        int turn = 0;
        for (long long t = first; t < tiles; t += step, turn++) {
            const int b = turn & 1;
            long long ti, tj;
            tile_of(t, a, &ti, &tj);
            const long long row = ti * 256 + rank * 128 + quad * 32 + lane, col0 = tj * 256;
            float *cs = col_s + b * 512;
            for (int i = et; i < 256; i += 128) {
                const bool live = col0 + i < a.p.n;
                cs[i] = live && a.p.col_scale ? a.p.col_scale[col0 + i] : 1.f;
                cs[256 + i] = live && a.p.bias ? load_any(a.p.bias, a.p.bias_dtype, col0 + i) : 0.f;
            }
            const float rs = row < a.p.m ? a.p.row_scale[row] : 0.f;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            // one lane of a warp asks: 128 threads that poll cost the copying thread a fifth of its rate
            const bool there = lane != 0 || mbar_wait(acc_full(b), (turn / 2) & 1, limit);
            if (!__all_sync(0xffffffffu, there)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c = 0; c < 256; c += 32) {
                if (col0 + c >= a.p.n) break; // (the same for all lanes)
                __syncwarp();
                int v[32];
                tmem_load32(tmem + ((uint32_t)(quad * 32) << 16) + b * 256 + c, v);
                float f[32];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 s4 = *reinterpret_cast<const float4 *>(cs + c + i), b4 = *reinterpret_cast<const float4 *>(cs + 256 + c + i);
                    f[i] = scaled(v[i], rs, s4.x, b4.x), f[i + 1] = scaled(v[i + 1], rs, s4.y, b4.y);
                    f[i + 2] = scaled(v[i + 2], rs, s4.z, b4.z), f[i + 3] = scaled(v[i + 3], rs, s4.w, b4.w);
                }
                const long long left = a.p.n - (col0 + c);
                if (left >= 32 && a.store_bytes >= 16) { // a lane's columns are whole vectors
                    if (row < a.p.m) store_row(out + row * a.p.out_stride + col0 + c, f, a.store_bytes);
                } else { // turned over in shared memory, so that a warp stores 32 neighbours of a row at a time
                    float *mine = turn_s + quad * kPairTurnFloats;
#pragma unroll
                    for (int i = 0; i < 32; i++) mine[lane * 33 + i] = f[i];
                    __syncwarp();
                    const long long top = row - lane; // the warp's first row
                    const int rows = a.p.m - top < 32 ? (int)(a.p.m - top) : 32;
                    T *to = out + top * a.p.out_stride + col0 + c + lane;
                    if (lane < left)
#pragma unroll 8
                        for (int i = 0; i < rows; i++, to += a.p.out_stride) *to = round_to<T>(mine[i * 33 + lane]);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(leader_empty + b * 8);
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

struct SplitProblem {
    I8Product p;
    long long tiles_j;  // blocks of 128 output columns
    int rows;           // output rows per CTA: 16, 32, 64 or 128
    int k_blocks;
    int stages;
    int q_bytes;        // bytes of a stage's rows operand
    int tmem_cols;
    int store_bytes;
};
struct SplitArgs {
    SplitProblem p[2];
    unsigned first;     // CTAs of p[0]; the others work on p[1]
    int split;          // CTAs of a cluster
    const void *x;      // tokens in place of p[0]'s rows operand
    long long x_stride;
    int x_vec;          // its rows begin on 16 bytes
    int whole_rows;     // every CTA reads whole rows for their largest magnitudes
    unsigned hasty;
};

constexpr int kSplitThreads = 128;
constexpr int kSplitMaxStages = 12;
constexpr size_t kSplitSmemMost = 212 * 1024;
constexpr int kTokenRows = 32;                      // most tokens that the kernel quantises by itself
constexpr int kTokenMaxValues = 4096;               // values a CTA quantises at the most: with more of them a launch of its own
                                                    // is sooner done (13 x 2051 fp16 on 5003 channels: 23 us here, 9 us so)

__device__ __forceinline__ void store1(void *out, int dtype, long long i, float v)
{
    if (dtype == REXSC_F32) static_cast<float *>(out)[i] = v;
    else if (dtype == REXSC_F16) static_cast<__half *>(out)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(out)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ void store4(void *out, int dtype, long long i, const float (&v)[4], int live, bool aligned)
{
    if (live >= 4 && aligned) {
        if (dtype == REXSC_F32)
            *reinterpret_cast<float4 *>(static_cast<float *>(out) + i) = make_float4(v[0], v[1], v[2], v[3]);
        else if (dtype == REXSC_F16)
            *reinterpret_cast<uint2 *>(static_cast<__half *>(out) + i) =
                make_uint2(pack2(__float2half_rn(v[0]), __float2half_rn(v[1])), pack2(__float2half_rn(v[2]), __float2half_rn(v[3])));
        else
            *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(out) + i) = make_uint2(
                pack2(__float2bfloat16_rn(v[0]), __float2bfloat16_rn(v[1])), pack2(__float2bfloat16_rn(v[2]), __float2bfloat16_rn(v[3])));
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (k < live) store1(out, dtype, i + k, v[k]);
    }
}

// X: int8_t where the rows operand is a matrix of tiles; else the type of up to 32 tokens that every CTA quantises for itself,
// its part of the contraction only: the CTAs of a cluster tell one another the largest magnitudes of their parts.
template <typename X>
__global__ void __launch_bounds__(kSplitThreads)
product_split_kernel(const __grid_constant__ SplitArgs args)
{
    constexpr bool kTokens = !std::is_same<X, int8_t>::value;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kSplitMaxStages + 1];
    __shared__ uint32_t tmem_slot, gave_up; // gave_up: 1 once a wait of this CTA has given up
    __shared__ uint32_t part_most[kTokenRows];
    __shared__ float row_a[kTokenRows], row_inv[kTokenRows], row_s[kSplitThreads];
    uint8_t *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const uint32_t bar0 = smem_addr(bars);
    auto full = [&](int s) { return bar0 + s * 8; };
    auto empty = [&](int s) { return bar0 + (kSplitMaxStages + s) * 8; };
    const uint32_t acc_full = bar0 + 2 * kSplitMaxStages * 8;
    const int warp = warp_number(), lane = threadIdx.x & 31;
    const int which = !kTokens && blockIdx.x >= args.first;
    const SplitProblem &a = args.p[which];
    const int split = args.split, rank = split > 1 ? (int)cluster_rank() : 0;
    const unsigned tile = (blockIdx.x - (which ? args.first : 0)) / split;
    const long long ti = tile / a.tiles_j, tj = tile - ti * a.tiles_j;
    const int k0 = (int)((long long)rank * a.k_blocks / split), nk = (int)((long long)(rank + 1) * a.k_blocks / split) - k0;
    const long long row0 = ti * a.rows, col0 = tj * 128;
    const int rows = a.p.m - row0 < a.rows ? (int)(a.p.m - row0) : a.rows; // that exist
    const uint32_t smem0 = smem_addr(smem), stage_bytes = kI8TileBytes + (kTokens ? 0 : a.q_bytes);
    const uint32_t tokens0 = smem0 + a.stages * stage_bytes; // the quantised tokens, [128 columns][rows][128 bytes]
    const int early = nk < a.stages ? nk : a.stages;
    const uint32_t limit = wait_limit(args.hasty);

    if (kTokens) wait_previous_launch(); // (it may be the one that quantises the weights)
    const int8_t *pw = a.p.b.data + ((size_t)(tj * a.p.b.step_mn) + (size_t)(k0 * a.p.b.step_k)) * kI8TileBytes;
    const size_t step_w = (size_t)a.p.b.step_k * kI8TileBytes;
    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < a.stages; s++) mbar_init(full(s), 1), mbar_init(empty(s), 1);
            mbar_init(acc_full, 1);
            gave_up = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        // the weights depend neither on the tokens nor, where that quantises the rows, on the launch before: begin with them
        for (int s = 0; s < early; s++) {
            mbar_expect_one(full(s), stage_bytes);
            copy_in_one(smem0 + s * stage_bytes, pw, kI8TileBytes, full(s));
            pw += step_w;
        }
    }
    // TMEM is taken once the CTAs of the cluster need nothing more from one another until it has been given back: a CTA that
    // holds some waits for nobody but its own copies and products, so that whoever waits for TMEM on this SM (of whatever
    // kernel) always gets it
    auto take_tmem = [&]() {
        if (warp == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)), "r"((uint32_t)a.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    };
    __syncwarp();
    if constexpr (kTokens) {
        const X *x = static_cast<const X *>(args.x);
        // warps to a row: all four have the only token, two each of two, else every warp has rows of its own, four of which
        // it reads side by side
        const int team = rows == 1 ? 4 : rows == 2 ? 2 : 1, part = warp % team, first_row = warp / team, pace = 4 / team;
        // where a row is short its largest magnitude is found by every CTA, else its parts' are exchanged
        const bool whole = split == 1 || args.whole_rows;
        const long long c0 = whole ? 0 : (long long)k0 * 128, c1 = whole ? a.p.k : (long long)(k0 + nk) * 128;
        if (threadIdx.x < kTokenRows) part_most[threadIdx.x] = 0;
        __syncthreads();
        for (int r0 = first_row; r0 < rows; r0 += 4 * pace) {
            uint32_t most[4] = {0, 0, 0, 0};
            for (long long c = c0 + (part * 32 + lane) * 8; c < c1; c += team * 256) {
                Raw<X> raw[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (r0 + i * pace < rows) load_raw(x + (r0 + i * pace) * args.x_stride, c, a.p.k, args.x_vec, raw[i]);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (r0 + i * pace < rows) most_of(raw[i], most[i]);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t all = __reduce_max_sync(0xffffffffu, most_as_f32<X>(most[i]));
                if (lane == 0 && r0 + i * pace < rows) atomicMax(&part_most[r0 + i * pace], all);
            }
        }
        if (whole) __syncthreads();
        else cluster_sync();
        if (threadIdx.x < kTokenRows) {
            uint32_t all = part_most[threadIdx.x];
            if (!whole)
                for (int r = 0; r < split; r++) {
                    uint32_t v;
                    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(map_rank(smem_addr(&part_most[threadIdx.x]), r)) : "memory");
                    all = max(all, v);
                }
            const bool fine = all < 0x7f800000u, live = fine && all != 0;
            row_a[threadIdx.x] = live ? __uint_as_float(all) : 0.f;
            row_inv[threadIdx.x] = live ? inverse_of(__uint_as_float(all)) : 0.f;
            row_s[threadIdx.x] = fine ? __fdiv_rn(__uint_as_float(all), 127.f) : __uint_as_float(0x7fc00000u);
        }
        __syncwarp();
        take_tmem();
        __syncthreads();
        for (int r0 = first_row; r0 < rows; r0 += 4 * pace)
            for (int c = (part * 32 + lane) * 8; c < nk * 128; c += team * 256) {
                Raw<X> raw[4];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (r0 + i * pace < rows)
                        load_raw(x + (r0 + i * pace) * args.x_stride, (long long)k0 * 128 + c, a.p.k, args.x_vec, raw[i]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = r0 + i * pace;
                    if (r >= rows) continue;
                    float f[8];
                    widen(raw[i], f);
                    const float largest = row_a[r];
                    const uint2 q = largest > 0.f ? quant8<sizeof(X) == 2>(f, largest, row_inv[r]) : make_uint2(0u, 0u);
                    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(tokens0 + (c >> 7) * a.q_bytes + r * 128 +
                                                                         ((((c >> 4) & 7) ^ (r & 7)) << 4) + (c & 8)),
                                 "r"(q.x), "r"(q.y) : "memory");
                }
            }
        // what was written is visible to the tensor core's reads
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
    } else {
        take_tmem();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        // ---- copies
        const int8_t *px = a.p.a.data + ((size_t)((row0 >> 7) * a.p.a.step_mn) + (size_t)(k0 * a.p.a.step_k)) * kI8TileBytes +
                           (a.p.a.mn_major ? 0 : (row0 & 127) * 128);
        const size_t step_x = (size_t)a.p.a.step_k * kI8TileBytes;
        auto copy_x = [&](int s) {
            if (!kTokens) copy_in_one(smem0 + s * stage_bytes + kI8TileBytes, px, a.q_bytes, full(s));
            px += step_x;
        };
        if (!kTokens) wait_previous_launch();
        allow_next_launch(); // (TMEM has been taken)
        for (int s = 0; s < early; s++) copy_x(s);
        int s = 0, phase = 0, filled = early;
        for (; filled < nk; filled++) {
            if (!mbar_wait_warp(empty(s), phase, limit)) break; // (the products' warp then gives up too)
            mbar_expect_one(full(s), stage_bytes);
            copy_in_one(smem0 + s * stage_bytes, pw, kI8TileBytes, full(s));
            pw += step_w;
            copy_x(s);
            if (++s == a.stages) s = 0, phase ^= 1;
        }
        // nothing on its way when this CTA leaves: the last filling of every stage
        for (int j = filled < a.stages ? 0 : filled - a.stages; j < filled; j++) mbar_wait_warp(full(j % a.stages), (j / a.stages) & 1);
    } else if (warp == 1) {
        // ---- products: lanes are output columns, columns of TMEM output rows
        if (!kTokens) wait_previous_launch(); // (which may take longer than a bounded wait)
        const uint32_t idesc = product_idesc(128, a.rows, a.p.b.mn_major, a.p.a.mn_major);
        const uint32_t adv_w = a.p.b.mn_major ? 4096 >> 4 : 32 >> 4, adv_x = a.p.a.mn_major ? 4096 >> 4 : 32 >> 4;
        const uint64_t desc_w = tile_desc(smem0), desc_x = tile_desc(kTokens ? tokens0 : smem0 + kI8TileBytes);
        int s = 0, phase = 0;
        for (int i = 0; i < nk; i++) {
            if (!mbar_wait_warp(full(s), phase, limit)) {
                gave_up = 1;
                break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            product_step<1>(tmem, desc_w + (s * stage_bytes >> 4), desc_x + ((kTokens ? i * a.q_bytes : s * stage_bytes) >> 4),
                            adv_w, adv_x, idesc, i > 0);
            if (i + a.stages < nk) commit_one(empty(s)); // (filled again)
            if (++s == a.stages) s = 0, phase ^= 1;
        }
        commit_one(acc_full); // (after a wait that gave up: of what was issued)
    }
    __syncwarp();
    if (!kTokens) {
        wait_previous_launch();
        if (threadIdx.x < rows) row_s[threadIdx.x] = a.p.row_scale[row0 + threadIdx.x];
        __syncwarp();
    }
    bool done = true;
    if (lane == 0) { // (one lane of a warp asks)
        done = mbar_wait(acc_full, 0, limit);
        if (!done) { // products in flight read this CTA's stages and write its TMEM
            gave_up = 1;
            mbar_wait(acc_full, 0);
        }
    }
    done = __all_sync(0xffffffffu, done);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_lane = tmem + ((uint32_t)(warp * 32) << 16);
    auto free_tmem = [&]() {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();
        if (warp == 1) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)a.tmem_cols) : "memory");
        }
    };
    // sums to shared memory, [row][column]; every CTA of the cluster finishes some of the rows, four columns a lane.  (The copies
    // have landed where the sums go: all of them have been multiplied, or a wait gave up and the sums are not used.)
    int *red = reinterpret_cast<int *>(smem);
    for (int c = 0; c < rows && done; c += 16) {
        int v[16];
        __syncwarp();
        tmem_load16(tmem_lane + c, v);
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (c + i < rows) red[(c + i) * 128 + warp * 32 + lane] = v[i];
    }
    __syncwarp();
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    free_tmem(); // (its barrier is enough for a CTA alone)
    __syncwarp();
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const long long col = col0 + lane * 4;
    const int live = a.p.n - col < 4 ? (int)(a.p.n - col) : 4; // (0 or less behind the last column: nothing is stored)
    float cs[4], bias[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        cs[i] = i < live && a.p.col_scale ? a.p.col_scale[col + i] : 1.f;
        bias[i] = i < live && a.p.bias ? load_any(a.p.bias, a.p.bias_dtype, col + i) : 0.f;
    }
    // whether any CTA of the cluster gave up: a lane asks one of them (the answer travels beside the first sums)
    uint32_t bad;
    if (split > 1)
        asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(bad) : "r"(map_rank(smem_addr(&gave_up), lane & (split - 1))) : "memory");
    else
        bad = gave_up;
    for (int c = rank * 4 + warp; c < rows; c += 4 * split) {
        int4 sum = *reinterpret_cast<const int4 *>(red + c * 128 + lane * 4);
        const uint32_t at = smem_addr(red + c * 128 + lane * 4);
        for (int i = 1; i < split; i++) {
            const int r = (rank + i) & (split - 1); // (each starts with another one)
            int4 v;
            asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(map_rank(at, r)) : "memory");
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        const float rs = row_s[c];
        const float f[4] = {scaled(sum.x, rs, cs[0], bias[0]), scaled(sum.y, rs, cs[1], bias[1]),
                            scaled(sum.z, rs, cs[2], bias[2]), scaled(sum.w, rs, cs[3], bias[3])};
        if (__any_sync(0xffffffffu, bad)) break;
        store4(a.p.out, a.p.out_dtype, (row0 + c) * a.p.out_stride + col, f, live, a.store_bytes >= 16);
    }
    if (split > 1) cluster_sync(); // the others still read this CTA's sums
}

// ---- host -----------------------------------------------------------------------------------------------------
int store_alignment(const I8Product &p)
{
    const uintptr_t bits = reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.out_stride * (long long)dtype_bytes(p.out_dtype));
    return bits & 15 ? 0 : bits & 31 ? 16 : 32;
}

// kSmemMost: what any launch of the kernel asks for.  The kernel is allowed that much once per device (and not what a launch
// needs: two threads would take it from one another).
template <auto kKernel, size_t kSmemMost, typename Args>
int launch_cluster(const Args &args, long long blocks, int cluster, int threads, size_t smem, bool overlap, cudaStream_t st,
                   const char *name)
{
    if (blocks > 0x7fffffffll) return REXSC_E_UNSUPPORTED;
    static std::atomic<unsigned long long> allowed{0};
    int device = 0;
    REXSC_CUDA_CHECK(cudaGetDevice(&device));
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        REXSC_CUDA_CHECK(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMost));
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    if (overlap) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = (unsigned)n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kKernel, args);
    note_kernel_launch();
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_cuda_error(e, name);
        return REXSC_E_CUDA;
    }
    return REXSC_OK;
}

// a matrix of tiles as rows of 128 bytes, taken 128 rows at a time
int tile_map(CUtensorMap *map, const I8Operand &o, long long k_tiles)
{
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                               const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<Encode>(fn);
    }();
    const long long rows = o.mn_tiles * k_tiles * kI8Tile;
    if (!encode || rows > 0x7fffffffll) return REXSC_E_UNSUPPORTED;
    const cuuint64_t extent[2] = {kI8Tile, (cuuint64_t)rows}, pitch[1] = {kI8Tile};
    const cuuint32_t box[2] = {kI8Tile, kI8Tile}, each[2] = {1, 1};
    const CUresult rc = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(o.data), extent, pitch, box, each,
                               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? REXSC_OK : REXSC_E_BAD_ARG;
}

template <typename T>
int launch_pair(const I8Product &p, bool overlap, cudaStream_t st)
{
    PairArgs a;
    a.p = p;
    int rc = tile_map(&a.map_a, p.a, i8_tiles(p.k));
    if (rc == REXSC_OK) rc = tile_map(&a.map_b, p.b, i8_tiles(p.k));
    if (rc != REXSC_OK) return rc;
    a.tiles_i = (p.m + 255) / 256;
    a.tiles_j = (p.n + 255) / 256;
    a.k_blocks = (int)i8_tiles(p.k);
    a.store_bytes = store_alignment(p);
    a.hasty = g_hasty.load(std::memory_order_relaxed) == kEverybody ? kEverybody : kNobody;
    const long long tiles = a.tiles_i * a.tiles_j, pairs = tiles < 74 ? tiles : 74;
    return launch_cluster<product_pair_kernel<T>, kPairSmem>(a, pairs * 2, 0, kPairThreads, kPairSmem, overlap, st, "product_pair_kernel");
}

// ---- which kernel, and its shape
long long split_shape(SplitProblem *a, const I8Product &p)
{
    a->p = p;
    a->tiles_j = (p.n + 127) / 128;
    a->k_blocks = (int)i8_tiles(p.k);
    a->rows = p.a.mn_major || p.m > 64 ? 128 : p.m > 32 ? 64 : p.m > 16 ? 32 : 16;
    a->q_bytes = p.a.mn_major ? kI8TileBytes : a->rows * 128;
    a->tmem_cols = a->rows < 32 ? 32 : a->rows;
    a->store_bytes = store_alignment(p);
    return a->tiles_j * ((p.m + a->rows - 1) / a->rows);
}

// CTAs that share a contraction: as many as leave each a step of 128 and all of them on the GPU at once.  One CTA that uses
// TMEM fits an SM, and clusters of 1, 2, 4 and 8 leave some of the 148 SMs out (132 and 120 of them can be had by 4 and 8).
int split_of(long long tiles, int k_blocks)
{
    const int most[4] = {148, 148, 132, 120};
    int split = 1;
    for (int i = 1; i < 4 && (1 << i) <= k_blocks; i++)
        if (tiles << i <= most[i]) split = 1 << i;
    return split;
}

// The kernel that takes less time by what they were measured at (us, B200, bf16): pairs 5.6 + 0.28 for every step of 128 along
// the contraction and wave of 74 output tiles; the split 2 and for every wave of 148 CTAs 3 + 0.027 rows and for every step
// of a CTA 0.14 + 0.0006 rows.  Whole calls: 1024 x 2048 x 512 pairs 9.9, split 12.3; 512 x 4096 x 4096 18.4 and 18.7;
// 192 x 8192 x 8192 29.7 and 25.3; 64 x 8192 x 8192 26.0 and 15.6.
bool use_pairs(const I8Product &p, int kernel)
{
    if (kernel != REXSC_INT8_AUTO) return kernel == REXSC_INT8_PAIR;
    SplitProblem a;
    const long long tiles = split_shape(&a, p), pairs = ((p.m + 255) / 256) * ((p.n + 255) / 256);
    const int split = split_of(tiles, a.k_blocks);
    const double waves = (double)((tiles * split + 147) / 148), steps = (a.k_blocks + split - 1) / split;
    return 5.6 + (double)((pairs + 73) / 74) * a.k_blocks * 0.28 < 2 + waves * (3 + 0.027 * a.rows + steps * (0.14 + 0.0006 * a.rows));
}

// stages of a CTA, and the shared memory that it needs
size_t split_stages(SplitProblem *a, int split, bool tokens)
{
    const int steps = (a->k_blocks + split - 1) / split, fixed = tokens ? steps * a->q_bytes : 0;
    const int stage = kI8TileBytes + (tokens ? 0 : a->q_bytes), most = ((int)kSplitSmemMost - 1024 - fixed) / stage;
    a->stages = steps < kSplitMaxStages ? steps : kSplitMaxStages;
    if (a->stages > most) a->stages = most;
    size_t smem = (size_t)a->stages * stage + fixed;
    if (smem < (size_t)a->rows * 512) smem = (size_t)a->rows * 512; // the sums
    return smem + 1024;
}

int launch_split(const I8Product &p, const I8Product *second, bool overlap, cudaStream_t st)
{
    SplitArgs a = {};
    a.hasty = g_hasty.load(std::memory_order_relaxed);
    const long long tiles = split_shape(&a.p[0], p), more = second ? split_shape(&a.p[1], *second) : 0;
    int k_blocks = a.p[0].k_blocks;
    if (second && a.p[1].k_blocks < k_blocks) k_blocks = a.p[1].k_blocks;
    a.split = split_of(tiles + more, k_blocks);
    size_t smem = split_stages(&a.p[0], a.split, false);
    if (second) {
        const size_t other = split_stages(&a.p[1], a.split, false);
        if (other > smem) smem = other;
    }
    if ((tiles + more) * a.split > 0x7fffffffll) return REXSC_E_UNSUPPORTED;
    a.first = (unsigned)(tiles * a.split);
    return launch_cluster<product_split_kernel<int8_t>, kSplitSmemMost>(a, (tiles + more) * a.split, a.split, kSplitThreads, smem,
                                                                        overlap, st, "product_split_kernel");
}

} // namespace

int launch_i8_product(const I8Product &p, int kernel, bool after_quantize, cudaStream_t st)
{
    if (!use_pairs(p, kernel)) return launch_split(p, nullptr, after_quantize, st);
    switch (p.out_dtype) {
    case REXSC_F32: return launch_pair<float>(p, after_quantize, st);
    case REXSC_F16: return launch_pair<__half>(p, after_quantize, st);
    default: return launch_pair<__nv_bfloat16>(p, after_quantize, st);
    }
}

int launch_i8_products(const I8Product &p, const I8Product &q, int kernel, bool after_quantize, cudaStream_t st)
{
    if (!use_pairs(p, kernel) && !use_pairs(q, kernel)) return launch_split(p, &q, after_quantize, st);
    const int rc = launch_i8_product(p, kernel, after_quantize, st);
    return rc == REXSC_OK ? launch_i8_product(q, kernel, true, st) : rc;
}

bool i8_tokens_fit(long long m, long long n, long long k, int kernel)
{
    if (m > kTokenRows || kernel == REXSC_INT8_PAIR) return false;
    const long long k_blocks = i8_tiles(k);
    const int split = split_of((n + 127) / 128, (int)k_blocks);
    return m * ((k_blocks + split - 1) / split) * 128 <= kTokenMaxValues;
}

int launch_i8_tokens(const void *x, int dtype, long long stride, const I8Product &p, cudaStream_t st)
{
    SplitArgs a = {};
    a.hasty = g_hasty.load(std::memory_order_relaxed);
    const long long tiles = split_shape(&a.p[0], p);
    a.split = split_of(tiles, a.p[0].k_blocks);
    const size_t smem = split_stages(&a.p[0], a.split, true);
    if (tiles * a.split > 0x7fffffffll) return REXSC_E_UNSUPPORTED;
    a.first = (unsigned)(tiles * a.split);
    a.x = x;
    a.x_stride = stride;
    // (16 KiB: a CTA's 128 threads read that much in about the time that an exchange within the cluster takes)
    a.whole_rows = p.m * p.k * (long long)dtype_bytes(dtype) <= 16 * 1024;
    a.x_vec = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(stride * (long long)dtype_bytes(dtype))) & 15) == 0;
#define REXSC_I8_TOKENS(X)                                                                                             \
    launch_cluster<product_split_kernel<X>, kSplitSmemMost>(a, tiles *a.split, a.split, kSplitThreads, smem, true, st,  \
                                                            "product_split_kernel")
    return dtype == REXSC_F32 ? REXSC_I8_TOKENS(float) : dtype == REXSC_F16 ? REXSC_I8_TOKENS(__half) : REXSC_I8_TOKENS(__nv_bfloat16);
#undef REXSC_I8_TOKENS
}

} // namespace rexsc

extern "C" int rexsc_int8_status(void *stream)
{
    using namespace rexsc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int seen = 0;
    const int none = 0;
    REXSC_CUDA_CHECK(cudaMemcpyFromSymbolAsync(&seen, g_i8_status, sizeof(seen), 0, cudaMemcpyDeviceToHost, st));
    REXSC_CUDA_CHECK(cudaStreamSynchronize(st));
    if (seen) REXSC_CUDA_CHECK(cudaMemcpyToSymbolAsync(g_i8_status, &none, sizeof(none), 0, cudaMemcpyHostToDevice, st));
    return seen ? REXSC_E_DEVICE_TIMEOUT : REXSC_OK;
}

extern "C" int rexsc_int8_test_waits(int64_t block)
{
    using namespace rexsc;
    if (block < -2 || block > 0x7fffffffll) return REXSC_E_BAD_ARG;
    g_hasty.store(block == -1 ? kNobody : block == -2 ? kEverybody : (unsigned)block, std::memory_order_relaxed);
    return REXSC_OK;
}
