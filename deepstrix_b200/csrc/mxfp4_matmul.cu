// out[m, n] = sum over terms and k of A_term[m, k] * W[n, k]: both operands MXFP4 rows as stored, on the block-scaled FP4 tensor
// cores (tcgen05.mma.kind::mxf4.block_scale), f32 accumulation in tensor memory, one rounding.
//
// Reference counterparts (paths relative to the deepstrix repository): the dense GEMV / GEMM of its projections and head
// (crates/v4flash-kernels/kernels/q8_0_matvec.hip:64-150, f16_gemm_wmma.hip) and the FP4 product of its CPU model
// (scripts/v41_oracle/kernel.py:161-167).
//
// Tile.  128 rows of W are the MMA's M side (a tensor-memory lane each), A's rows its N side, so that one token and a few hundred run on the
// same kernel: a decode batch is a narrow N under a stream of weights.  Terms of A: a single CTA takes up to 208 rows of all terms together
// as N -- an MMA costs 50 clocks to issue and no less, so one of N = 48 replaces three of N = 16 -- and the read-out adds each token's terms; a
// pair of CTAs takes up to 128 tokens and runs a term after the other into the same accumulator.  Either way W is read once for all terms.
// A pipeline stage is 256 columns: 128-byte rows (128-byte swizzle) of W and of A, each one TMA box, zero-filled past the operand's edges.
// Scales are read as stored (row-major bytes; nothing is laid out beforehand), 16 bytes of every row -- 512 columns, two stages -- at a time
// into a ring of their own: by TMA where rows of scales are 16-byte aligned (K a multiple of 512), else by four loader warps, a row of
// every 128-row group a thread, as the aligned 16-byte words that hold them, requested a step ahead and shifted into place (8192 x 8192 x 4128
// takes 165 us, with K of 4096 and TMA 118; when it took 160, words of 4 bytes took 178 and loaders that moved every other buffer to
// tensor memory as well 168).  Scale warps, one per lane quarter, move a
// buffer to a slot of tensor memory at a time (ld.shared + tcgen05.st; the tensor core's own copy would queue behind its MMAs); where TMA
// brings the scales the loader warps are a second set of them, and the sets take alternate buffers: one set alone needed 800 clocks a stage.
// Warp roles: TMA of codes, MMA issue, TMA of scales, one idle, 4 scale warps, 4 epilogue warps, 4 loaders or scale warps; two accumulators, so that a
// tile is read out under the next one's MMAs.
// Few tiles: the columns are split over the CTAs of a cluster; each leaves its partial tile in shared memory and the cluster adds
// them in rank order through distributed shared memory, so results do not depend on timing and need no workspace.
// Every wait on a barrier in shared memory is bounded; when one runs out the block lets what it has in flight finish (bounded too: MMAs and copies
// are waited for by the roles that issue them, always, since another role may give up after they have ended), frees its tensor memory and sets bit 1
// of the error word.  Not bounded, because they end by themselves: the wait for the kernel before this one, the barriers of
// a cluster (every role of every block comes to them) and the wait for tensor memory, which kernels of this library give back without
// waiting for another block, or hold alone on their SM (see the two sizes of block below).
//
// Bound and measured (launches back to back, operands that rotate; a burst, and in brackets after a second of it, at the clock of the power cap).
// A few tokens: the weights' bytes; 8 x 131072 x 4096 of three terms takes 54 us (55), 5.3 TB/s, of which about 7 us are start and end -- every
// further 37888 rows of W take 12.8 us, 6.45 TB/s.  One small matrix (1 x 1024 x 2048): 6 us, all of it latency.  Many tokens: the issuing
// warp's clocks and the power cap; 8192 x 8192 x 4096 takes 119 us (139) with one term, 4.6 PFLOP/s (4.0), 289 (333) with three, 5.7 PFLOP/s (4.9)
// of MMAs executed; 64 x 131072 x 4096 of three terms 62 (74), 777 x 5119 x 2336 20.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "head.cuh"
#include "prefill.cuh"

namespace dsx {
namespace {

__device__ uint32_t g_head_error = 0;

constexpr int kEpiWarp0 = 8, kLoadWarp0 = 12, kThreads = 512;   // roles start on warp-group boundaries
constexpr int kLoaders = 128;
constexpr int kWRows = 128;          // W rows of a tile
constexpr int kStageK = 256;         // columns of a stage
constexpr int kRowBytes = kStageK / 2;
constexpr int kWBytes = kWRows * kRowBytes;
constexpr int kGroupBytes = 2048;    // scale bytes of a group of 128 rows: 16 a row, two stages
constexpr int kMaxScaleBufs = 4;     // two or four: see plan_block
constexpr int kMaxSlots = 4;         // of scales in tensor memory, two stages each
constexpr int kMaxStages = 8;
constexpr int kMaxN = 208;           // of an MMA: two accumulators and two scale slots fill tensor memory
constexpr uint32_t kPolls = 1u << 22;     // of a wait, unless dsx_mxfp4_matmul_set_polls says otherwise; a poll that fails takes 2 to 4 us
constexpr uint32_t kDrainPolls = 1u << 16;   // for what is in flight when a role has nothing more to do

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Takes `bytes` off what a barrier's phase still expects, as a copy of that size would.
__device__ __forceinline__ void mbar_complete_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// How long a wait lasts, and where a role that has given up says so to the others of its block.
struct Patience {
    volatile uint32_t* abort_flag;
    uint32_t polls;
};
// Bounded wait that also gives up when another role of the block has.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const Patience& p) {
    for (uint32_t i = 0; i < p.polls; i++) {
        if (mbar_try(bar, parity)) return true;
        if ((i & 15u) == 15u && *p.abort_flag) return false;
    }
    *p.abort_flag = 1u;
    return false;
}
// The same for a warp that goes on as one.  Its lanes may see the phase complete at different polls, and what follows (tcgen05 loads and
// stores, MMAs from uniform registers) wants them together: hence the __syncwarp, and no branch on the outcome -- when the wait runs out the
// warp goes on to the tile's end, and what it then computes is reported as missing.  `leader` is cleared in a lane whose wait ran out.
__device__ __forceinline__ void mbar_wait_on(uint32_t bar, uint32_t parity, const Patience& p, uint32_t& leader) {
    for (uint32_t i = 0; !mbar_try(bar, parity); i++) {
        if (i < p.polls && ((i & 15u) != 15u || !*p.abort_flag)) continue;
        *p.abort_flag = 1u;
        leader = 0u;
        break;
    }
    __syncwarp();
}
__device__ __forceinline__ void mbar_wait_on(uint32_t bar, uint32_t parity, const Patience& p) {
    uint32_t unused = 0u;
    mbar_wait_on(bar, parity, p, unused);
}
// Whether a role of the block has given up, the same for all lanes: asked once a tile.
__device__ __forceinline__ bool gave_up(volatile uint32_t* abort_flag) { return __any_sync(0xFFFFFFFFu, *abort_flag != 0u); }
// PAIR: `bar` is a barrier of either CTA of a pair (a shared::cluster address); the copy's bytes count there.
template <bool PAIR = false>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
                     "r"(c0), "r"(c1), "r"(bar)
                     : "memory");
    else asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map),
                 "r"(c0), "r"(c1), "r"(bar)
                 : "memory");
}
template <bool PAIR = false>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
                     : "memory");
    else asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrives on a barrier -- a pair: on the same one of both CTAs -- when the MMAs issued so far have completed.
template <bool PAIR>
__device__ __forceinline__ void tc_commit(uint32_t leader, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
            "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(bar), "r"(leader),
            "h"((uint16_t)3)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
            "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader)
            : "memory");
}
// The same, on a barrier of this CTA only.
template <bool PAIR>
__device__ __forceinline__ void tc_commit_here(uint32_t leader, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
            "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(leader)
            : "memory");
    else tc_commit<false>(leader, bar);
}
// Arrival on a barrier of the other CTA of a pair, for tensor-memory accesses of this warp and nothing else: waited for (tcgen05.wait) and
// fenced (fence::before_thread_sync) they are ordered by a relaxed arrival, as the instruction set's own hand-over of tensor memory between
// threads is.  What lies in shared memory is not: see the stage barriers.  (A release at cluster scope holds the thread for about a microsecond.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// D[M x N] (+)= A[M x 64] . B[N x 64]^T, E2M1 operands, one E8M0 scale per 32 columns of either operand; M = 128, or 256 over the two
// CTAs of a pair (rows 0 .. 127 of A and D in the even one, each holding N / 2 rows of B).  Issued by the lanes whose `leader` is set (one
// of the warp), under a predicate and not a branch: see the MMA warp.
template <bool PAIR>
__device__ __forceinline__ void tc_mma_mxf4(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
            "setp.ne.b32 p, %7, 0;\n\t"
            "setp.ne.b32 q, %8, 0;\n\t"
            "mov.b64 da, {%1, %3};\n\t"
            "mov.b64 db, {%2, %3};\n\t"
            "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %4, [%5], [%6], p;\n\t}"
            ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(leader)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
            "setp.ne.b32 p, %7, 0;\n\t"
            "setp.ne.b32 q, %8, 0;\n\t"
            "mov.b64 da, {%1, %3};\n\t"
            "mov.b64 db, {%2, %3};\n\t"
            "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %4, [%5], [%6], p;\n\t}"
            ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(leader)
            : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// lane l of the warp writes N columns of its tensor-memory lane
__device__ __forceinline__ void tc_st(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
                 "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tc_st(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Scales of two landed stages, GROUPS groups of this lane's rows (row 32 j + lane of group i at src + i * kGroupBytes + j * 512, 16 bytes), to
// 16 * GROUPS columns of a slot: quarter k of the 512 columns (a scale-factor chunk) takes 4 columns a group, the groups side by side.
template <int GROUPS>
__device__ __forceinline__ void store_scales(const uint8_t* src, uint32_t dst) {
    uint32_t v[16 * GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint4 row = *reinterpret_cast<const uint4*>(src + i * kGroupBytes + j * 512);
            v[4 * i + j] = row.x;
            v[4 * GROUPS + 4 * i + j] = row.y;
            v[8 * GROUPS + 4 * i + j] = row.z;
            v[12 * GROUPS + 4 * i + j] = row.w;
        }
    tc_st(dst, v);
}
__device__ __forceinline__ uint32_t cluster_ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t saddr, uint32_t cta) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(cta));
    return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync_all() {
    __syncwarp();   // the .aligned forms want the warp together, whatever branch came before
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same where nothing written is read behind it: a release would wait for the stores of results, most of a microsecond.
__device__ __forceinline__ void cluster_sync_relaxed() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// K-major operand tile of 128-byte rows, 128-byte swizzle: 8-row groups of 1024 bytes.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);       // start address
    d |= (uint64_t)(1024u >> 4) << 32;              // stride between 8-row groups
    d |= (uint64_t)1 << 46;                         // descriptor version (sm_100)
    d |= (uint64_t)2 << 61;                         // 128-byte swizzle
    return d;
}
// kind::mxf4: E2M1 x E2M1 -> f32, E8M0 scales, K-major operands, K = 64; sf = byte (0 or 2) of the 4-byte scale words
// that holds this k step's first block.
__device__ __forceinline__ uint32_t mxf4_idesc(uint32_t m, int n, uint32_t sf) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | (sf << 4) | (sf << 29);
}

// Sixteen tokens of the lane's output column (32 neighbouring columns a warp).  16-bit results leave in pairs of columns where the rows
// allow 4-byte stores: even lanes take the even tokens of their own and the next lane's column, odd lanes the odd ones, so a store
// instruction carries two tokens.
template <typename T>
__device__ __forceinline__ void store_tokens(T* __restrict__ o, int64_t stride, const uint32_t (&v)[16], int rows, bool live, int pairs, int lane) {
    if constexpr (sizeof(T) == 2) {
        if (pairs) {   // N is even: both columns of a pair exist or neither does
            const bool odd = lane & 1;
            uint32_t* p = reinterpret_cast<uint32_t*>(o + (odd ? stride - 1 : 0));
            const int64_t step = stride;   // two rows, in 32-bit words
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float mine = __uint_as_float(odd ? v[j + 1] : v[j]), theirs = __uint_as_float(odd ? v[j] : v[j + 1]);
                const float got = __shfl_xor_sync(0xFFFFFFFFu, theirs, 1);
                const uint32_t w = odd ? pack2<T>(got, mine) : pack2<T>(mine, got);
                if (live && j + (odd ? 1 : 0) < rows) *p = w;
                p += step;
            }
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < 16; j++)
        if (live && j < rows) o[j * stride] = from_f32<T>(__uint_as_float(v[j]));
}

struct MatmulArgs {
    const uint8_t* w_scales;
    const uint8_t* a_scales;
    void* out;
    int64_t row_stride;
    int64_t M, N;
    int K;
    int tokens;              // tokens of a tile (multiple of 16)
    int fold;                // terms laid side by side in N (single CTAs; TERMS is 1 then), or 1
    int stages, stage_bytes; // ring of codes
    int slots;               // ring of scale slots in tensor memory, two stages each
    int scale_bufs;          // ring of scales, kGroupBytes a group
    int groups;              // 128-row groups of scales: 1 (W) + TERMS * ceil(tokens * fold / 128)
    int tmem_cols;
    int splits;              // CTAs of a cluster that share a tile's columns
    int tiles_w, tiles;      // tile t: W tile t % tiles_w, token tile t / tiles_w
    int scale_tma;           // rows of scales are 16-byte aligned: TMA brings them
    int pairs;               // results are 16-bit and pairs of columns 4-byte aligned in every row
    uint32_t polls;          // of a wait
};

// PAIR: clusters of two CTAs.  A pair takes 256 W rows, 128 each, and every MMA spans both; each CTA loads and holds half of the tile's A
// rows (and the scales of all of them).  The even CTA issues; the codes of both CTAs count on the even one's stage barriers -- so that the copies
// themselves make both halves visible to the MMAs, no thread passing the word on --, scales on their own CTA's, the scale warps of both report
// to the even one, commits arrive in both.  No load is broadcast.
template <int DT, int TERMS, bool PAIR>
__global__ void __launch_bounds__(kThreads, PAIR ? 1 : 2)
mxfp4_matmul_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_ws,
                    const __grid_constant__ CUtensorMap tmap_as, const MatmulArgs g) {
    using T = typename Elem<DT>::T;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ __align__(8) uint64_t s_bars[2 * kMaxStages + 4 + 2 * kMaxScaleBufs + 2 * kMaxSlots + 1];
    // tensor memory, abort flag; a pair: where the rings of stages (and how many loads that were) and slots have got to; the odd CTA's stages
    __shared__ uint32_t s_misc[10];
    const uint32_t sbase = smem_u32(smem), bar0 = smem_u32(s_bars);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // FULL[s]: the codes of the stage have landed (even CTA of a pair: in both; odd one: not used); EMPTY[s]: the MMAs that read it have completed;
    // ACC_FULL / ACC_EMPTY[b]: accumulator b is complete / read out; RAW_FULL / RAW_EMPTY[d]: two stages' scales have landed / are in tensor
    // memory; SLOT_FULL / SLOT_EMPTY[v]: and lie in slot v (a pair: of both CTAs) / the MMAs that used them have completed.
    constexpr int FULL = 0, EMPTY = FULL + kMaxStages, ACC_FULL = EMPTY + kMaxStages, ACC_EMPTY = ACC_FULL + 2, RAW_FULL = ACC_EMPTY + 2,
                  RAW_EMPTY = RAW_FULL + kMaxScaleBufs, SLOT_FULL = RAW_EMPTY + kMaxScaleBufs, SLOT_EMPTY = SLOT_FULL + kMaxSlots,
                  DRAIN = SLOT_EMPTY + kMaxSlots;   // DRAIN: all MMAs have completed
    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
    volatile uint32_t* abort_flag = s_misc + 1;
    const Patience patience{abort_flag, g.polls};
    if (threadIdx.x == 0) {
        for (int i = 0; i < kMaxStages; i++) {
            mbar_init(bar(FULL + i), 1);
            mbar_init(bar(EMPTY + i), 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(bar(ACC_FULL + b), 1);
            mbar_init(bar(ACC_EMPTY + b), PAIR ? 8 : 4);
        }
        for (int d = 0; d < kMaxScaleBufs; d++) {
            mbar_init(bar(RAW_FULL + d), g.scale_tma ? 1 : kLoaders);
            mbar_init(bar(RAW_EMPTY + d), 4);
        }
        for (int v = 0; v < kMaxSlots; v++) {
            mbar_init(bar(SLOT_FULL + v), PAIR ? 8 : 4);
            mbar_init(bar(SLOT_EMPTY + v), 1);
        }
        mbar_init(bar(DRAIN), 1);
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_a) : "memory");
    }
    if (warp == 1) {
        __syncwarp();
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_misc)), "r"(g.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(s_misc)), "r"(g.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)s_misc;
    if constexpr (PAIR) cluster_sync_relaxed();   // both CTAs' barriers exist before either signals the other
    pdl_wait();   // the operands may come from the kernel before this one

    const int half = PAIR ? (int)cluster_ctarank() : 0;   // of a pair
    const int rank = !PAIR && g.splits > 1 ? (int)cluster_ctarank() : 0;   // among the splits of a tile
    const int n_kc = (g.K + kStageK - 1) / kStageK;
    const int kc0 = (int)((int64_t)n_kc * rank / g.splits), kc1 = (int)((int64_t)n_kc * (rank + 1) / g.splits);
    const int per_tile = PAIR ? 2 : g.splits;               // CTAs
    const int tile0 = (int)blockIdx.x / per_tile, tile_step = (int)gridDim.x / per_tile;
    const int tokens = g.tokens, BN = tokens * g.fold, held = PAIR ? BN / 2 : BN;   // of a tile; N of its MMAs; rows of that in this CTA
    constexpr int kTileW = PAIR ? 2 * kWRows : kWRows;
    const uint32_t b_bytes = (uint32_t)(TERMS * held * kRowBytes);
    // scales behind the ring of codes: [buffer][W, term 0, ...][row][16]; a term's group has room for 128 rows behind the previous one's rows
    const uint32_t raw0 = (uint32_t)(g.stages * g.stage_bytes), raw_bytes = (uint32_t)(g.groups * kGroupBytes);
    const uint32_t group_step = BN > 128 ? (uint32_t)kGroupBytes : (uint32_t)BN * 16u;
    // scale slots behind the accumulators: W's 16 columns, then the terms' (nb == 2, one term: its two groups interleaved by quarter)
    const uint32_t slot0 = tmem + 2u * (uint32_t)BN, slot_cols = 16u * (uint32_t)g.groups;
    const int nb = (BN + 127) >> 7;

    if (warp == 0) {
        // -------------------------------------------------------------- producer
        if (lane == 0) {
            uint32_t s = 0, ph = 0, n_loads = 0;
            bool ok = true;
            const uint32_t full0 = PAIR ? map_to_cta(bar(FULL), 0u) : bar(FULL);
            for (int tile = tile0; tile < g.tiles && ok; tile += tile_step) {
                const int w0 = (tile % g.tiles_w) * kTileW + half * kWRows, a0 = (tile / g.tiles_w) * tokens + half * held;
                for (int kc = kc0; kc < kc1; kc++) {
                    ok = mbar_wait(bar(EMPTY) + 8u * s, ph ^ 1u, patience);
                    if (!ok) break;
                    const uint32_t dst = sbase + s * (uint32_t)g.stage_bytes, full = full0 + 8u * s;
                    // The even CTA of a pair announces both halves.  (The odd one's may land first: the barrier's phase cannot end before the
                    // announcement, and the odd CTA's next load of the stage waits for the MMAs of that phase.)
                    if (half == 0) mbar_expect_tx(bar(FULL) + 8u * s, (PAIR ? 2u : 1u) * (kWBytes + b_bytes));
                    tma_load_2d<PAIR>(dst, &tmap_w, kc * kRowBytes, w0, full);
                    tma_load_3d<PAIR>(dst + kWBytes, &tmap_a, kc * kRowBytes, a0, 0, full);
                    n_loads++;
                    if (++s == (uint32_t)g.stages) { s = 0; ph ^= 1u; }
                }
            }
            if constexpr (PAIR) {
                s_misc[2] = s;
                s_misc[3] = ph;
                s_misc[6] = n_loads;
            } else   // all copies have landed before this role ends, whoever gives up and when (a pair: see the end)
                for (uint32_t i = 0; i < (uint32_t)g.stages; i++)
                    for (uint32_t n = 0; n < kDrainPolls && !mbar_try(bar(FULL) + 8u * i, i < s ? ph : ph ^ 1u); n++) {}
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issue
        // The whole warp walks the loop and one lane issues, under a predicate: the instruction takes its operands from uniform registers, and
        // inside a branch of one lane each of them had to be carried there first -- 230 clocks an MMA, whatever its size, against 50.  This
        // warp bounds large products: a pair's stage takes it 580 clocks (four MMAs 200, a satisfied wait 80 each, a commit 35) with MMAs of
        // N = 208, which run 424, as of N = 16, with and without the copies and the scales.  Two warps that took turns were no faster.
        uint32_t leader = lane == 0 ? 1u : 0u;   // cleared for good when a wait runs out: no MMA and no commit from there on
        uint32_t s = 0, ph = 0, t = 0, v = 0, vph = 0;
        const uint64_t d0 = operand_desc(sbase);
        const uint32_t hi = (uint32_t)(d0 >> 32), lo0 = (uint32_t)d0;
        const uint32_t tm = __ballot_sync(0xFFFFFFFFu, (tmem >> lane) & 1u);   // tmem itself, as a value known to be uniform
        const uint32_t slots = tm + 2u * (uint32_t)BN;
        const uint32_t term_step = (uint32_t)(held * kRowBytes) >> 4, stage_step = (uint32_t)g.stage_bytes >> 4;
        const uint32_t quarter = nb == 2 ? 8u : 4u;   // columns of a quarter of A's scales
        const uint32_t idesc0 = mxf4_idesc(kTileW, BN, 0u), idesc2 = mxf4_idesc(kTileW, BN, 2u);
        for (int tile = tile0; tile < g.tiles && half == 0; tile += tile_step, t++) {
            if (gave_up(abort_flag)) break;
            const uint32_t b = t & 1u, acc = tm + b * (uint32_t)BN;
            uint32_t started = 0u;
            mbar_wait_on(bar(ACC_EMPTY) + 8u * b, ((t >> 1) & 1u) ^ 1u, patience, leader);
            tc_fence_after();
            // the MMAs of one stage, the slot's first or second half
            auto stage = [&](uint32_t at, int kc, int h) {
                const uint32_t a_lo = lo0 + at * stage_step, b_lo = a_lo + (kWBytes >> 4), sc = slots + v * slot_cols;
                auto step = [&](int ks) {
                    const uint32_t k = 2u * (uint32_t)h + (uint32_t)(ks >> 1);
#pragma unroll
                    for (int q = 0; q < TERMS; q++) {
                        tc_mma_mxf4<PAIR>(leader, acc, a_lo + 2u * ks, b_lo + (uint32_t)q * term_step + 2u * ks, hi, (ks & 1) ? idesc2 : idesc0, sc + 4u * k,
                                          sc + 16u + 16u * (uint32_t)q + quarter * k, ks == 0 && q == 0 ? started : 1u);
                    }
                };
                if ((kc + 1) * kStageK <= g.K) {
#pragma unroll
                    for (int ks = 0; ks < 4; ks++) step(ks);
                } else {   // the columns' end
                    const int steps = (g.K - kc * kStageK + 63) >> 6;
#pragma unroll
                    for (int ks = 0; ks < 4; ks++)
                        if (ks < steps) step(ks);
                }
                started = 1u;
            };
            for (int kc = kc0; kc < kc1;) {   // a slot of scales at a time: its waits first, then the MMAs of both stages
                mbar_wait_on(bar(SLOT_FULL) + 8u * v, vph, patience, leader);
                mbar_wait_on(bar(FULL) + 8u * s, ph, patience, leader);
                const uint32_t s0 = s;
                if (++s == (uint32_t)g.stages) { s = 0; ph ^= 1u; }
                if ((kc & 1) == 0 && kc + 1 < kc1) {
                    mbar_wait_on(bar(FULL) + 8u * s, ph, patience, leader);
                    tc_fence_after();
                    stage(s0, kc, 0);
                    tc_commit<PAIR>(leader, bar(EMPTY) + 8u * s0);
                    stage(s, kc + 1, 1);
                    tc_commit<PAIR>(leader, bar(EMPTY) + 8u * s);
                    if (++s == (uint32_t)g.stages) { s = 0; ph ^= 1u; }
                    kc += 2;
                } else {
                    tc_fence_after();
                    stage(s0, kc, kc & 1);
                    tc_commit<PAIR>(leader, bar(EMPTY) + 8u * s0);
                    kc++;
                }
                tc_commit<PAIR>(leader, bar(SLOT_EMPTY) + 8u * v);
                if (++v == (uint32_t)g.slots) { v = 0; vph ^= 1u; }
            }
            tc_commit<PAIR>(leader, bar(ACC_FULL) + 8u * b);
        }
        if (half == 0) {   // all MMAs have finished before this role ends, whoever gives up and when
            tc_commit_here<PAIR>(lane == 0 ? 1u : 0u, bar(DRAIN));
            for (uint32_t n = 0; n < kDrainPolls && !mbar_try(bar(DRAIN), 0u); n++) {}
        }
        __syncwarp();
    } else if (warp == 2) {
        // --------------------------------------------------------- TMA of scales
        if (lane == 0 && g.scale_tma) {
            uint32_t d = 0, ph = 0;
            bool ok = true;
            for (int tile = tile0; tile < g.tiles && ok; tile += tile_step) {
                const int w0 = (tile % g.tiles_w) * kTileW + half * kWRows, a0 = (tile / g.tiles_w) * tokens;
                for (int kc = kc0 & ~1; kc < kc1; kc += 2) {
                    ok = mbar_wait(bar(RAW_EMPTY) + 8u * d, ph ^ 1u, patience);
                    if (!ok) break;
                    const uint32_t dst = sbase + raw0 + d * raw_bytes, full = bar(RAW_FULL) + 8u * d;
                    mbar_expect_tx(full, kGroupBytes + (uint32_t)(TERMS * BN * 16));
                    tma_load_2d(dst, &tmap_ws, kc * 8, w0, full);
                    tma_load_3d(dst + kGroupBytes, &tmap_as, kc * 8, a0, 0, full);
                    if (++d == (uint32_t)g.scale_bufs) { d = 0; ph ^= 1u; }
                }
            }
            for (uint32_t i = 0; i < (uint32_t)g.scale_bufs; i++)
                for (uint32_t n = 0; n < kDrainPolls && !mbar_try(bar(RAW_FULL) + 8u * i, i < d ? ph : ph ^ 1u); n++) {}
        }
    } else if (warp == 3) {
        // idle: roles that use whole warp groups start on their boundaries
    } else if (warp >= kLoadWarp0 && !g.scale_tma) {
        // --------------------------------------------------------- scale loaders
        {
            const int r = threadIdx.x - kLoadWarp0 * 32;   // row of every group
            const int nblk = g.K >> 5;
            constexpr int kGroups = PAIR && TERMS == 3 ? 4 : 3;   // at most: W and a group a term, or two of one term
            uint32_t d = 0, ph = 0;
            bool ok = true;
            for (int tile = tile0; tile < g.tiles && ok; tile += tile_step) {
                const int64_t w_row = (int64_t)(tile % g.tiles_w) * kTileW + half * kWRows + r, a_row0 = (int64_t)(tile / g.tiles_w) * tokens;
                // this thread's row of every group, null where the operand has none
                const uint8_t* row[kGroups];
                bool place[kGroups];   // the group has room for it
                row[0] = w_row < g.N ? g.w_scales + w_row * nblk : nullptr;
                place[0] = true;
#pragma unroll
                for (int i = 1; i < kGroups; i++) {
                    const int rn = (TERMS == 1 ? (i - 1) * 128 : 0) + r;   // row of N; the term it belongs to and its token
                    const int q = TERMS == 1 ? rn / tokens : i - 1, ra = TERMS == 1 ? rn % tokens : rn;
                    place[i] = i < g.groups && rn < BN;
                    row[i] = place[i] && a_row0 + ra < g.M ? g.a_scales + ((int64_t)q * g.M + a_row0 + ra) * nblk : nullptr;
                }
                // A row is a stream of aligned 16-byte words, one a step -- an instruction that touches 32 lines takes as long for 4 bytes of each
                // as for 16 -- of which two hold the step's bytes; words without a byte of the row are not read.
                auto word = [&](const uint8_t* p, int i) {   // the word with byte 16 i of the row and those before it up to the boundary
                    const uintptr_t at = ((uintptr_t)p & ~(uintptr_t)15) + 16 * (uintptr_t)i;
                    return p && at < (uintptr_t)p + nblk ? __ldg(reinterpret_cast<const uint4*>(at)) : make_uint4(0, 0, 0, 0);
                };
                uint4 cur[kGroups], next[kGroups];
#pragma unroll
                for (int i = 0; i < kGroups; i++) {
                    cur[i] = word(row[i], kc0 >> 1);
                    next[i] = word(row[i], (kc0 >> 1) + 1);
                }
                for (int kc = kc0 & ~1; kc < kc1; kc += 2) {
                    ok = mbar_wait(bar(RAW_EMPTY) + 8u * d, ph ^ 1u, patience);
                    if (!ok) break;
                    const uint32_t dst = sbase + raw0 + d * raw_bytes + (uint32_t)r * 16u;
                    const int n = nblk - kc * 8;   // bytes past the row's end belong to the next row
#pragma unroll
                    for (int i = 0; i < kGroups; i++) {
                        if (i >= g.groups) break;
                        const uint32_t at = (uint32_t)(uintptr_t)row[i];
                        uint32_t v[8] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w, next[i].x, next[i].y, next[i].z, next[i].w};
#pragma unroll
                        for (int j = 0; j < 6; j++) v[j] = at & 8u ? v[j + 2] : v[j];
#pragma unroll
                        for (int j = 0; j < 5; j++) v[j] = at & 4u ? v[j + 1] : v[j];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            v[j] = __funnelshift_r(v[j], v[j + 1], at * 8u);   // takes it modulo 32
                            if (n < 4 * j + 4) v[j] = n > 4 * j ? v[j] & ((1u << (8 * (n - 4 * j))) - 1u) : 0u;
                        }
                        cur[i] = next[i];
                        next[i] = word(row[i], (kc >> 1) + 2);
                        if (place[i])
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (i ? kGroupBytes + (i - 1) * group_step : 0u)), "r"(v[0]), "r"(v[1]),
                                         "r"(v[2]), "r"(v[3])
                                         : "memory");
                    }
                    mbar_arrive(bar(RAW_FULL) + 8u * d);
                    if (++d == (uint32_t)g.scale_bufs) { d = 0; ph ^= 1u; }
                }
            }
        }
    } else if (warp >= kEpiWarp0 && warp < kLoadWarp0) {
        // -------------------------------------------------------------- epilogue
        const uint32_t q = (uint32_t)(warp & 3);
        uint32_t t = 0;
        for (int tile = tile0; tile < g.tiles && !gave_up(abort_flag); tile += tile_step, t++) {
            const int64_t n = (int64_t)(tile % g.tiles_w) * kTileW + half * kWRows + q * 32 + lane, m0 = (int64_t)(tile / g.tiles_w) * tokens;
            const uint32_t b = t & 1u, acc = tmem + b * (uint32_t)BN + ((q * 32u) << 16);
            mbar_wait_on(bar(ACC_FULL) + 8u * b, (t >> 1) & 1u, patience);
            tc_fence_after();
            const int rows = (int)min((int64_t)tokens, g.M - m0);     // tokens that exist
            T* o = reinterpret_cast<T*>(g.out) + m0 * g.row_stride + n;
            for (int c0 = 0; c0 < tokens; c0 += 16) {
                uint32_t v[16];
                __syncwarp();   // stores above may have parted the lanes
                tc_ld16(acc + (uint32_t)c0, v);
                tc_wait_ld();
                if constexpr (!PAIR)
                    for (int f = 1; f < g.fold; f++) {   // the token's further terms
                        uint32_t more[16];
                        tc_ld16(acc + (uint32_t)(f * tokens + c0), more);
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(more[j]));
                    }
                if (!PAIR && g.splits > 1) {   // the partial tile, token-major, in the ring's memory (every stage has been consumed)
                    float* p = reinterpret_cast<float*>(smem) + (size_t)c0 * kWRows + q * 32 + lane;
#pragma unroll
                    for (int j = 0; j < 16; j++) p[j * kWRows] = __uint_as_float(v[j]);
                } else {
                    store_tokens<T>(o, g.row_stride, v, rows - c0, n < g.N, g.pairs, lane);
                    o += 16 * g.row_stride;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && tile + 2 * tile_step < g.tiles) {   // only where it is waited for: nothing may be on its way to a block that has ended
                if (PAIR && half != 0) mbar_arrive_cluster(map_to_cta(bar(ACC_EMPTY) + 8u * b, 0u));
                else mbar_arrive(bar(ACC_EMPTY) + 8u * b);
            }
        }
    } else {
        // ----------------------------------------------------------- scale warps
        // The tensor core wants, in every lane quarter, lane l's column j of a scale-factor chunk to hold the chunk's four bytes of row 32 j + l.
        const uint32_t q = (uint32_t)(warp & 3);
        const uint32_t set = warp >= kLoadWarp0 ? 1u : 0u, sets = g.scale_tma ? 2u : 1u;
        uint32_t u = 0, d = 0, dph = 0, v = 0, vph = 0;   // buffers so far; ring positions
        for (int tile = tile0; tile < g.tiles && !gave_up(abort_flag); tile += tile_step)
            for (int kc = kc0; kc < kc1; kc = (kc | 1) + 1, u++) {
                if (sets == 1u || (u & 1u) == set) {
                    mbar_wait_on(bar(RAW_FULL) + 8u * d, dph, patience);
                    mbar_wait_on(bar(SLOT_EMPTY) + 8u * v, vph ^ 1u, patience);
                    tc_fence_after();
                    const uint8_t* src = smem + raw0 + d * raw_bytes + lane * 16;
                    const uint32_t dst = slot0 + v * slot_cols + ((q * 32u) << 16);
                    store_scales<1>(src, dst);
                    if (TERMS == 1 && nb == 2) store_scales<2>(src + kGroupBytes, dst + 16u);
                    else {
#pragma unroll 1
                        for (int i = 0; i < TERMS; i++) store_scales<1>(src + kGroupBytes + i * group_step, dst + 16u + 16u * (uint32_t)i);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(bar(RAW_EMPTY) + 8u * d);
                        if (PAIR && half != 0) mbar_arrive_cluster(map_to_cta(bar(SLOT_FULL) + 8u * v, 0u));
                        else mbar_arrive(bar(SLOT_FULL) + 8u * v);
                    }
                }
                if (++d == (uint32_t)g.scale_bufs) { d = 0; dph ^= 1u; }
                if (++v == (uint32_t)g.slots) { v = 0; vph ^= 1u; }
            }
        if (PAIR && warp == 4 && lane == 0) {
            s_misc[4] = v;
            s_misc[5] = vph;
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) {
        // Neither CTA's shared or tensor memory goes away while the other may still use it: nor while an arrival is on its way to it.  The last
        // releases of stages and slots, which no role waited for, are waited for here (everything else on them has happened by now).
        const uint32_t other = (uint32_t)half ^ 1u;
        if (warp == 0 && !gave_up(abort_flag)) {   // a lane a barrier
            const bool slot = lane >= 16;
            const uint32_t n = (uint32_t)(slot ? g.slots : g.stages), i = (uint32_t)lane & 15u, next = s_misc[slot ? 4 : 2] + i;
            if (i < n) mbar_wait(bar(slot ? SLOT_EMPTY : EMPTY) + 8u * (next < n ? next : next - n), s_misc[slot ? 5 : 3] ^ (next < n ? 1u : 0u), patience);
        }
        if (warp == 0) {
            __syncwarp();
            if (gave_up(abort_flag) && lane == 0) {   // the other CTA hears of it
                st_cluster(map_to_cta(smem_u32(s_misc + 1), other), 1u);
                __threadfence();
            }
        }
        cluster_sync_relaxed();
        if (*abort_flag) {   // from here on the same in both
            // Copies may be in flight, on the even CTA's barriers.  It gets to know how far the odd one came, and makes up for what a stage that
            // only one of them has asked for still lacks, so that the stage's phase ends when the copies that were made have landed.  (Neither
            // can be further ahead than the ring is long: nothing was released by the MMA warp since its first wait ran out.)
            if (threadIdx.x == 0 && half != 0) {
                for (uint32_t i = 0; i < 2; i++) st_cluster(map_to_cta(smem_u32(s_misc + 7 + i), 0u), s_misc[2 + i]);
                st_cluster(map_to_cta(smem_u32(s_misc + 9), 0u), s_misc[6]);
            }
            cluster_sync_all();
            if (threadIdx.x == 0 && half == 0) {
                const int ahead = (int)(s_misc[6] - s_misc[9]);   // loads this CTA asked for and the odd one did not
                uint32_t s = s_misc[ahead >= 0 ? 2 : 7], ph = s_misc[ahead >= 0 ? 3 : 8];
                for (int i = 1; i <= g.stages; i++) {   // back from the last load
                    if (s == 0) { s = (uint32_t)g.stages; ph ^= 1u; }
                    const uint32_t full = bar(FULL) + 8u * --s;
                    if (i <= ahead) mbar_complete_tx(full, kWBytes + b_bytes);
                    else if (i <= -ahead) mbar_expect_tx(full, kWBytes + b_bytes);
                    for (uint32_t n = 0; n < kDrainPolls && !mbar_try(full, ph); n++) {}
                }
            }
            cluster_sync_all();
        }
    }
    if (threadIdx.x == 0 && *abort_flag) atomicOr(&g_head_error, 1u);
    if (!PAIR && g.splits > 1) {
        cluster_sync_all();
        // CTA `rank` adds the tokens rank, rank + splits, ... of all partial tiles, in rank order
        const int64_t w0 = (int64_t)(tile0 % g.tiles_w) * kWRows, m0 = (int64_t)(tile0 / g.tiles_w) * tokens;
        // (a warp a token, four columns a lane; the parts are requested together)
        for (int c = rank + g.splits * warp; c < tokens && m0 + c < g.M; c += g.splits * (kThreads / 32)) {
            const uint32_t at = sbase + (uint32_t)(c * kWRows + lane * 4) * 4u;
            float4 part[8], sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int p = 0; p < 8; p++)
                if (p < g.splits) part[p] = ld_cluster_f32x4(map_to_cta(at, (uint32_t)p));
#pragma unroll
            for (int p = 0; p < 8; p++)
                if (p < g.splits) {
                    sum.x += part[p].x;
                    sum.y += part[p].y;
                    sum.z += part[p].z;
                    sum.w += part[p].w;
                }
            const int64_t n = w0 + lane * 4;
            T* o = reinterpret_cast<T*>(g.out) + (m0 + c) * g.row_stride + n;
            if (n < g.N) o[0] = from_f32<T>(sum.x);
            if (n + 1 < g.N) o[1] = from_f32<T>(sum.y);
            if (n + 2 < g.N) o[2] = from_f32<T>(sum.z);
            if (n + 3 < g.N) o[3] = from_f32<T>(sum.w);
        }
        cluster_sync_relaxed();   // nobody's shared memory goes away while another CTA reads it (what it read has gone into its stores)
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_cols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_cols) : "memory");
    }
}

// Two sizes of block, so that tensor memory is never over-committed by blocks of this kernel that share an SM (a cluster whose
// blocks wait for tensor memory held by another such cluster could wait for ever): at most 112 KB of shared memory and 256
// columns (two blocks an SM, a third does not fit beside 77 KB or more), or at least 160 KB (alone on its SM).  Nor does either fit beside the
// layer's own kernel of CTA pairs (225 KB); the layer's single-CTA kernels wait for no other block, so they give their columns back.
constexpr int kSmallMin = 77 * 1024, kSmallMax = 112 * 1024, kLargeMin = 160 * 1024, kLargeMax = 225 * 1024;

struct Plan {
    int tokens, fold, stages, slots, stage_bytes, scale_bufs, groups, tmem_cols, smem, per_sm, splits, tiles_w, tiles_m, at_once;
    bool pair;
};

bool plan_block(int terms, int tokens, bool pair, Plan* p) {
    p->tokens = tokens;
    p->pair = pair;
    p->fold = pair ? 1 : terms;
    const int n = tokens * p->fold;
    if (n > kMaxN || (pair && terms > 1 && n > 128)) return false;   // a pair's terms have one group of scales each
    const int groups = 1 + (pair ? terms : 1) * ((n + 127) / 128);
    p->groups = groups;
    p->stage_bytes = kWBytes + terms * (pair ? tokens / 2 : tokens) * kRowBytes;
    auto pow2 = [](int c) { int r = 32; while (r < c) r *= 2; return r; };
    // stages and scale slots that fit behind `bufs` buffers of scales into `smem` bytes and `cols` columns
    auto fit = [&](int smem, int bufs, int cols, int per_sm) {
        p->stages = std::min(kMaxStages, (smem - 1024 - bufs * groups * kGroupBytes) / p->stage_bytes);
        p->slots = std::min(kMaxSlots, (cols - 2 * n) / (16 * groups));
        p->scale_bufs = bufs;
        p->per_sm = per_sm;
        return p->stages >= (per_sm == 2 ? 3 : 2) && p->slots >= 2;
    };
    // An even number of buffers of scales, so that each belongs to one of the two sets of scale warps: a set that shared a buffer with the other
    // could ask for a phase of its barrier whose predecessor had not completed yet, and a parity wait lets that pass.  (Slots: the set that
    // comes to a slot has waited for one that the tensor core finished behind the slot's last use but one.)  Four only where a ring of that
    // length is to be fed.
    if (!(!pair && fit(kSmallMax, 2, 256, 2)) && !(fit(kLargeMax, 4, 512, 1) && p->stages > 4) && !fit(kLargeMax, 2, 512, 1)) return false;
    p->smem = std::max(p->per_sm == 2 ? kSmallMin : kLargeMin, p->stages * p->stage_bytes + p->scale_bufs * groups * kGroupBytes + 1024);
    p->tmem_cols = pow2(2 * n + p->slots * 16 * groups);
    return p->stages * p->stage_bytes >= tokens * kWRows * 4;   // a partial tile fits into the ring
}

// What a device runs at once: clusters of 1, 2, 4 and 8 CTAs with an SM each (clusters do not reach across the groups that SMs come in, so there
// are fewer than SMs suggest: 148, 74, 33, 15; on a partition of a device there may be none); of small blocks, at least twice as many.  Looked
// up, and the opt-in to large shared memory made, once per device.
struct Device {
    int sms;
    int clusters[4];   // [log2 of the size]
};

// A tiling set by dsx_mxfp4_matmul_pin: -1 and 0 leave a part to the model.
struct Pin {
    int8_t pair = -1;
    uint8_t tokens = 0, splits = 0, unused = 0;
};
std::atomic<Pin> g_pin{Pin{}};
std::atomic<uint32_t> g_polls{kPolls};

// Tokens a tile, pairs or single CTAs, and splits of the columns, from a model of the time in clocks.  A stage takes its MMAs on the tensor
// core (N / 2 clocks each, 50 at least), or the issuing warp's 50 an MMA and what surrounds them (two blocks on an SM issue side by side), or
// its copies at 80 bytes a clock and SM from L2; a round of tiles about 5500 clocks before and after its stages, a joined tile another 2500;
// and the operands come from HBM at 26 bytes a clock and SM.  The constants were fitted to 600 tilings of 40 products, of 1 to 8192 tokens and 3
// to 131072 rows of W: the model's choice is 0.5 % slower than the best of them on average, 16 % at worst (3176 x 3 x 3104).
bool make_plan(int64_t M, int64_t N, int K, int terms, const Device& dev, const Pin& pin, Plan* best) {
    const int n_kc = (K + kStageK - 1) / kStageK;
    double best_t = 1e300;
    for (int pair = 0; pair <= 1; pair++)
        for (int tokens = 16; tokens <= kMaxN && (tokens < M + 16 || tokens == pin.tokens); tokens += 16) {
            Plan p;
            if ((pin.pair >= 0 && pair != pin.pair) || (pin.tokens > 0 && tokens != pin.tokens)) continue;
            if (!plan_block(terms, tokens, pair != 0, &p)) continue;
            p.tiles_w = (int)((N + kWRows * (1 + pair) - 1) / (kWRows * (1 + pair)));
            p.tiles_m = (int)((M + tokens - 1) / tokens);
            const int64_t tiles = (int64_t)p.tiles_w * p.tiles_m;
            const double mmas = 4.0 * (pair ? terms : 1), tensor = mmas * std::max(50.0, tokens * p.fold / 2.0);
            const double issue = pair ? 50.0 * mmas + 250.0 : p.per_sm == 1 ? 50.0 * mmas + 300.0 : (50.0 * mmas + 700.0) / 2;
            const double stage = std::max({tensor, issue, p.stage_bytes / 80.0});
            const double hbm = ((double)N + (double)terms * M) * K * 17 / 32 / (26.0 * dev.sms);
            for (int l = 0; l <= (pair ? 0 : 3) && 1 << l <= n_kc; l++) {
                if (pin.splits > 0 && 1 << l != pin.splits) continue;
                p.at_once = p.per_sm * dev.clusters[l + pair];   // tiles
                if (p.at_once == 0 || (l > 0 && tiles > p.at_once)) break;
                const int64_t rounds = (tiles + p.at_once - 1) / p.at_once;
                const int64_t busiest = (tiles * p.per_sm + p.at_once - 1) / p.at_once;   // tiles an SM
                const double t = std::max((double)busiest * ((n_kc + (1 << l) - 1) >> l) * stage, hbm) + 5500.0 * rounds + (l > 0 ? 2500.0 + 2.0 * tokens : 0.0) +
                                 45.0 * tokens;
                if (t < best_t) {
                    best_t = t;
                    p.splits = 1 << l;
                    *best = p;
                }
            }
        }
    return best_t < 1e300;
}

template <int DT, int TERMS, bool PAIR>
int launch(const Plan& p, const CUtensorMap (&maps)[4], const MatmulArgs& g, cudaStream_t stream) {
    const int cluster = PAIR ? 2 : p.splits;
    const int64_t tiles = (int64_t)p.tiles_w * p.tiles_m;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(cluster * std::min<int64_t>(tiles, p.at_once)));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)p.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    DSX_CUDA(cudaLaunchKernelEx(&cfg, mxfp4_matmul_kernel<DT, TERMS, PAIR>, maps[0], maps[1], maps[2], maps[3], g));
    DSX_LAUNCHED();
    return DSX_OK;
}

template <int DT>
int launch_for(int terms, const Plan& p, const CUtensorMap (&maps)[4], const MatmulArgs& g, cudaStream_t stream) {
    if (!p.pair) return launch<DT, 1, false>(p, maps, g, stream);
    if (terms == 1) return launch<DT, 1, true>(p, maps, g, stream);
    if (terms == 2) return launch<DT, 2, true>(p, maps, g, stream);
    return launch<DT, 3, true>(p, maps, g, stream);
}

template <int DT>
int allow_shared() {
    DSX_CUDA(cudaFuncSetAttribute(mxfp4_matmul_kernel<DT, 1, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLargeMax));
    DSX_CUDA(cudaFuncSetAttribute(mxfp4_matmul_kernel<DT, 1, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLargeMax));
    DSX_CUDA(cudaFuncSetAttribute(mxfp4_matmul_kernel<DT, 2, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLargeMax));
    DSX_CUDA(cudaFuncSetAttribute(mxfp4_matmul_kernel<DT, 3, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLargeMax));
    return DSX_OK;
}

template <bool PAIR>
int max_clusters(int log2_size) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(8);
    lc.blockDim = dim3(kThreads);
    lc.dynamicSmemBytes = kLargeMax;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1u << log2_size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, mxfp4_matmul_kernel<DSX_F32, 1, PAIR>, &lc) != cudaSuccess) {
        (void)cudaGetLastError();
        return 0;
    }
    return n;
}
int configure(const Device** out) {
    constexpr int kMaxDevices = 64;
    static Device devices[kMaxDevices];
    static std::atomic<int> known[kMaxDevices];
    static std::mutex mutex;
    int dev = 0;
    DSX_CUDA(cudaGetDevice(&dev));
    DSX_REQUIRE(dev >= 0 && dev < kMaxDevices, "mxfp4_matmul: device index %d out of range", dev);
    *out = &devices[dev];
    if (known[dev].load(std::memory_order_acquire)) return DSX_OK;
    std::lock_guard<std::mutex> lock(mutex);
    if (known[dev].load(std::memory_order_relaxed)) return DSX_OK;   // by a thread that held the lock before: others may be reading it
    Device& d = devices[dev];
    DSX_CUDA(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev));
    if (int rc = allow_shared<DSX_F32>()) return rc;
    if (int rc = allow_shared<DSX_BF16>()) return rc;
    if (int rc = allow_shared<DSX_F16>()) return rc;
    d.clusters[0] = d.sms;
    for (int l = 1; l < 4; l++) d.clusters[l] = max_clusters<false>(l);
    d.clusters[1] = std::min(d.clusters[1], max_clusters<true>(1));
    known[dev].store(1, std::memory_order_release);
    return DSX_OK;
}

}  // namespace
}  // namespace dsx

using namespace dsx;

namespace {
// Sizes that make_plan takes.  2^24 columns: the longest a wait lasts (a tile's MMAs, 20 ms) stays far inside its limit (about ten seconds).
int check_sizes(int n_terms, int64_t m, int64_t n, int64_t k) {
    DSX_REQUIRE(m >= 0 && n >= 0 && k >= 32 && k % 32 == 0 && m < ((int64_t)1 << 22) && n < ((int64_t)1 << 31) && k <= ((int64_t)1 << 24),
                "mxfp4_matmul: %lld x %lld x %lld (k a multiple of 32, at most 2^24; m below 2^22)", (long long)m, (long long)n, (long long)k);
    DSX_REQUIRE(n_terms >= 1 && n_terms <= 3, "mxfp4_matmul: %d terms (1 to 3)", n_terms);
    return DSX_OK;
}
int choose_plan(int n_terms, int64_t m, int64_t n, int64_t k, Plan* p) {
    const Device* dev = nullptr;
    if (int rc = configure(&dev)) return rc;
    if (!make_plan(m, n, (int)k, n_terms, *dev, g_pin.load(std::memory_order_relaxed), p))
        return set_error(DSX_ERR_UNSUPPORTED, "mxfp4_matmul: no tiling for %d terms (or not the pinned one)", n_terms);
    DSX_REQUIRE((int64_t)p->tiles_w * p->tiles_m < ((int64_t)1 << 30), "mxfp4_matmul: too many tiles");
    return DSX_OK;
}
}  // namespace

extern "C" {

int dsx_mxfp4_matmul_tiling(int n_terms, int64_t m, int64_t n, int64_t k, int32_t* tiling) {
    if (int rc = check_sizes(n_terms, m, n, k)) return rc;
    DSX_REQUIRE(m > 0 && n > 0 && tiling, "mxfp4_matmul_tiling: nothing to multiply, or a null argument");
    Plan p;
    if (int rc = choose_plan(n_terms, m, n, k, &p)) return rc;
    const int32_t values[8] = {p.pair, p.tokens, p.splits, p.tiles_w * p.tiles_m, p.at_once, p.stages, p.scale_bufs, p.slots};
    std::copy(values, values + 8, tiling);
    return DSX_OK;
}

int dsx_mxfp4_matmul_pin(int pair, int tokens, int splits) {
    DSX_REQUIRE(pair >= -1 && pair <= 1 && tokens >= 0 && tokens <= kMaxN && tokens % 16 == 0 && splits >= 0 && splits <= 8 && (splits & (splits - 1)) == 0,
                "mxfp4_matmul_pin: pair %d (-1 to 1), %d tokens (a multiple of 16, at most 208), %d splits (0, 1, 2, 4, 8)", pair, tokens, splits);
    Pin pin;
    pin.pair = (int8_t)pair;
    pin.tokens = (uint8_t)tokens;
    pin.splits = (uint8_t)splits;
    g_pin.store(pin, std::memory_order_relaxed);
    return DSX_OK;
}

int dsx_mxfp4_matmul_set_polls(uint32_t polls) {
    g_polls.store(polls ? polls : kPolls, std::memory_order_relaxed);
    return DSX_OK;
}

int dsx_mxfp4_matmul(const void* a_codes, const void* a_scales, int n_terms, int64_t m, const void* w_codes, const void* w_scales, int64_t n,
                     int64_t k, void* out, int dtype, int64_t row_stride, dsx_stream_t stream) {
    DSX_REQUIRE(dtype_ok(dtype), "mxfp4_matmul: unknown element type %d", dtype);
    if (int rc = check_sizes(n_terms, m, n, k)) return rc;
    if (m == 0 || n == 0) return DSX_OK;
    DSX_REQUIRE(a_codes && a_scales && w_codes && w_scales && out, "mxfp4_matmul: null argument");
    DSX_REQUIRE(row_stride >= n || m == 1, "mxfp4_matmul: row stride %lld below the %lld columns of a row", (long long)row_stride, (long long)n);
    DSX_REQUIRE((((uintptr_t)a_codes | (uintptr_t)w_codes) & 15) == 0 && ((uintptr_t)out & (dtype_size(dtype) - 1)) == 0,
                "mxfp4_matmul: codes must be 16-byte aligned, out aligned to its elements");
    Plan p;
    if (int rc = choose_plan(n_terms, m, n, k, &p)) return rc;
    // codes and scales of both operands as (bytes, row) and (bytes, row, term); the maps of scales only where TMA can read them
    const bool scale_tma = k % 512 == 0 && (((uintptr_t)a_scales | (uintptr_t)w_scales) & 15) == 0;
    CUtensorMap maps[4];
    auto encode_w = [&](CUtensorMap* map, const void* base, int64_t row_bytes, int box_bytes, CUtensorMapSwizzle swizzle) {
        const cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)n};
        const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
        const cuuint32_t box[2] = {(cuuint32_t)box_bytes, (cuuint32_t)kWRows};
        return tmap_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, swizzle);
    };
    auto encode_a = [&](CUtensorMap* map, const void* base, int64_t row_bytes, int box_bytes, int box_rows, CUtensorMapSwizzle swizzle) {
        const cuuint64_t dims[3] = {(cuuint64_t)row_bytes, (cuuint64_t)m, (cuuint64_t)n_terms};
        const cuuint64_t strides[2] = {(cuuint64_t)row_bytes, (cuuint64_t)(m * row_bytes)};
        const cuuint32_t box[3] = {(cuuint32_t)box_bytes, (cuuint32_t)box_rows, (cuuint32_t)n_terms};
        return tmap_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box, swizzle);
    };
    if (int rc = encode_w(&maps[0], w_codes, k / 2, kRowBytes, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    if (int rc = encode_a(&maps[1], a_codes, k / 2, kRowBytes, p.pair ? p.tokens / 2 : p.tokens, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    maps[2] = maps[0];
    maps[3] = maps[1];
    if (scale_tma) {
        if (int rc = encode_w(&maps[2], w_scales, k / 32, 16, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
        if (int rc = encode_a(&maps[3], a_scales, k / 32, 16, p.tokens, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
    }
    MatmulArgs g{};
    g.w_scales = (const uint8_t*)w_scales;
    g.a_scales = (const uint8_t*)a_scales;
    g.out = out;
    g.row_stride = row_stride;
    g.M = m; g.N = n; g.K = (int)k;
    g.tokens = p.tokens; g.fold = p.fold; g.stages = p.stages; g.slots = p.slots; g.stage_bytes = p.stage_bytes; g.groups = p.groups; g.tmem_cols = p.tmem_cols; g.splits = p.splits;
    g.tiles_w = p.tiles_w; g.tiles = p.tiles_w * p.tiles_m;
    g.scale_tma = scale_tma;
    g.scale_bufs = p.scale_bufs;
    g.polls = g_polls.load(std::memory_order_relaxed);
    g.pairs = dtype != DSX_F32 && n % 2 == 0 && (row_stride % 2 == 0 || m == 1) && ((uintptr_t)out & 3) == 0;
    const cudaStream_t s = (cudaStream_t)stream;
    if (dtype == DSX_F32) return launch_for<DSX_F32>(n_terms, p, maps, g, s);
    if (dtype == DSX_BF16) return launch_for<DSX_BF16>(n_terms, p, maps, g, s);
    return launch_for<DSX_F16>(n_terms, p, maps, g, s);
}

int dsx_head_check(dsx_stream_t stream_, uint32_t* error_word) {
    cudaStream_t stream = (cudaStream_t)stream_;
    uint32_t w = 0;
    DSX_CUDA(cudaMemcpyFromSymbolAsync(&w, g_head_error, 4, 0, cudaMemcpyDeviceToHost, stream));
    DSX_CUDA(cudaStreamSynchronize(stream));
    if (w) {
        const uint32_t zero = 0;
        DSX_CUDA(cudaMemcpyToSymbolAsync(g_head_error, &zero, 4, 0, cudaMemcpyHostToDevice, stream));
        DSX_CUDA(cudaStreamSynchronize(stream));
    }
    if (error_word) *error_word = w;
    if (w) return set_error(DSX_ERR_DEVICE, "the MXFP4 product reported error word 0x%x (a bounded wait ran out)", w);
    return DSX_OK;
}

}  // extern "C"
