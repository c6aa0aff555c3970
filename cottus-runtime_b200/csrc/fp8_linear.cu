// Block-scaled e4m3 matrix product on the 5th-generation tensor cores:
//
//   out[m][n] = sum_b sx[b][m] sw[n/128][b] D_b[m][n]  (+ residual[m][n]),
//   D_b[m][n] = sum_{k in group b} x[m][k] w[n][k],  groups of 128 along k.
//
// Replaces gemmCUDA (cuBLAS SGEMM, compute_primitives_cuda.cu:30-55) and the
// residualAddCUDA that follows the O-projection.
//
// The scales differ from group to group, so a group's 128-deep product is
// accumulated in tensor memory (four tcgen05.mma of kind::f8f6f4, K = 32
// each) and then added, scaled, to fp32 sums in registers.  Per CTA:
//
//   warps 0-7   the sums: warp w reads TMEM lanes 32 (w mod 4) .. + 31, and
//               half (w / 4) of the product's columns
//   warp 8      TMA producer (one thread): ring of stages, one group per stage
//   warp 9      TMEM allocation and MMA issue (one thread)
//   warps 10-11 scales: bring each group's row and weight scales to a ring of
//               their own, kScaleBatch groups at once and kScaleSlots batches
//               ahead (read by the sums themselves, one group ahead, a group
//               took an L2 round trip; so it did with one 4-byte cp.async and
//               one asynchronous arrival per group)
//
// TMEM holds two to four product buffers, so the tensor cores work on one
// group while another is being added up.
//
// Up to 16 rows of x by a small weight go to fp8_linear_thin_kernel, which
// takes the weight straight to registers: without barriers, tensor memory and
// clusters to set up, one row by 2048 x 2048 takes 2.4 us against 4.5.
//
// Two tiles:
//   narrow  128 rows of the weight (TMEM lanes) by XR = 16, 32, 64 or 128 rows
//           of x (columns), one CTA.  A decode batch reads the weight once and
//           is bound by HBM or latency; the multiplies are as many as the
//           batch needs (with the rows of x as lanes, 128 whatever the batch,
//           a 37-row product over a 128256-row weight held the GPU at its
//           power limit, 1.4 GHz).  Where the weight has fewer tiles than the
//           GPU has SMs, `splits` CTAs of one cluster share a tile: each takes
//           a contiguous run of groups and sends its sums to the CTA that adds
//           them (distributed shared memory, every CTA a share of the weight's
//           rows), in rank order, so a result does not depend on timing.
//   wide    256 x 256 by a pair of CTAs (cta_group::2): each holds 128 rows of
//           x and of the weight, and the pair's MMA reads both halves, so an
//           SM moves 32 KB per 128 x 256 x 128 multiplies.  With the same
//           128 x 256 per SM as one CTA (48 KB) shared memory was the limit,
//           reads by the MMA and writes by TMA together: 1270 cycles a group
//           against the 512 of the multiplies.  Here a row of x is a lane, and
//           a thread's scale one number for its 128 columns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <string>

#include "common.cuh"
#include "cottus_b200.h"
#include "internal.h"
#include "lowp.cuh"
#include "per_device.h"

namespace cb200 {
CUtensorMap make_tensor_map_2d_u8(const void* base, uint64_t inner, uint64_t outer, uint64_t pitch_bytes,
                                  uint32_t box_inner, uint32_t box_outer, bool swizzle128, cudaError_t* err);
int device_sm_count(int device);

namespace {

constexpr int kBM = 128;        // rows of x per CTA
constexpr int kBK = 128;        // elements (bytes) of k per stage: one scale group
constexpr int kWRows = 128;     // rows of the weight per CTA and stage
constexpr int kSumWarps = 8;    // warps that add up the groups
constexpr int kThreads = (kSumWarps + 4) * 32;  // and one warpgroup for the producer, the MMA issue and the scales
// Registers per thread of the wide tile after the launch's even split: the
// sums (128 per thread) take what the other warpgroup gives back.  The launch
// must have brought that many (checked on the host).
constexpr int kSumRegs = 224, kCtrlRegs = 56;
constexpr int kMinLaunchRegs = (kSumRegs * kSumWarps * 32 + kCtrlRegs * 128 + kThreads - 1) / kThreads;
constexpr int kMaxStages = 12;
constexpr int kMaxSplits = 8;   // portable cluster size
constexpr int kMaxBufs = 4;     // product buffers in TMEM
constexpr int kStagePitch = 20; // words per staged row of 16 columns (conflict-free 16-byte accesses)
constexpr int kScaleSlots = 3;  // of kScaleBatch groups each
constexpr int kScaleBatch = 4;
constexpr int kPrefetch = 4;   // groups whose weights are prefetched into L2
constexpr int kScaleWords = kBM + 4;  // a group's scales: 128 rows, then one per 128 columns of the tile
constexpr size_t kSmemMax = 232448;   // dynamic shared memory per CTA, 227 KB
constexpr size_t kSplitSmem = 115712;  // half of an SM's, 113 KB: at least this for splits
constexpr int kWarpStaging = 32 * 128;  // per sum warp: 128 bytes of each of its rows (or 16 padded columns)
// scales, barriers and words behind the ring and the staging area
constexpr size_t kTailBytes =
    (size_t)kScaleSlots * kScaleBatch * kScaleWords * 4 + (2 * kMaxStages + 2 * kMaxBufs + 2 * kScaleSlots + 1) * 8 + 16 + 32 * 4;

struct LinArgs {
    const float* xs;
    const float* ws;
    const float* residual;
    void* out;
    uint32_t* status;
    int M, N, groups, n_blocks, m_tiles, n_tiles, splits, stages, out_dtype;
    int staging_bytes;
    int tma_out;  // whole 128-byte pieces of out may be stored by TMA
    int vec;  // rows of out and residual start on 16 bytes and hold whole runs of 4
};

__device__ __forceinline__ uint64_t sw128_kmajor_desc(uint32_t smem_byte_addr) {
    // K-major tile of 128-byte rows, 128B swizzle, 8-row groups 1024 bytes apart
    return (uint64_t)((smem_byte_addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f8f6f4: e4m3 A and B (format 0), fp32 accumulator, both K-major.
template <int M, int N>
constexpr uint32_t f8_idesc() {  // M lanes, N columns
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Arrival on `bar` (of both CTAs of a pair) once this thread's multiplies so far are done.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::
                         "r"(bar), "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                     : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
            : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    if constexpr (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
// 8 or 16 columns of this warp's 32 lanes, waited for.
__device__ __forceinline__ void tmem_get8(uint32_t addr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_get16(uint32_t addr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(addr)
        : "memory");
}
// 32 columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
// Waits for this warp's TMEM loads; v passes through, so that no use of it is
// scheduled before the wait (30 operands are the most an asm statement takes).
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile(""
                     : "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]),
                       "+r"(v[i + 6]), "+r"(v[i + 7]));
}

// 2-D tiled TMA store from this CTA's shared memory, in the thread's bulk group.
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(c0), "r"(c1), "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// The thread's stores have read their shared memory / are complete.
__device__ __forceinline__ void tma_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Address of CTA `rank`'s copy of a shared-memory address.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t local, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
    return a;
}
__device__ __forceinline__ void st_cluster_f(uint32_t a, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t a, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void st_shared_u4(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Barrier operations on 32-bit shared-memory addresses (64-bit pointers cost
// the sums registers that they need for their accumulators).
// (the thread may sleep up to a millisecond in each try, so that waiting warps
// leave the issue slots to the sums)
__device__ __forceinline__ bool bar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(1000000u)
        : "memory");
    return ok != 0;
}
// mbar_wait_bounded by a whole warp; the same answer in every lane.  (The
// control warps run their loops with all lanes and elect one for the copies
// and multiplies: with lane 0 alone in the loop every operand of those went
// from a per-thread to a uniform register first, 800 cycles a group.)
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
    bool ok = bar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return true;
    const long long t0 = clock64();
    bool all, late;
    do {
        ok = ok || bar_try_wait(bar, parity);
        all = __all_sync(0xffffffffu, ok);
        late = __any_sync(0xffffffffu, clock64() - t0 > kWaitLimitCycles);
    } while (!all && !late);
    return all;
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrival at cluster address `bar` of a warp whose reads of a product buffer are
// complete (tcgen05.wait::ld) and fenced (tc_before): no memory of this CTA has
// to become visible to the other one, which a release over the cluster would
// wait for (8000 x 6144 x 4096 376 us against 205).
template <bool PAIR>
__device__ __forceinline__ void buffer_release(uint32_t bar) {
    if constexpr (PAIR) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
    else bar_arrive(bar);
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ float ld_shared_f(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared_f(uint32_t a, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(p));
    return p != 0;
}
// First run of 4 columns that split q of a 128-wide tile sums up.
__device__ __forceinline__ int first_run(int q, int splits) { return (q * 32 + splits - 1) / splits; }
// 2-D tiled TMA load into this CTA's shared memory, completion counted on the
// barrier at cluster address `bar` (of either CTA of the pair).
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
            " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
            : "memory");
}

// Four sums of row m, columns n .. n + 3: residual added, rounded once, stored.
__device__ __forceinline__ void store_out4(const LinArgs& a, int m, int n, float4 v) {
    const size_t e = (size_t)m * a.N + n;
    if (a.vec && n + 4 <= a.N) {
        if (a.residual) {
            const float4 r = *reinterpret_cast<const float4*>(a.residual + e);
            v.x += r.x;
            v.y += r.y;
            v.z += r.z;
            v.w += r.w;
        }
        if (a.out_dtype == COTTUS_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + e) = v;
        else if (a.out_dtype == COTTUS_F16)
            *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(a.out) + e) = make_uint2(pack_h2(v.x, v.y), pack_h2(v.z, v.w));
        else
            *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + e) =
                make_uint2(pack_bf2(v.x, v.y), pack_bf2(v.z, v.w));
        return;
    }
    const float s[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (n + j >= a.N) break;
        const float y = a.residual ? s[j] + a.residual[e + j] : s[j];
        if (a.out_dtype == COTTUS_F32) reinterpret_cast<float*>(a.out)[e + j] = y;
        else if (a.out_dtype == COTTUS_F16) reinterpret_cast<__half*>(a.out)[e + j] = __float2half_rn(y);
        else reinterpret_cast<__nv_bfloat16*>(a.out)[e + j] = __float2bfloat16_rn(y);
    }
}

// Sums of weight row n (this thread's) and rows m0 .. of x: a warp stores runs
// of 32 columns.
template <int HC>
__device__ __forceinline__ void store_column(const LinArgs& a, int m0, int n, const float2 (&acc)[HC / 2]) {
    if (n >= a.N) return;
    const float* res = a.residual ? a.residual + (size_t)m0 * a.N + n : nullptr;
    const size_t e = (size_t)m0 * a.N + n;
    const int rows = a.M - m0;
    auto each = [&](auto put) {
#pragma unroll
        for (int c = 0; c < HC; ++c)
            if (c < rows) {
                const float v = c & 1 ? acc[c / 2].y : acc[c / 2].x;
                put((size_t)c * a.N, res ? v + res[(size_t)c * a.N] : v);
            }
    };
    if (a.out_dtype == COTTUS_F32) each([&](size_t o, float v) { reinterpret_cast<float*>(a.out)[e + o] = v; });
    else if (a.out_dtype == COTTUS_F16) each([&](size_t o, float v) { reinterpret_cast<__half*>(a.out)[e + o] = __float2half_rn(v); });
    else each([&](size_t o, float v) { reinterpret_cast<__nv_bfloat16*>(a.out)[e + o] = __float2bfloat16_rn(v); });
}

// Position in a ring of n slots and the parity of its current pass.
struct Ring {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int n) {
        if (++slot == n) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// XR: rows of x per CTA.  PAIR: the wide tile, two CTAs of one; else the narrow
// one, by one CTA or a.splits of them.
template <int XR, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) fp8_linear_kernel(const __grid_constant__ CUtensorMap xmap,
                                                                 const __grid_constant__ CUtensorMap wmap,
                                                                 const __grid_constant__ CUtensorMap omap,
                                                                 const LinArgs a) {
    static_assert(!PAIR || XR == kBM, "a pair's CTA brings 128 rows of x and of the weight");
    constexpr int BN = PAIR ? 2 * kWRows : kWRows;   // rows of the weight in a tile
    constexpr int COLS = PAIR ? BN : XR;             // TMEM columns of a product
    constexpr int HALF = COLS / 2;                   // and of a sum warp's share
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    // everything in shared memory by 32-bit address
    const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;
    constexpr uint32_t stage_bytes = (XR + kWRows) * kBK;
    const uint32_t staging = ring + a.stages * stage_bytes;
    const uint32_t scales = staging + a.staging_bytes;
    const uint32_t full = scales + kScaleSlots * kScaleBatch * kScaleWords * 4;
    const uint32_t empty = full + kMaxStages * 8;
    const uint32_t tm_full = empty + kMaxStages * 8;
    const uint32_t tm_empty = tm_full + kMaxBufs * 8;
    const uint32_t sc_full = tm_empty + kMaxBufs * 8;
    const uint32_t sc_empty = sc_full + kScaleSlots * 8;
    const uint32_t done = sc_empty + kScaleSlots * 8;
    const uint32_t words = done + 8;
    uint8_t* generic = smem_raw + (words - smem_addr(smem_raw));
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(generic);
    volatile uint32_t* s_failed = s_tmem + 1;  // a wait of this CTA ran out; one of the cluster did
    uint32_t* s_run = s_tmem + 4;              // splits: where a run of 4 columns is summed up (cluster address)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int splits = PAIR ? 1 : a.splits;
    // (splits have few groups, and with half of the TMEM the next launch's CTA
    // can allocate its own while this one runs)
    const int bufs = PAIR || (XR == 128 && splits > 1) ? 2 : 4;
    const uint32_t tmem_cols = bufs * COLS;
    const int cluster = PAIR ? 2 : splits;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    const int first = blockIdx.x / cluster, step = gridDim.x / cluster;
    const int tiles = a.m_tiles * a.n_tiles;
    // this CTA's groups of every tile it works on
    const int g0 = PAIR ? 0 : (int)((long long)a.groups * rank / splits);
    const int g1 = PAIR ? a.groups : (int)((long long)a.groups * (rank + 1) / splits);
    // first row of x, and first column, of tile t in this CTA
    auto tile_m = [&](int t) { return PAIR ? (t % a.m_tiles * 2 + rank) * kBM : t % a.m_tiles * XR; };
    auto tile_n = [&](int t) { return t / a.m_tiles * BN; };

    if (threadIdx.x == 0) {
        prefetch_tensormap(&xmap);
        prefetch_tensormap(&wmap);
        for (int i = 0; i < a.stages; ++i) {
            bar_init(full + i * 8, 1);
            bar_init(empty + i * 8, 1);
        }
        for (int i = 0; i < bufs; ++i) {
            bar_init(tm_full + i * 8, 1);
            bar_init(tm_empty + i * 8, (PAIR ? 2 : 1) * kSumWarps);
        }
        for (int i = 0; i < kScaleSlots; ++i) {
            bar_init(sc_full + i * 8, 2);
            bar_init(sc_empty + i * 8, kSumWarps);
        }
        bar_init(done, 1);
        fence_barrier_init();
        s_failed[0] = s_failed[1] = 0;
    }
    if (warp == kSumWarps + 1) tmem_alloc<PAIR>(words, tmem_cols);
    if (!PAIR && splits > 1 && warp == kSumWarps + 2) {
        // run r of 32 (4 rows of the weight each) belongs to split r * splits
        // / 32; its sums lie at [split][row of x][run] there
        const int q = (lane * splits) >> 5;
        s_run[lane] = cluster_addr(staging, q) + (lane - first_run(q, splits)) * 16;
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *s_tmem;
    // every CTA of the cluster has started and set up its barriers (a pair
    // needs that now, splits before they send their sums)
    if (cluster > 1) cluster_arrive();
    if (PAIR) cluster_wait();
    // the first groups' weights start on their way to L2 before the preceding
    // kernel is done (a hint: nothing is read here, and what that kernel still
    // writes, L2 sees): 64 x 4096 x 4096 8.8 -> 8.6 us in a chain of launches
    if (warp == kSumWarps && first < tiles && elect_one()) {
        const int w0 = tile_n(first) + (PAIR ? rank * kWRows : 0);
        for (int g = g0; g < g1 && g < g0 + kPrefetch; ++g) tma_prefetch_l2_2d(&wmap, g * kBK, w0);
    }
    grid_dependency_wait();
    // (after the allocation above: a dependent that also allocates TMEM can
    // then only wait for this grid, never the other way round)
    grid_dependents_launch();

    bool ok = true;
    if (warp >= kSumWarps) {
        if constexpr (PAIR) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtrlRegs));
        if (warp == kSumWarps) {
            // ---- producer ------------------------------------------------
            Ring r;
            int issued = 0;
            for (int t = first; t < tiles && ok; t += step) {
                const int m0 = tile_m(t), w0 = tile_n(t) + (PAIR ? rank * kWRows : 0);
                for (int g = g0; g < g1; ++g) {
                    const uint32_t bar = full + r.slot * 8, st = ring + r.slot * stage_bytes;
                    ok = bar_wait(empty + r.slot * 8, r.phase ^ 1);
                    if (!ok) break;
                    if (elect_one()) {
                        // (a pair: the first CTA's barrier counts both CTAs' bytes)
                        const uint32_t at = PAIR ? cluster_addr(bar, 0) : bar;
                        if (!PAIR || rank == 0) bar_expect(bar, (PAIR ? 2 : 1) * stage_bytes);
                        tma_load<PAIR>(st, &xmap, at, g * kBK, m0);
                        tma_load<PAIR>(st + XR * kBK, &wmap, at, g * kBK, w0);
                    }
                    __syncwarp();
                    ++issued;
                    r.next(a.stages);
                }
            }
            if (!ok) {
                // let the copies in flight land before giving up (a pair's
                // second CTA leaves it to the first, whose barriers count
                // them, and waits for it at the end)
                Ring q = r;
                for (int i = 0; i < a.stages && i < issued && !(PAIR && rank); ++i) {
                    if (q.slot == 0) {
                        q.slot = a.stages;
                        q.phase ^= 1;
                    }
                    --q.slot;
                    (void)bar_wait(full + q.slot * 8, q.phase);
                }
                if (lane == 0) s_failed[0] = 1;
            }
        } else if (warp == kSumWarps + 1 && !(PAIR && rank)) {
            // ---- MMA issue -----------------------------------------------
            constexpr uint32_t idesc = PAIR ? f8_idesc<2 * kBM, BN>() : f8_idesc<kWRows, XR>();
            Ring r, b;
            const uint64_t xdesc = sw128_kmajor_desc(ring);
            const uint64_t wdesc = sw128_kmajor_desc(ring + XR * kBK);
            for (int t = first; t < tiles && ok; t += step) {
                for (int g = g0; g < g1; ++g) {
                    // (descriptors count 16 bytes; the sums' release comes
                    // last and is what the multiplies usually wait for)
                    const uint32_t off = r.slot * (stage_bytes / 16);
                    const uint64_t ad = (PAIR ? xdesc : wdesc) + off, bd = (PAIR ? wdesc : xdesc) + off;
                    const uint32_t d = tmem + (uint32_t)(b.slot * COLS);
                    ok = bar_wait(full + r.slot * 8, r.phase) && bar_wait(tm_empty + b.slot * 8, b.phase ^ 1);
                    if (!ok) break;
                    tc_after();
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < kBK / 32; ++kk) mma_f8<PAIR>(d, ad + 2 * kk, bd + 2 * kk, idesc, (uint32_t)kk);
                        mma_commit<PAIR>(tm_full + b.slot * 8);
                        mma_commit<PAIR>(empty + r.slot * 8);
                    }
                    __syncwarp();
                    r.next(a.stages);
                    b.next(bufs);
                }
            }
            if (!ok) {
                // every multiply issued so far ends before the memory is given back
                if (elect_one()) mma_commit<PAIR>(done);
                __syncwarp();
                (void)bar_wait(done, 0);
                if (lane == 0) s_failed[0] = 1;
            }
        } else if (warp >= kSumWarps + 2) {
            // ---- scales: half of the rows each, kScaleBatch groups at once ----
            const int part = warp - kSumWarps - 2;
            Ring r;
            for (int t = first; t < tiles && ok; t += step) {
                // (the wide tile keeps its two weight scales apart; the narrow
                // one's single scale goes into the rows')
                const int r0 = part * 64 + lane, m = tile_m(t) + r0, nb = tile_n(t) / 128 + (PAIR ? lane : 0);
                const bool live0 = r0 < XR && m < a.M, live1 = r0 + 32 < XR && m + 32 < a.M;
                const bool live_w = PAIR ? part == 0 && lane < BN / 128 && nb < a.n_blocks : live0 || live1;
                const float* xs = a.xs + m;
                const float* ws = a.ws + (size_t)nb * a.groups;
                for (int gb = g0; gb < g1 && ok; gb += kScaleBatch) {
                    float v0[kScaleBatch], v1[kScaleBatch], w[kScaleBatch];
#pragma unroll
                    for (int j = 0; j < kScaleBatch; ++j) {
                        const int g = gb + j;
                        v0[j] = live0 && g < g1 ? xs[(size_t)g * a.M] : 0.f;
                        v1[j] = live1 && g < g1 ? xs[(size_t)g * a.M + 32] : 0.f;
                        w[j] = live_w && g < g1 ? ws[g] : 0.f;
                    }
                    ok = bar_wait(sc_empty + r.slot * 8, r.phase ^ 1);
                    if (!ok) break;
#pragma unroll
                    for (int j = 0; j < kScaleBatch; ++j) {
                        const uint32_t dst = scales + ((r.slot * kScaleBatch + j) * kScaleWords + lane) * 4;
                        if (r0 < XR) st_shared_f(dst + part * 256, PAIR ? v0[j] : v0[j] * w[j]);
                        if (r0 + 32 < XR) st_shared_f(dst + part * 256 + 128, PAIR ? v1[j] : v1[j] * w[j]);
                        if (PAIR && part == 0 && lane < BN / 128) st_shared_f(dst + kBM * 4, w[j]);
                    }
                    __syncwarp();
                    if (lane == 0) bar_arrive(sc_full + r.slot * 8);
                    r.next(kScaleSlots);
                }
            }
            if (!ok && lane == 0) s_failed[0] = 1;
        }
        __syncwarp();
        if (!PAIR && cluster > 1) cluster_wait();
    } else {
        if constexpr (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        // ---- sums ----------------------------------------------------------
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * HALF);
        // a buffer's release goes to the CTA that issues the multiplies
        const uint32_t tm_free = PAIR ? cluster_addr(tm_empty, 0) : tm_empty;
        const uint32_t stg = staging + warp * kWarpStaging;
        if (!PAIR && cluster > 1) cluster_wait();
        Ring b, r;
        for (int t = first; t < tiles && ok; t += step) {
            // this warp's first row of x and of the weight
            const int m0 = tile_m(t) + (PAIR ? quad * 32 : half * HALF), nh = tile_n(t) + (PAIR ? half * HALF : quad * 32);
            const bool rows_live = m0 < a.M;  // (uniform in the warp)
            float2 acc[HALF / 2];
#pragma unroll
            for (int c = 0; c < HALF / 2; ++c) acc[c] = make_float2(0.f, 0.f);
            for (int gb = g0; gb < g1; gb += kScaleBatch) {
                ok = bar_wait(sc_full + r.slot * 8, r.phase);
                if (!ok) break;
                const uint32_t sc = scales + r.slot * (kScaleBatch * kScaleWords * 4);
                float sg[kScaleBatch];
                if constexpr (PAIR) {
                    // (the weight's scale is the same word for the whole warp)
#pragma unroll
                    for (int j = 0; j < kScaleBatch; ++j)
                        sg[j] = ld_shared_f(sc + (j * kScaleWords + quad * 32 + lane) * 4) *
                                ld_shared_f(sc + (j * kScaleWords + kBM + half) * 4);
                    __syncwarp();
                    if (lane == 0) bar_arrive(sc_empty + r.slot * 8);
                    r.next(kScaleSlots);
                }
#pragma unroll
                for (int j = 0; j < kScaleBatch; ++j) {
                    if (gb + j >= g1) break;
                    const uint32_t at = taddr + (uint32_t)(b.slot * COLS);
                    const uint32_t freed = tm_free + b.slot * 8;
                    ok = bar_wait(tm_full + b.slot * 8, b.phase);
                    if (!ok) break;
                    b.next(bufs);
                    tc_after();
                    if (rows_live) {
                        // the next 32 columns are on their way while these are
                        // added (a load takes about 75 cycles whatever its width);
                        // the buffer is free once the last ones are here
                        constexpr int W = HALF < 32 ? HALF : 32;
                        uint32_t v[2][32];
                        if constexpr (W == 8) tmem_get8(at, v[0]);
                        else if constexpr (W == 16) tmem_get16(at, v[0]);
                        else tmem_ld32(at, v[0]);
#pragma unroll
                        for (int i = 0; i < HALF / W; ++i) {
                            if constexpr (W == 32) tmem_wait_ld(v[i & 1]);
                            if (i + 1 < HALF / W) {
                                tmem_ld32(at + (uint32_t)(i + 1) * 32, v[(i + 1) & 1]);
                            } else {
                                tc_before();
                                if (lane == 0) buffer_release<PAIR>(freed);
                            }
#pragma unroll
                            for (int c = 0; c < W; c += 4) {
                                float2 sa, sb;
                                if constexpr (PAIR) {
                                    sa = sb = make_float2(sg[j], sg[j]);
                                } else {
                                    const float4 s4 = ld_shared_f4(sc + (j * kScaleWords + half * HALF + i * W + c) * 4);
                                    sa = make_float2(s4.x, s4.y);
                                    sb = make_float2(s4.z, s4.w);
                                }
                                const uint32_t(&u)[32] = v[i & 1];
                                float2 &ta = acc[(i * W + c) / 2], &tb = acc[(i * W + c) / 2 + 1];
                                ta = ffma2(make_float2(__uint_as_float(u[c]), __uint_as_float(u[c + 1])), sa, ta);
                                tb = ffma2(make_float2(__uint_as_float(u[c + 2]), __uint_as_float(u[c + 3])), sb, tb);
                            }
                        }
                    } else if (lane == 0) {
                        buffer_release<PAIR>(freed);
                    }
                }
                if constexpr (!PAIR) {
                    __syncwarp();
                    if (lane == 0) bar_arrive(sc_empty + r.slot * 8);
                    r.next(kScaleSlots);
                }
                if (!ok) break;
            }
            if (!ok) break;
            if (!PAIR && splits > 1) {
                // (the only tile of this cluster) every sum goes to the CTA that
                // adds its weight row up
                if constexpr (!PAIR) {
                    const int runs = (32 + splits - 1) / splits, row = quad * 32 + lane;
                    const uint32_t to = s_run[row >> 2] + (uint32_t)((rank * XR + half * HALF) * runs * 16 + (row & 3) * 4);
#pragma unroll
                    for (int c = 0; c < HALF; ++c)
                        if (m0 + c < a.M) st_cluster_f(to + c * runs * 16, c & 1 ? acc[c / 2].y : acc[c / 2].x);
                }
            } else if constexpr (!PAIR) {
                if (rows_live) store_column<HALF>(a, m0, nh + lane, acc);
            } else if (a.tma_out) {
                // 128 bytes of each of the warp's rows at a time, swizzled as
                // the tensor map has it, stored by TMA (which drops what lies
                // past the last row or column)
                if (rows_live) {
                    const uint32_t row = stg + lane * 128;
                    const uint32_t swz = lane & 7;
                    if (a.out_dtype == COTTUS_F32) {
#pragma unroll
                        for (int c0 = 0; c0 < HALF; c0 += 32) {
                            if (lane == 0) tma_store_read();
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float2 u = acc[c0 / 2 + 2 * j], w = acc[c0 / 2 + 2 * j + 1];
                                st_shared_u4(row + ((j ^ swz) << 4), make_uint4(__float_as_uint(u.x), __float_as_uint(u.y),
                                                                               __float_as_uint(w.x), __float_as_uint(w.y)));
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0 && nh + c0 < a.N) tma_store(&omap, stg, (nh + c0) * 4, m0);
                        }
                    } else {
                        const bool f16 = a.out_dtype == COTTUS_F16;
#pragma unroll
                        for (int c0 = 0; c0 < HALF; c0 += 64) {
                            if (lane == 0) tma_store_read();
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                uint32_t p[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float2 u = acc[c0 / 2 + 4 * j + e];
                                    p[e] = f16 ? pack_h2(u.x, u.y) : pack_bf2(u.x, u.y);
                                }
                                st_shared_u4(row + ((j ^ swz) << 4), make_uint4(p[0], p[1], p[2], p[3]));
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0 && nh + c0 < a.N) tma_store(&omap, stg, (nh + c0) * 2, m0);
                        }
                    }
                }
            } else if (rows_live) {
                // 16 columns at a time through shared memory, so that four
                // lanes store (and read the residual of) one run of a row
#pragma unroll
                for (int c0 = 0; c0 < HALF; c0 += 16) {
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 16; c += 4) {
                        const float2 u = acc[(c0 + c) / 2], w = acc[(c0 + c) / 2 + 1];
                        st_shared_u4(stg + (lane * kStagePitch + c) * 4, make_uint4(__float_as_uint(u.x), __float_as_uint(u.y),
                                                                                   __float_as_uint(w.x), __float_as_uint(w.y)));
                    }
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = i * 8 + (lane >> 2), n = nh + c0 + (lane & 3) * 4;
                        const float4 v = ld_shared_f4(stg + (rr * kStagePitch + (lane & 3) * 4) * 4);
                        if (m0 + rr < a.M && n < a.N) store_out4(a, m0 + rr, n, v);
                    }
                }
            }
        }
        if (lane == 0) tma_store_done();
        if (!ok && lane == 0) s_failed[0] = 1;
    }
    __syncwarp();
    if (!PAIR && splits > 1) {
        __syncthreads();
        if (threadIdx.x < splits && s_failed[0]) st_cluster_u32(cluster_addr(words + 8, threadIdx.x), 1u);
        __syncwarp();
        cluster_arrive();
        cluster_wait();  // every CTA's partial sums are where they are added
        if (!s_failed[1]) {
            const int m0 = tile_m(first), n0 = tile_n(first);
            const int rows = a.M - m0 < XR ? a.M - m0 : XR;
            const int run0 = first_run(rank, splits), runs = first_run(rank + 1, splits) - run0;
            const int sh = runs > 16 ? 5 : (runs > 8 ? 4 : (runs > 4 ? 3 : 2));  // lanes per row
            const int run = threadIdx.x & ((1 << sh) - 1), n = n0 + (run0 + run) * 4;
            if (run < runs && n < a.N) {
                const int pitch = (32 + splits - 1) / splits * 16;
                for (int row = threadIdx.x >> sh; row < rows; row += kThreads >> sh) {
                    const uint32_t p = staging + row * pitch + run * 16;
                    float4 v = ld_shared_f4(p);
                    for (int q = 1; q < splits; ++q) {
                        const float4 w = ld_shared_f4(p + q * XR * pitch);
                        v.x += w.x;
                        v.y += w.y;
                        v.z += w.z;
                        v.w += w.w;
                    }
                    store_out4(a, m0 + row, n, v);
                }
            }
        }
    }
    tc_before();
    __syncthreads();
    if (PAIR) {  // neither CTA leaves while the other's multiplies and arrivals may reach it
        cluster_arrive();
        cluster_wait();
    }
    if (threadIdx.x == 0 && s_failed[0]) report(a.status, COTTUS_STATUS_TIMEOUT);
    if (warp == kSumWarps + 1) tmem_free<PAIR>(tmem, tmem_cols);
}

// ---------------------------------------------------------------------------
// few rows of x by a small weight
// ---------------------------------------------------------------------------
constexpr int kThinTile = 16;   // rows of the weight per CTA
constexpr int kThinWarps = 16;  // each takes every 16th group

// Two e4m3 values as two fp16 ones (exact).
__device__ __forceinline__ uint32_t half2_of(uint32_t e4m3x2) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)e4m3x2));
    return r;
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Up to 8 NT rows of x by 16 rows of the weight per CTA.  No shared memory,
// tensor memory or cluster on the way of the weight: a lane loads 16 bytes each
// of weight rows l / 4 and l / 4 + 8 and of rows l / 4 (+ 8 ...) of x at the same
// columns, which is what it needs for four multiplies, as long as both sides
// number the columns alike (in the multiply's terms columns 2t, 2t + 1, 2t + 8
// and 2t + 9 of step i are bytes 4i to 4i + 3 of the lane's 16).  Products of
// two e4m3 values are exact in fp16's tensor core and its sums fp32.
template <int NT>
__global__ void __launch_bounds__(kThinWarps * 32) fp8_linear_thin_kernel(const uint8_t* x, const uint8_t* w, const LinArgs a,
                                                                          const int K) {
    __shared__ float part[kThinWarps][kThinTile][8 * NT + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * kThinTile;
    const bool live0 = n0 + r < a.N, live1 = n0 + r + 8 < a.N;
    const uint8_t* w0 = w + (size_t)(n0 + r) * K + t * 16;
    const uint8_t* w1 = w0 + (size_t)8 * K;
    const uint8_t* xr = x + (size_t)r * K + t * 16;
    const float* ws = a.ws + (size_t)(n0 / 128) * a.groups;
    // (the first weights' way to L2 before the preceding kernel is done: a hint, as above)
    if (t == 0 && live0 && warp * kBK < K) asm volatile("prefetch.global.L2 [%0];" ::"l"(w0 + warp * kBK));
    if (t == 0 && live1 && warp * kBK < K) asm volatile("prefetch.global.L2 [%0];" ::"l"(w1 + warp * kBK));
    grid_dependency_wait();
    grid_dependents_launch();
    float sum[NT][4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int g = warp; g < a.groups; g += kThinWarps) {
        uint4 wa[2], wb[2], xv[2][NT];
        float s[NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = g * kBK + h * 64;
            const bool in = c + t * 16 < K;
            wa[h] = in && live0 ? ld_once(w0 + c) : zero;
            wb[h] = in && live1 ? ld_once(w1 + c) : zero;
#pragma unroll
            for (int q = 0; q < NT; ++q)
                // (no restricted pointers here: a read that counts as constant might move ahead of the wait)
                xv[h][q] = in && r + q * 8 < a.M ? *reinterpret_cast<const uint4*>(xr + (size_t)q * 8 * K + c) : zero;
        }
        const float sw = ws[g];
        const float* xs = a.xs + (size_t)g * a.M;
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int m = q * 8 + 2 * t + j;
                s[q][j] = m < a.M ? xs[m] * sw : 0.f;
            }
        float d[NT][4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t ua[4] = {wa[h].x, wa[h].y, wa[h].z, wa[h].w}, ub[4] = {wb[h].x, wb[h].y, wb[h].z, wb[h].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t f[4] = {half2_of(ua[i]), half2_of(ub[i]), half2_of(ua[i] >> 16), half2_of(ub[i] >> 16)};
#pragma unroll
                for (int q = 0; q < NT; ++q) {
                    const uint32_t ux = i == 0 ? xv[h][q].x : (i == 1 ? xv[h][q].y : (i == 2 ? xv[h][q].z : xv[h][q].w));
                    mma_16816(d[q], f, half2_of(ux), half2_of(ux >> 16));
                }
            }
        }
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[q][j] = fmaf(d[q][j], s[q][j & 1], sum[q][j]);
    }
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[warp][r + (j >> 1) * 8][q * 8 + 2 * t + (j & 1)] = sum[q][j];
    __syncthreads();
    const int row = threadIdx.x & 15, n = n0 + row, m = threadIdx.x >> 4;
    if (m < a.M && n < a.N) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kThinWarps; ++q) v += part[q][row][m];
        const size_t e = (size_t)m * a.N + n;
        if (a.residual) v += a.residual[e];
        if (a.out_dtype == COTTUS_F32) reinterpret_cast<float*>(a.out)[e] = v;
        else if (a.out_dtype == COTTUS_F16) reinterpret_cast<__half*>(a.out)[e] = __float2half_rn(v);
        else reinterpret_cast<__nv_bfloat16*>(a.out)[e] = __float2bfloat16_rn(v);
    }
}
template <int NT>
cudaError_t launch_thin(const cottus_fp8_linear_params* p, const LinArgs& a, cudaStream_t st) {
    return launch_pdl(fp8_linear_thin_kernel<NT>, dim3((unsigned)((a.N + kThinTile - 1) / kThinTile)), dim3(kThinWarps * 32), 0,
                      st, static_cast<const uint8_t*>(p->x), static_cast<const uint8_t*>(p->weight), a, p->in_features);
}

int fail(int code, const std::string& msg) { return set_error(code, msg); }

// What a device allows, found at the first call that asks.
struct DeviceLimits {
    int clusters[kMaxSplits + 1] = {};  // narrow-tile clusters of each size that are resident at once
    int pairs = 0;                      // and wide-tile pairs (not every SM has a partner); 0: no wide tile
};
cudaError_t find_limits(DeviceLimits& l) {
    auto resident = [](auto kern, int size, int& n) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(size);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kSmemMax;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
    };
    cudaError_t e = cudaSuccess;
    auto set_up = [&](auto kern) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax);
    };
    set_up(fp8_linear_kernel<16, false>);
    set_up(fp8_linear_kernel<32, false>);
    set_up(fp8_linear_kernel<64, false>);
    set_up(fp8_linear_kernel<128, false>);
    set_up(fp8_linear_kernel<128, true>);
    for (int s = 1; s <= kMaxSplits && e == cudaSuccess; ++s) e = resident(fp8_linear_kernel<128, false>, s, l.clusters[s]);
    // (a warp is given registers in steps of 8 per thread; compiled to fewer
    // than its split needs, the wide tile is left out)
    cudaFuncAttributes wide = {};
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&wide, fp8_linear_kernel<128, true>);
    if (e == cudaSuccess && (wide.numRegs + 7) / 8 * 8 >= kMinLaunchRegs) e = resident(fp8_linear_kernel<128, true>, 2, l.pairs);
    return e;
}
cudaError_t limits(int dev, DeviceLimits& l) {
    static PerDevice<DeviceLimits, cudaError_t> known;
    return known.get(dev, l, cudaErrorInvalidDevice, find_limits);
}

template <int XR, bool PAIR>
cudaError_t launch_linear(const cottus_fp8_linear_params* p, LinArgs a, int grid, cudaStream_t st) {
    cudaError_t err = cudaSuccess;
    a.staging_bytes = PAIR ? kSumWarps * kWarpStaging : 0;
    if (a.splits > 1) a.staging_bytes = a.splits * XR * ((32 + a.splits - 1) / a.splits) * 16;
    const size_t stage = (size_t)(XR + kWRows) * kBK;
    const size_t rest = 1024 + (size_t)a.staging_bytes + kTailBytes;
    a.stages = (int)((kSmemMax - rest) / stage);
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    // no more stages than a split has groups: a launch that needs little
    // shared memory can become resident beside the one before it
    const int most = (a.groups + a.splits - 1) / a.splits;
    if (a.splits > 1 && a.stages > most) a.stages = most;
    const CUtensorMap xmap = make_tensor_map_2d_u8(p->x, p->in_features, p->rows, p->in_features, kBK, XR, true, &err);
    if (err != cudaSuccess) return err;
    const CUtensorMap wmap =
        make_tensor_map_2d_u8(p->weight, p->in_features, p->out_features, p->in_features, kBK, kWRows, true, &err);
    if (err != cudaSuccess) return err;
    CUtensorMap omap = wmap;  // (not read without tma_out)
    const int es = dtype_bytes(p->out_dtype);
    a.tma_out = PAIR && !p->residual && aligned(p->out, 16) && (size_t)p->out_features * es % 16 == 0;
    if (a.tma_out) {
        omap = make_tensor_map_2d_u8(p->out, (uint64_t)p->out_features * es, p->rows, (uint64_t)p->out_features * es, 128, 32,
                                     true, &err);
        if (err != cudaSuccess) return err;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = rest + (size_t)a.stages * stage;
    // A cluster's CTAs wait for one another with their tensor memory allocated,
    // and an allocation waits for as long as it takes: CTAs of two such kernels
    // that met on the same SMs in opposite order could hold what the other one
    // needs.  The wide tile's registers (64512 of 65536) keep everything else
    // off its SMs; splits take half of an SM's shared memory, so that a kernel
    // that uses the rest of it for its own multiplies does not join them (two
    // of these do: with 256 columns each at most their tensor memory fits).
    // Decode projections take the same time with it.
    if (a.splits > 1 && cfg.dynamicSmemBytes < kSplitSmem) cfg.dynamicSmemBytes = kSplitSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = PAIR ? 2 : a.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR || a.splits > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, fp8_linear_kernel<XR, PAIR>, xmap, wmap, omap, a);
}

}  // namespace
}  // namespace cb200

extern "C" int cottus_fp8_linear(const cottus_fp8_linear_params* p, cottus_stream_t stream) {
    using namespace cb200;
    if (!p) return fail(COTTUS_ERR_INVALID_ARGUMENT, "params must not be NULL");
    if (p->rows < 0 || p->out_features <= 0 || p->in_features <= 0)
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "rows must be non-negative, out_features and in_features positive");
    if (!lowp_input_dtype(p->out_dtype)) return fail(COTTUS_ERR_INVALID_ARGUMENT, "unknown out dtype");
    if (p->in_features % 16 != 0) return fail(COTTUS_ERR_UNSUPPORTED, "in_features must be a multiple of 16");
    if (p->rows == 0) return COTTUS_OK;
    if (!p->x || !p->x_scales || !p->weight || !p->w_scales || !p->out)
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "NULL pointer argument");
    const int es = dtype_bytes(p->out_dtype);
    if (!aligned(p->x, 16) || !aligned(p->weight, 16)) return fail(COTTUS_ERR_INVALID_ARGUMENT, "x and weight must be 16-byte aligned");
    if (!aligned(p->out, es) || !aligned(p->residual, 4) || !aligned(p->x_scales, 4) || !aligned(p->w_scales, 4))
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its element");
    const int M = p->rows, N = p->out_features, K = p->in_features;
    if (M > kMaxWidth || N > kMaxWidth || K > kMaxWidth) return fail(COTTUS_ERR_UNSUPPORTED, "product too large");
    const int groups = (K + 127) / 128;
    const size_t mn = (size_t)M * N;
    const Span so{p->out, mn * es}, sr{p->residual, p->residual ? mn * 4 : 0}, sx{p->x, (size_t)M * K},
        sw{p->weight, (size_t)N * K}, sxs{p->x_scales, (size_t)M * groups * 4},
        sws{p->w_scales, (size_t)((N + 127) / 128) * groups * 4};
    if ((overlap(so, sr) && !(p->out_dtype == COTTUS_F32 && p->out == p->residual)) || overlap(so, sx) ||
        overlap(so, sw) || overlap(so, sxs) || overlap(so, sws))
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "out overlaps another buffer");
    LinArgs a = {};
    a.xs = p->x_scales;
    a.ws = p->w_scales;
    a.residual = p->residual;
    a.out = p->out;
    a.status = p->status;
    a.M = M;
    a.N = N;
    a.groups = groups;
    a.n_blocks = (N + 127) / 128;
    a.out_dtype = p->out_dtype;
    a.vec = N % 4 == 0 && aligned(p->out, es * 4) && aligned(p->residual, 16);
    auto cuda_fail = [](cudaError_t e) { return fail(COTTUS_ERR_CUDA, std::string("CUDA error: ") + cudaGetErrorString(e)); };
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return cuda_fail(e);
    const int sms = device_sm_count(device);
    const int64_t narrow = (int64_t)((M + 127) / 128) * ((N + 127) / 128), wide = (int64_t)((M + 255) / 256) * ((N + 255) / 256);
    if (narrow >= (int64_t(1) << 30)) return fail(COTTUS_ERR_UNSUPPORTED, "product too large");
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // The thin kernel while its CTAs are few and short, against the narrow tile
    // in us.  Up to 8 rows two CTAs share an SM.  All of them resident at once, one
    // row: 1000 x 512 1.6 : 3.1, 2048 x 2048 2.4 : 4.5, 4096 x 4096 4.8 : 6.9, 4096 x
    // 8192 8.2 : 10.1; 512 x 28672 18.6 : 11.1.  In two waves the second is part
    // empty, which the narrow tile makes up for once a warp has more than two
    // groups or the last of them leaves many warps idle: 6144 x 4096 7.7 : 8.9, 8192 x
    // 4096 8.5 : 9.7, 9472 x 512 3.9 : 4.1, 6144 x 3584 7.9 : 8.2; 6144 x 2560 7.5 : 7.0,
    // 5120 x 5120 9.8 : 8.8, 8192 x 8192 15.1 : 15.0, and with 8 rows 10.7 : 8.9 and
    // 16.0 : 15.3.  Three waves: 16384 x 1024 8.6 : 5.6, 32000 x 2048 17.9 : 14.8.
    // 16 rows (its registers then leave one CTA per SM): 2368 x 4096 4.6 : 6.2, 2048 x
    // 2048 2.8 : 4.6; 4096 x 4096 8.5 : 7.1, 1184 x 8192 7.5 : 6.4.
    const int64_t thin = (N + kThinTile - 1) / kThinTile;
    const int rounds = (groups + kThinWarps - 1) / kThinWarps;  // groups of a warp
    const bool two_waves = thin <= 4 * sms && (rounds == 1 || (rounds == 2 && groups >= 28));
    if (M <= 8 && ((thin <= 2 * sms && rounds <= 4) || two_waves)) {
        e = launch_thin<1>(p, a, st);
        return e == cudaSuccess ? COTTUS_OK : cuda_fail(e);
    }
    if (M <= 16 && thin <= sms && groups <= 2 * kThinWarps) {
        e = launch_thin<2>(p, a, st);
        return e == cudaSuccess ? COTTUS_OK : cuda_fail(e);
    }
    DeviceLimits dev;
    e = limits(device, dev);
    if (e != cudaSuccess) return cuda_fail(e);
    if (M > 128 && dev.pairs > 0 && narrow > sms) {
        // The wide tile where the narrow ones do not fit the GPU at once.  K = 4096,
        // narrow against wide in us: 144 narrow tiles (384 x 6144) 15.4 : 19.4,
        // 192 (512 x 6144) 25.2 : 19.6, 384 (1024 x 6144) 36.7 : 34.0, 1152 (3000 x
        // 6144) 90 : 71.  Up to 128 rows half of the wide tile would be empty.
        a.m_tiles = (M + 255) / 256;
        a.n_tiles = (N + 255) / 256;
        a.splits = 1;
        e = launch_linear<128, true>(p, a, 2 * (int)(wide < dev.pairs ? wide : dev.pairs), st);
    } else {
        a.m_tiles = (M + 127) / 128;
        a.n_tiles = (N + 127) / 128;
        // as many splits as leave all clusters resident at once
        a.splits = 1;
        for (int s = 2; s <= kMaxSplits && s <= groups; ++s)
            if (narrow <= dev.clusters[s]) a.splits = s;
        const int grid = a.splits > 1 ? (int)narrow * a.splits : (int)(narrow < sms ? narrow : sms);
        e = M <= 16   ? launch_linear<16, false>(p, a, grid, st)
            : M <= 32 ? launch_linear<32, false>(p, a, grid, st)
            : M <= 64 ? launch_linear<64, false>(p, a, grid, st)
                      : launch_linear<128, false>(p, a, grid, st);
    }
    return e == cudaSuccess ? COTTUS_OK : cuda_fail(e);
}
