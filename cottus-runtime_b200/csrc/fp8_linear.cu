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
// each) and then added, scaled, to fp32 sums in registers.  CTA tile: 128
// rows of x (the MMA's M) by BN rows of the weight (its N).  A row of x is a
// TMEM lane, so a thread's scale is one number for its whole run of columns:
// one fused multiply-add per element and group.
//
//   warps 0-7   the sums: warp w reads TMEM lanes 32 (w mod 4) .. + 31,
//               columns BN/2 (w / 4) .. + BN/2
//   warp 8      TMA producer (one thread): ring of stages, one group per stage
//   warp 9      TMEM allocation and MMA issue (one thread)
//
// TMEM holds 512 / BN product buffers, so the tensor cores work on the next
// groups while a finished one is being added up.
//
// A decode batch (rows <= 128) reads the weight once and is bound by HBM.
// Where the weight has fewer tiles than the GPU has SMs, `splits` CTAs of one
// cluster share a tile: each takes a contiguous run of groups, and the
// partial sums meet in distributed shared memory, added in rank order, so a
// result does not depend on timing.  Only the rows that exist are fetched
// (the TMA box is as high as the batch, rounded up to 8); the remaining MMA
// lanes read whatever follows in the same stage and their results are never
// stored.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <string>

#include "common.cuh"
#include "cottus_b200.h"
#include "internal.h"
#include "lowp.cuh"

namespace cb200 {
CUtensorMap make_tensor_map_2d_u8(const void* base, uint64_t inner, uint64_t outer, uint64_t pitch_bytes,
                                  uint32_t box_inner, uint32_t box_outer, bool swizzle128, cudaError_t* err);
int device_sm_count(int device);

namespace {

constexpr int kBM = 128;        // rows of x per tile
constexpr int kBK = 128;        // elements (bytes) of k per stage: one scale group
constexpr int kSumWarps = 8;    // warps that add up the groups
constexpr int kThreads = (kSumWarps + 4) * 32;  // and one warpgroup for the producer and the MMA issue
// Registers per thread of the wide tile after the launch's even split: the
// sums (128 per thread) take what the producer's warpgroup gives back.  The
// launch must have brought that many (checked on the host).
constexpr int kSumRegs = 232, kCtrlRegs = 40;
constexpr int kMinLaunchRegs = (kSumRegs * kSumWarps * 32 + kCtrlRegs * 128 + kThreads - 1) / kThreads;
constexpr int kMaxStages = 12;
constexpr int kMaxSplits = 8;   // portable cluster size
constexpr int kStagePitch = 20; // words per staged row of 16 columns (conflict-free 16-byte accesses)
constexpr uint32_t kTmemCols = 512;
constexpr size_t kSmemMax = 232448;  // dynamic shared memory per CTA, 227 KB

struct LinArgs {
    const float* xs;
    const float* ws;
    const float* residual;
    void* out;
    uint32_t* status;
    int M, N, groups, m_tiles, n_tiles, splits, stages, x_rows, out_dtype;
    int vec;  // rows of out and residual start on 16 bytes and hold whole runs of 4
};

__device__ __forceinline__ uint64_t sw128_kmajor_desc(uint32_t smem_byte_addr) {
    // K-major tile of 128-byte rows, 128B swizzle, 8-row groups 1024 bytes apart
    return (uint64_t)((smem_byte_addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f8f6f4: e4m3 A and B (format 0), fp32 accumulator, both K-major.
template <int BN>
constexpr uint32_t f8_idesc() {
    return (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
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
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// 16 bytes of CTA `rank`'s shared memory at this CTA's address `local`.
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t local, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t local, uint32_t rank) {
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
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

template <int BN>
constexpr size_t lin_tail_bytes() {  // staging rows and barriers behind the ring
    return (size_t)kSumWarps * 32 * kStagePitch * 4 + (2 * kMaxStages + 2 * (kTmemCols / BN) + 1) * 8 + 8;
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) fp8_linear_kernel(const __grid_constant__ CUtensorMap xmap,
                                                                 const __grid_constant__ CUtensorMap wmap,
                                                                 const LinArgs a) {
    constexpr int HALF = BN / 2, NBUF = kTmemCols / BN, PART_PITCH = BN + 4;
    constexpr bool SPLIT = BN == 128;  // the wide tile is for products with tiles enough
    const int splits = SPLIT ? a.splits : 1;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int stage_bytes = (a.x_rows + BN) * kBK;
    float* staging = reinterpret_cast<float*>(smem + (size_t)a.stages * stage_bytes);
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + kSumWarps * 32 * kStagePitch);
    uint64_t* empty = full + kMaxStages;
    uint64_t* tm_full = empty + kMaxStages;
    uint64_t* tm_empty = tm_full + NBUF;
    uint64_t* done = tm_empty + NBUF;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(done + 1);
    uint32_t* s_failed = s_tmem + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = splits > 1 ? (int)cluster_rank() : 0;
    const int first = blockIdx.x / splits, step = gridDim.x / splits;
    const int tiles = a.m_tiles * a.n_tiles;
    // this CTA's groups of every tile it works on
    const int g0 = (int)((long long)a.groups * rank / splits), g1 = (int)((long long)a.groups * (rank + 1) / splits);

    if (threadIdx.x == 0) {
        prefetch_tensormap(&xmap);
        prefetch_tensormap(&wmap);
        for (int i = 0; i < a.stages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < NBUF; ++i) {
            mbar_init(&tm_full[i], 1);
            mbar_init(&tm_empty[i], kSumWarps);
        }
        mbar_init(done, 1);
        fence_barrier_init();
        *s_failed = 0;
    }
    if (warp == kSumWarps + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(s_tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *s_tmem;
    grid_dependency_wait();
    // (after the allocation above: a dependent that also allocates TMEM can
    // then only wait for this grid, never the other way round)
    grid_dependents_launch();

    bool ok = true;
    if (warp >= kSumWarps) {
    if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtrlRegs));
    if (warp == kSumWarps) {
        if (lane == 0) {
            // ---- producer ------------------------------------------------
            Ring r;
            int issued = 0;
            for (int t = first; t < tiles && ok; t += step) {
                const int m0 = (t % a.m_tiles) * kBM, n0 = (t / a.m_tiles) * BN;
                for (int g = g0; g < g1; ++g) {
                    if (!mbar_wait_bounded(&empty[r.slot], r.phase ^ 1)) {
                        ok = false;
                        break;
                    }
                    uint8_t* st = smem + (size_t)r.slot * stage_bytes;
                    mbar_arrive_expect_tx(&full[r.slot], (uint32_t)stage_bytes);
                    tma_load_2d(st, &xmap, &full[r.slot], g * kBK, m0);
                    tma_load_2d(st + a.x_rows * kBK, &wmap, &full[r.slot], g * kBK, n0);
                    ++issued;
                    r.next(a.stages);
                }
            }
            if (!ok) {
                // let this CTA's copies in flight land before it gives up
                Ring q = r;
                for (int i = 0; i < a.stages && i < issued; ++i) {
                    if (q.slot == 0) {
                        q.slot = a.stages;
                        q.phase ^= 1;
                    }
                    --q.slot;
                    (void)mbar_wait_bounded(&full[q.slot], q.phase);
                }
                *s_failed = 1;
            }
        }
    } else if (warp == kSumWarps + 1) {
        if (lane == 0) {
            // ---- MMA issue -----------------------------------------------
            constexpr uint32_t idesc = f8_idesc<BN>();
            Ring r, b;
            for (int t = first; t < tiles && ok; t += step) {
                for (int g = g0; g < g1; ++g) {
                    if (!mbar_wait_bounded(&tm_empty[b.slot], b.phase ^ 1) || !mbar_wait_bounded(&full[r.slot], r.phase)) {
                        ok = false;
                        break;
                    }
                    tc_after();
                    const uint32_t xa = smem_addr(smem + (size_t)r.slot * stage_bytes), wa = xa + a.x_rows * kBK;
#pragma unroll
                    for (int kk = 0; kk < kBK / 32; ++kk) {
                        const uint64_t ad = sw128_kmajor_desc(xa + kk * 32), bd = sw128_kmajor_desc(wa + kk * 32);
                        asm volatile(
                            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(
                                tmem + (uint32_t)(b.slot * BN)),
                            "l"(ad), "l"(bd), "r"(idesc), "r"((uint32_t)kk)
                            : "memory");
                    }
                    mma_commit(&empty[r.slot]);
                    mma_commit(&tm_full[b.slot]);
                    r.next(a.stages);
                    b.next(NBUF);
                }
            }
            if (!ok) {
                // every multiply issued so far ends before the memory is given back
                mma_commit(done);
                (void)mbar_wait_bounded(done, 0);
                *s_failed = 1;
            }
        }
    }
    } else {
        if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
        // ---- sums ----------------------------------------------------------
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * HALF);
        float* stg = staging + warp * 32 * kStagePitch;
        Ring b;
        for (int t = first; t < tiles && ok; t += step) {
            const int m0 = (t % a.m_tiles) * kBM, n0 = (t / a.m_tiles) * BN;
            const int m = m0 + quad * 32 + lane, nh = n0 + half * HALF;
            const bool rows_live = m0 + quad * 32 < a.M;  // (uniform in the warp)
            const float* xs = a.xs + (m < a.M ? m : 0);
            const float* ws = a.ws + (size_t)((nh < a.N ? nh : 0) / 128) * a.groups;
            float acc[HALF];
#pragma unroll
            for (int c = 0; c < HALF; ++c) acc[c] = 0.f;
            float sx = g0 < g1 ? xs[(size_t)g0 * a.M] : 0.f, sw = g0 < g1 ? ws[g0] : 0.f;
            for (int g = g0; g < g1; ++g) {
                const float s = sx * sw;
                if (g + 1 < g1) {
                    sx = xs[(size_t)(g + 1) * a.M];
                    sw = ws[g + 1];
                }
                ok = ok && mbar_wait_bounded(&tm_full[b.slot], b.phase);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_after();
                if (rows_live) {
#pragma unroll
                    for (int c0 = 0; c0 < HALF; c0 += 32) {
                        uint32_t v[32];
                        tmem_ld32(taddr + (uint32_t)(b.slot * BN + c0), v);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) acc[c0 + c] = fmaf(s, __uint_as_float(v[c]), acc[c0 + c]);
                    }
                }
                tc_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&tm_empty[b.slot]);
                b.next(NBUF);
            }
            if (!ok) break;
            if (splits > 1) {
                // the only tile of this cluster: its ring is idle (every stage
                // has been multiplied), so it takes the partial sums
                float* part = reinterpret_cast<float*>(smem) + (size_t)(quad * 32 + lane) * PART_PITCH + half * HALF;
                if (m < a.M) {
#pragma unroll
                    for (int c = 0; c < HALF; c += 4)
                        *reinterpret_cast<float4*>(part + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
                }
            } else if (rows_live) {
                // 16 columns at a time through shared memory, so that four
                // lanes store (and read the residual of) one run of a row
#pragma unroll
                for (int c0 = 0; c0 < HALF; c0 += 16) {
                    __syncwarp();
#pragma unroll
                    for (int c = 0; c < 16; c += 4)
                        *reinterpret_cast<float4*>(stg + lane * kStagePitch + c) =
                            make_float4(acc[c0 + c], acc[c0 + c + 1], acc[c0 + c + 2], acc[c0 + c + 3]);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = i * 8 + (lane >> 2), mm = m0 + quad * 32 + rr, n = nh + c0 + (lane & 3) * 4;
                        const float4 v = *reinterpret_cast<const float4*>(stg + rr * kStagePitch + (lane & 3) * 4);
                        if (mm < a.M && n < a.N) store_out4(a, mm, n, v);
                    }
                }
            }
        }
        if (!ok && lane == 0) *s_failed = 1;
    }
    __syncwarp();
    if (splits > 1) {
        cluster_sync_all();  // every CTA's partial sums are in its shared memory
        const int m0 = (first % a.m_tiles) * kBM, n0 = (first / a.m_tiles) * BN;
        const int rows = a.M - m0 < kBM ? a.M - m0 : kBM;
        uint32_t failed = 0;
        for (int q = 0; q < splits; ++q) failed |= ld_cluster_u32(smem_addr(s_failed), q);
        if (!failed) {
            for (int i = rank * kThreads + threadIdx.x; i < rows * (BN / 4); i += splits * kThreads) {
                const int r = i / (BN / 4), c = (i % (BN / 4)) * 4;
                if (n0 + c >= a.N) continue;
                const uint32_t at = smem_addr(reinterpret_cast<float*>(smem) + (size_t)r * PART_PITCH + c);
                float4 p[kMaxSplits];
#pragma unroll
                for (int q = 0; q < kMaxSplits; ++q)
                    if (q < splits) p[q] = ld_cluster_f4(at, q);
                float4 v = p[0];
#pragma unroll
                for (int q = 1; q < kMaxSplits; ++q)
                    if (q < splits) {
                        v.x += p[q].x;
                        v.y += p[q].y;
                        v.z += p[q].z;
                        v.w += p[q].w;
                    }
                store_out4(a, m0 + r, n0 + c, v);
            }
        }
        cluster_sync_all();  // nobody leaves while its shared memory is being read
    }
    tc_before();
    __syncthreads();
    if (threadIdx.x == 0 && *s_failed) report(a.status, COTTUS_STATUS_TIMEOUT);
    if (warp == kSumWarps + 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

int fail(int code, const std::string& msg) { return set_error(code, msg); }

// Once per device: the shared-memory limit, and the register count that the
// wide tile's redistribution relies on.
template <int BN>
cudaError_t prepare_kernel() {
    static std::atomic<uint64_t> ready{0};  // a bit per device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (ready.load(std::memory_order_acquire) >> dev & 1)) return cudaSuccess;
    auto kern = fp8_linear_kernel<BN>;
    cudaFuncAttributes fa = {};
    e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return e;
    if (BN == 256 && fa.numRegs < kMinLaunchRegs) return cudaErrorInvalidConfiguration;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax);
    if (e == cudaSuccess && dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    return e;
}

template <int BN>
cudaError_t launch_linear(const cottus_fp8_linear_params* p, LinArgs a, int grid, cudaStream_t st) {
    cudaError_t err = cudaSuccess;
    a.x_rows = p->rows < kBM ? (p->rows + 7) / 8 * 8 : kBM;
    const size_t stage = (size_t)(a.x_rows + BN) * kBK;
    const size_t room = kSmemMax - 1024 - lin_tail_bytes<BN>();
    a.stages = (int)(room / stage);
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    const CUtensorMap xmap = make_tensor_map_2d_u8(p->x, p->in_features, p->rows, p->in_features, kBK, a.x_rows, true, &err);
    if (err != cudaSuccess) return err;
    const CUtensorMap wmap = make_tensor_map_2d_u8(p->weight, p->in_features, p->out_features, p->in_features, kBK, BN,
                                                   true, &err);
    if (err != cudaSuccess) return err;
    auto kern = fp8_linear_kernel<BN>;
    const size_t smem = (size_t)a.stages * stage + lin_tail_bytes<BN>() + 1024;
    err = prepare_kernel<BN>();
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.splits > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, xmap, wmap, a);
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
    a.out_dtype = p->out_dtype;
    a.vec = N % 4 == 0 && aligned(p->out, es * 4) && aligned(p->residual, 16);
    a.m_tiles = (M + kBM - 1) / kBM;
    int dev = 0;
    cudaGetDevice(&dev);
    const int sms = device_sm_count(dev);
    const int n256 = (N + 255) / 256, n128 = (N + 127) / 128;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    cudaError_t e;
    if ((long long)a.m_tiles * n128 >= (int64_t(1) << 30)) return fail(COTTUS_ERR_UNSUPPORTED, "product too large");
    if (a.m_tiles > 1 && (long long)a.m_tiles * n256 >= sms) {
        // enough tiles for every SM: the wide tile reads a third less shared memory per multiply
        a.n_tiles = n256;
        a.splits = 1;
        const int tiles = a.m_tiles * n256;
        e = launch_linear<256>(p, a, tiles < sms ? tiles : sms, st);
    } else {
        a.n_tiles = n128;
        const int tiles = a.m_tiles * n128;
        int s = tiles < sms ? sms / tiles : 1;
        if (s > kMaxSplits) s = kMaxSplits;
        if (s > groups) s = groups;
        a.splits = s;
        e = launch_linear<128>(p, a, s > 1 ? tiles * s : (tiles < sms ? tiles : sms), st);
    }
    return e == cudaSuccess ? COTTUS_OK : fail(COTTUS_ERR_CUDA, std::string("CUDA error: ") + cudaGetErrorString(e));
}
