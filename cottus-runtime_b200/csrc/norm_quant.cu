// RMS norm with the residual's addition, and quantisation to e4m3 with one
// scale per 128 values.  Replaces residualAddCUDA + rmsnormCUDA
// (compute_primitives_cuda.cu:58-89), whose every thread sums the whole row.
//
//   h = x (+ r);  y = h * (mean(h^2) + eps)^(-1/2) * g
//   s = max(amax_128 |y| / 448, 2^-126);  q = e4m3(y / s)
//
// Both only move bytes (a few operations per element), so HBM bounds them at
// many rows and the latency of one load, one block reduction and one store at
// few.  Each input is read once: a row stays in registers between the sum of
// squares and the output.  Eight consecutive elements per thread and step
// (16 bytes of a 16-bit type), so that 16 neighbouring lanes hold one group
// of 128 and its amax is four shuffles.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <string>

#include "common.cuh"
#include "cottus_b200.h"
#include "internal.h"
#include "lowp.cuh"

namespace cb200 {
int device_sm_count(int device);

namespace {

struct NormArgs {
    const void* x;
    const float* residual;
    float* residual_out;
    const float* weight;
    void* out;
    float* scales;
    long long rows;
    int hidden, out_dtype;
    float eps;
};

// Sum over the block, the same value in every thread (fixed order).
__device__ __forceinline__ float block_sum(float v, float* smem) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) smem[warp] = v;
    __syncthreads();
    v = lane < warps ? smem[lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over a row whose vector t + i T has the sum s[i] in thread t: by 32
// neighbouring vectors, then over those, so that it does not depend on V and T
// (a row comes out the same whatever the number of rows).
template <int V>
__device__ __forceinline__ float row_sum(float (&s)[V], float* smem, int nvec) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int o = 16; o; o >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
        if (lane == 0) smem[i * warps + warp] = s[i];
    }
    __syncthreads();
    const int blocks = (nvec + 31) >> 5;
    float v = 0.f;  // (at most 1024 threads: 32 V such sums)
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (lane + i * 32 < blocks) v += smem[lane + i * 32];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ void store_out8(void* out, int dtype, size_t e, const float (&y)[8]) {
    if (dtype == COTTUS_F32) store8_wide(reinterpret_cast<float*>(out) + e, y);
    else if (dtype == COTTUS_F16) store8(reinterpret_cast<__half*>(out) + e, y);
    else store8(reinterpret_cast<__nv_bfloat16*>(out) + e, y);
}
__device__ __forceinline__ void store_out1(void* out, int dtype, size_t e, float y) {
    if (dtype == COTTUS_F32) reinterpret_cast<float*>(out)[e] = y;
    else if (dtype == COTTUS_F16) reinterpret_cast<__half*>(out)[e] = __float2half_rn(y);
    else reinterpret_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(y);
}

// Threads per CTA at most (with 1024 a thread has up to 64 registers).
template <int V>
constexpr int kNormThreads = V == 2 ? 768 : 1024;

// One CTA per row, the row in registers: thread t holds the vectors of eight
// t, t + T, ... (V of them).  hidden a multiple of 8, rows 32-byte aligned in
// fp32 and 16-byte aligned in 16 bits.
template <typename XT, int V>
__global__ void __launch_bounds__(kNormThreads<V>) rms_norm_vec_kernel(const NormArgs a) {
    __shared__ float red[128];  // (one per 32 vectors of up to 4096)
    const int nvec = a.hidden >> 3, T = blockDim.x;
    const long long row = blockIdx.x;
    const XT* x = reinterpret_cast<const XT*>(a.x) + row * a.hidden;
    grid_dependency_wait();
    grid_dependents_launch();
    float h[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = threadIdx.x + i * T;
        if (v < nvec) load8_stream(x + v * 8, h[i]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
    }
    if (a.residual) {
        const float* r = a.residual + row * a.hidden;
        float* ro = a.residual_out + row * a.hidden;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int v = threadIdx.x + i * T;
            if (v < nvec) {
                float t[8];
                load8_stream(r + v * 8, t);
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] += t[j];
                store8_wide(ro + v * 8, h[i]);
            }
        }
    }
    float part[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        part[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) part[i] = fmaf(h[i][j], h[i][j], part[i]);
    }
    const float ss = row_sum<V>(part, red, nvec);
    const float inv = __frsqrt_rn(__fdiv_rn(ss, (float)a.hidden) + a.eps);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = threadIdx.x + i * T;
        const bool live = v < nvec;
        float w[8];
        if (live) load8_kept(a.weight + v * 8, w);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = live ? h[i][j] * inv * w[j] : 0.f;
        const size_t e = (size_t)row * a.hidden + v * 8;
        if (a.out_dtype != COTTUS_E4M3) {
            if (live) store_out8(a.out, a.out_dtype, e, h[i]);
            continue;
        }
        const float s = group_scale(amax16(amax8(h[i])));
        if (live) {
            *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(a.out) + e) = e4m3x8_times(h[i], Divisor(s));
            if ((v & 15) == 0) a.scales[(size_t)(v >> 4) * a.rows + row] = s;
        }
    }
}

// Any width up to 16384 and any alignment: one CTA per row, G groups of 128 per
// warp, the row in registers, four elements per lane and group (a warp reads 32
// consecutive ones at a time).
template <typename XT, int G>
__global__ void __launch_bounds__(G == 1 ? 512 : 1024) rms_norm_elem_kernel(const NormArgs a) {
    __shared__ float red[32];
    const long long row = blockIdx.x;
    const size_t base = (size_t)row * a.hidden;
    const XT* x = reinterpret_cast<const XT*>(a.x) + base;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    grid_dependency_wait();
    grid_dependents_launch();
    // (element j of group g of this lane)
    auto index = [&](int g, int j) { return (warp + g * warps) * 128 + j * 32 + lane; };
    float h[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) h[g][j] = index(g, j) < a.hidden ? to_f32(x[index(g, j)]) : 0.f;
    if (a.residual) {
        const float* r = a.residual + base;
        float* ro = a.residual_out + base;
        float t[G][4];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[g][j] = index(g, j) < a.hidden ? r[index(g, j)] : 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h[g][j] += t[g][j];
                if (index(g, j) < a.hidden) ro[index(g, j)] = h[g][j];
            }
    }
    float ss = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(h[g][j], h[g][j], ss);
    ss = block_sum(ss, red);
    const float inv = __frsqrt_rn(__fdiv_rn(ss, (float)a.hidden) + a.eps);
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = index(g, j);
            h[g][j] = i < a.hidden ? h[g][j] * inv * a.weight[i] : 0.f;
            if (i < a.hidden && a.out_dtype != COTTUS_E4M3) store_out1(a.out, a.out_dtype, base + i, h[g][j]);
            m = max_nan(m, fabsf(h[g][j]));
        }
        if (a.out_dtype != COTTUS_E4M3) continue;
        m = amax16(m);
        const float s = group_scale(max_nan(m, __shfl_xor_sync(0xffffffffu, m, 16)));
        const uint32_t q = e4m3x4_times(h[g], Divisor(s));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (index(g, j) < a.hidden) reinterpret_cast<uint8_t*>(a.out)[base + index(g, j)] = (uint8_t)(q >> (8 * j));
        if (lane == 0 && index(g, 0) < a.hidden) a.scales[(size_t)(warp + g * warps) * a.rows + row] = s;
    }
}

// Any width and alignment: one CTA per row, the row read twice (the second
// time from L1 or L2), one warp per group of 128.
template <typename XT>
__global__ void __launch_bounds__(512) rms_norm_any_kernel(const NormArgs a) {
    __shared__ float red[32];
    const long long row = blockIdx.x;
    const size_t base = (size_t)row * a.hidden;
    const XT* x = reinterpret_cast<const XT*>(a.x) + base;
    grid_dependency_wait();
    grid_dependents_launch();
    float ss = 0.f;
    for (int i = threadIdx.x; i < a.hidden; i += blockDim.x) {
        float h = to_f32(x[i]);
        if (a.residual) h += a.residual[base + i];
        ss = fmaf(h, h, ss);
    }
    ss = block_sum(ss, red);  // (its barrier: every read of the row above precedes every write below)
    const float inv = __frsqrt_rn(__fdiv_rn(ss, (float)a.hidden) + a.eps);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int groups = (a.hidden + 127) / 128;
    for (int g = warp; g < groups; g += warps) {
        float y[4];
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = g * 128 + j * 32 + lane;
            y[j] = 0.f;
            if (i < a.hidden) {
                float h = to_f32(x[i]);
                if (a.residual) {
                    h += a.residual[base + i];
                    a.residual_out[base + i] = h;
                }
                y[j] = h * inv * a.weight[i];
                if (a.out_dtype != COTTUS_E4M3) store_out1(a.out, a.out_dtype, base + i, y[j]);
            }
            m = max_nan(m, fabsf(y[j]));
        }
        if (a.out_dtype == COTTUS_E4M3) {
            const float s = group_scale(max_nan(amax16(m), __shfl_xor_sync(0xffffffffu, amax16(m), 16)));
            const uint32_t q = e4m3x4_times(y, Divisor(s));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = g * 128 + j * 32 + lane;
                if (i < a.hidden) reinterpret_cast<uint8_t*>(a.out)[base + i] = (uint8_t)(q >> (8 * j));
            }
            if (lane == 0) a.scales[(size_t)g * a.rows + row] = s;
        }
    }
}

template <typename XT>
cudaError_t launch_norm(const NormArgs& a, bool vec, cudaStream_t st) {
    // one row per CTA; the grid's x dimension holds any row count below 2^31
    if (!vec) {
        // 8192 x 4095, fp32 with residual to fp16: 79 us against 132 with the row
        // read twice; fp16 to e4m3 70 against 109; 64 x 8191 6.1 against 17.9
        const int groups = (a.hidden + 127) / 128;
        const dim3 rows((unsigned)a.rows);
        if (groups <= 16) return launch_pdl(rms_norm_elem_kernel<XT, 1>, rows, dim3(groups * 32), 0, st, a);
        if (groups <= 64) return launch_pdl(rms_norm_elem_kernel<XT, 2>, rows, dim3((groups + 1) / 2 * 32), 0, st, a);
        if (groups <= 128) return launch_pdl(rms_norm_elem_kernel<XT, 4>, rows, dim3((groups + 3) / 4 * 32), 0, st, a);
        const int want = (a.hidden + 31) / 32 * 32;
        return launch_pdl(rms_norm_any_kernel<XT>, dim3((unsigned)a.rows), dim3(want < 512 ? want : 512), 0, st, a);
    }
    const int nvec = a.hidden / 8;
    auto threads = [&](int V) { return ((nvec + V - 1) / V + 31) / 32 * 32; };
    const dim3 grid((unsigned)a.rows);
    // Vectors per thread (us, inputs in HBM).  One while every row has an SM to
    // itself (100 x 4096 fp16 + residual 3.1 against 3.9 with two, 100 x 8192 fp32
    // 3.4 : 3.5); beyond that two, so that several rows share an SM (16384 x 8192 bf16
    // + residual to e4m3 228 against 243 with one and 240 with four, 16384 x 4096 fp32
    // 80 : 82 : 81); four where a row is 2 bytes per element and there are many
    // (16384 x 8192 fp16 to e4m3 104 against 114 with two, 16384 x 2048 27.6 : 28.3;
    // 600 x 8192 7.9 : 7.1), or where more than 768 threads would share a barrier
    // (8192 x 16384 fp16 + residual 248 : 282).
    int dev = 0;
    cudaGetDevice(&dev);
    const long long sms = device_sm_count(dev);
    const bool thin = sizeof(XT) == 2 && !a.residual && a.rows > 8 * sms;
    if (nvec <= kNormThreads<1> && a.rows <= sms) return launch_pdl(rms_norm_vec_kernel<XT, 1>, grid, dim3(threads(1)), 0, st, a);
    if (nvec <= 2 * kNormThreads<2> && !thin) return launch_pdl(rms_norm_vec_kernel<XT, 2>, grid, dim3(threads(2)), 0, st, a);
    return launch_pdl(rms_norm_vec_kernel<XT, 4>, grid, dim3(threads(4)), 0, st, a);
}

// ---------------------------------------------------------------------------
// quantisation
// ---------------------------------------------------------------------------
struct QuantArgs {
    const void* x;
    uint8_t* out;
    float* scales;
    long long rows;
    int cols;
};

// Rows: half a warp per (row, group of 128), a CTA per 16 RT rows by GT groups.
// VEC (cols a multiple of 8, x 16-byte and out 8-byte aligned): eight elements
// per lane; else lanes take every 16th element.  With RT = GT = 2 every thread
// has four loads in flight and the scales of 32 rows, one run of the group-major
// array, leave together.
template <typename XT, bool VEC, int RT, int GT>
__global__ void __launch_bounds__(256) quant_rows_kernel(const QuantArgs a, const int group_tiles) {
    constexpr int U = RT * GT;
    const int groups = (a.cols + 127) / 128;
    const uint32_t tile = blockIdx.x / group_tiles;
    const int lane = threadIdx.x & 15;
    const long long row0 = (long long)tile * (16 * RT) + (threadIdx.x >> 4);
    const int g0 = (int)(blockIdx.x - tile * group_tiles) * GT;
    grid_dependency_wait();
    grid_dependents_launch();
    Vec8<XT> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long row = row0 + (u % RT) * 16;
        const int c0 = (g0 + u / RT) * 128, n = a.cols - c0 < 128 ? a.cols - c0 : 128;
        const XT* p = reinterpret_cast<const XT*>(a.x) + (size_t)row * a.cols + c0;
        x[u].clear();
        if (row >= a.rows) continue;
        if constexpr (VEC) {
            if (lane * 8 < n) x[u].load(p + lane * 8);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (lane + j * 16 < n) x[u].set(j, p[lane + j * 16]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long row = row0 + (u % RT) * 16;
        const int g = g0 + u / RT, c0 = g * 128, n = a.cols - c0 < 128 ? a.cols - c0 : 128;
        const float s = group_scale(amax16(x[u].amax()));  // (all lanes take part)
        if (row >= a.rows || g >= groups) continue;
        uint8_t* o = a.out + (size_t)row * a.cols + c0;
        const Divisor d(s);
        float v[8];
        x[u].get(v);
        if constexpr (VEC) {
            if (lane * 8 < n) *reinterpret_cast<uint2*>(o + lane * 8) = e4m3x8(v, d);
        } else {
            const uint2 q = e4m3x8(v, d);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (lane + j * 16 < n) o[lane + j * 16] = (uint8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
        }
        if (lane == 0) a.scales[(size_t)g * a.rows + row] = s;
    }
}

// Blocks: one CTA per 128 x 128 block, 32 elements per thread, kept as they
// were loaded (as fp32 they took 64 registers of 256 threads, 2 CTAs per SM and
// 2.4 TB/s).
template <typename XT, bool VEC>
__global__ void __launch_bounds__(512, sizeof(XT) == 4 ? 2 : 3) quant_blocks_kernel(const QuantArgs a) {
    __shared__ float red[16];
    constexpr int R = 4;
    const int cb = blockIdx.x, groups = gridDim.x;
    const long long rb = blockIdx.y;
    const int c0 = cb * 128;
    const int nc = a.cols - c0 < 128 ? a.cols - c0 : 128;
    const int lane = threadIdx.x & 15, r0 = threadIdx.x >> 4;
    grid_dependency_wait();
    grid_dependents_launch();
    Vec8<XT> x[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const long long row = rb * 128 + r0 + i * 32;
        const XT* p = reinterpret_cast<const XT*>(a.x) + (size_t)row * a.cols + c0;
        x[i].clear();
        if (row < a.rows) {
            if constexpr (VEC) {
                if (lane * 8 < nc) x[i].load(p + lane * 8);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (lane + j * 16 < nc) x[i].set(j, p[lane + j * 16]);
            }
        }
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) m = max_nan(m, x[i].amax());
    m = amax16(m);
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 16));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = amax16(red[lane]);
    const float s = group_scale(m);
    const Divisor d(s);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const long long row = rb * 128 + r0 + i * 32;
        if (row >= a.rows) continue;
        uint8_t* o = a.out + (size_t)row * a.cols + c0;
        float v[8];
        x[i].get(v);
        if constexpr (VEC) {
            if (lane * 8 < nc) *reinterpret_cast<uint2*>(o + lane * 8) = e4m3x8(v, d);
        } else {
            const uint2 q = e4m3x8(v, d);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (lane + j * 16 < nc) o[lane + j * 16] = (uint8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
        }
    }
    if (threadIdx.x == 0) a.scales[(size_t)rb * groups + cb] = s;
}

template <typename XT, bool VEC>
cudaError_t launch_quant(const QuantArgs& a, bool blocks, cudaStream_t st) {
    const long long groups = (a.cols + 127) / 128;
    if (blocks)
        return launch_pdl(quant_blocks_kernel<XT, VEC>, dim3((unsigned)groups, (unsigned)((a.rows + 127) / 128)),
                          dim3(512), 0, st, a);
    auto rows = [&](auto kern, int rt, int gt) {
        const long long tiles = (groups + gt - 1) / gt;
        return launch_pdl(kern, dim3((unsigned)((a.rows + 16 * rt - 1) / (16 * rt) * tiles)), dim3(256), 0, st, a, (int)tiles);
    };
    // four groups per thread once the small tiles fill the GPU's 8 CTAs per SM:
    // 16384 x 8192 fp16 78 us against 97, 64 x 4096 (128 small tiles) 2.0 against
    // 1.4.  Element by element they do not help (8192 x 8191 bf16 117 against 79).
    if constexpr (VEC) {
        int dev = 0;
        cudaGetDevice(&dev);
        if ((a.rows + 15) / 16 * groups >= 8LL * device_sm_count(dev)) return rows(quant_rows_kernel<XT, true, 2, 2>, 2, 2);
    }
    return rows(quant_rows_kernel<XT, VEC, 1, 1>, 1, 1);
}

int fail(int code, const std::string& msg) { return set_error(code, msg); }
int cuda_fail(cudaError_t e) { return fail(COTTUS_ERR_CUDA, std::string("CUDA error: ") + cudaGetErrorString(e)); }

}  // namespace
}  // namespace cb200

extern "C" {

int cottus_rms_norm(const cottus_rms_norm_params* p, cottus_stream_t stream) {
    using namespace cb200;
    if (!p) return fail(COTTUS_ERR_INVALID_ARGUMENT, "params must not be NULL");
    if (p->rows < 0 || p->hidden <= 0) return fail(COTTUS_ERR_INVALID_ARGUMENT, "rows must be non-negative and hidden positive");
    if (!lowp_input_dtype(p->x_dtype)) return fail(COTTUS_ERR_INVALID_ARGUMENT, "unknown x dtype");
    if (!lowp_input_dtype(p->out_dtype) && p->out_dtype != COTTUS_E4M3)
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "unknown out dtype");
    if (!(p->eps >= 0.f) || std::isinf(p->eps)) return fail(COTTUS_ERR_INVALID_ARGUMENT, "eps must be non-negative and finite");
    if (p->rows == 0) return COTTUS_OK;
    if (!p->x || !p->weight || !p->out) return fail(COTTUS_ERR_INVALID_ARGUMENT, "NULL pointer argument");
    if (!p->residual != !p->residual_out)
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "give both residual and residual_out or neither");
    if ((p->out_dtype == COTTUS_E4M3) != (p->scales != nullptr))
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "scales go with an e4m3 output, and only with one");
    if (p->rows >= (int64_t(1) << 31)) return fail(COTTUS_ERR_UNSUPPORTED, "too many rows for one launch");
    if (p->hidden > kMaxWidth) return fail(COTTUS_ERR_UNSUPPORTED, "hidden is too large");
    const size_t n = (size_t)p->rows * p->hidden;
    const int xs = dtype_bytes(p->x_dtype), os = dtype_bytes(p->out_dtype);
    const size_t sb = p->scales ? (size_t)p->rows * ((p->hidden + 127) / 128) * 4 : 0;
    const Span sx{p->x, n * xs}, sr{p->residual, p->residual ? n * 4 : 0}, sro{p->residual_out, p->residual ? n * 4 : 0},
        sw{p->weight, (size_t)p->hidden * 4}, so{p->out, n * os}, ss{p->scales, sb};
    if ((overlap(so, sx) && !(p->out == p->x && os == xs)) || overlap(so, sr) || overlap(so, sro) || overlap(so, sw) ||
        overlap(so, ss) || (overlap(sro, sr) && p->residual_out != p->residual) || overlap(sro, sx) ||
        overlap(sro, sw) || overlap(ss, sx) || overlap(ss, sr) || overlap(ss, sro) || overlap(ss, sw))
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "an output overlaps another buffer");
    if (!aligned(p->x, xs) || !aligned(p->out, os) || !aligned(p->residual, 4) || !aligned(p->residual_out, 4) ||
        !aligned(p->weight, 4) || !aligned(p->scales, 4))
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its element");
    NormArgs a;
    a.x = p->x;
    a.residual = p->residual;
    a.residual_out = p->residual_out;
    a.weight = p->weight;
    a.out = p->out;
    a.scales = p->scales;
    a.rows = p->rows;
    a.hidden = p->hidden;
    a.out_dtype = p->out_dtype;
    a.eps = p->eps;
    // the register kernel holds rows of up to 32768 elements (4 vectors of 8 per thread)
    // and takes eight of them at a time
    const bool vec = p->hidden % 8 == 0 && p->hidden <= 32768 && aligned(p->x, 8 * xs) && aligned(p->residual, 32) &&
                     aligned(p->residual_out, 32) && aligned(p->weight, 32) && aligned(p->out, 8 * os);
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = p->x_dtype == COTTUS_F32   ? launch_norm<float>(a, vec, st)
                          : p->x_dtype == COTTUS_F16 ? launch_norm<__half>(a, vec, st)
                                                     : launch_norm<__nv_bfloat16>(a, vec, st);
    return e == cudaSuccess ? COTTUS_OK : cuda_fail(e);
}

int cottus_quantize_fp8(const cottus_quantize_params* p, cottus_stream_t stream) {
    using namespace cb200;
    if (!p) return fail(COTTUS_ERR_INVALID_ARGUMENT, "params must not be NULL");
    if (p->rows < 0 || p->cols <= 0) return fail(COTTUS_ERR_INVALID_ARGUMENT, "rows must be non-negative and cols positive");
    if (!lowp_input_dtype(p->x_dtype)) return fail(COTTUS_ERR_INVALID_ARGUMENT, "unknown x dtype");
    if (p->block_rows != 1 && p->block_rows != 128) return fail(COTTUS_ERR_INVALID_ARGUMENT, "block_rows must be 1 or 128");
    if (p->rows == 0) return COTTUS_OK;
    if (!p->x || !p->out || !p->scales) return fail(COTTUS_ERR_INVALID_ARGUMENT, "NULL pointer argument");
    if (p->cols > kMaxWidth) return fail(COTTUS_ERR_UNSUPPORTED, "cols is too large");
    const bool blocks = p->block_rows == 128;
    const int64_t groups = (p->cols + 127) / 128, row_blocks = p->rows / 128 + (p->rows % 128 != 0);
    if (blocks ? row_blocks > 65535 : (p->rows >> 4) >= (int64_t(1) << 31) / groups - 1)
        return fail(COTTUS_ERR_UNSUPPORTED, "too many rows for one launch");
    const size_t n = (size_t)p->rows * p->cols;
    const int xs = dtype_bytes(p->x_dtype);
    const Span sx{p->x, n * xs}, so{p->out, n}, ss{p->scales, (size_t)((blocks ? row_blocks : p->rows) * groups) * 4};
    if (overlap(so, sx) || overlap(so, ss) || overlap(ss, sx))
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "an output overlaps another buffer");
    if (!aligned(p->x, xs) || !aligned(p->scales, 4))
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its element");
    QuantArgs a;
    a.x = p->x;
    a.out = static_cast<uint8_t*>(p->out);
    a.scales = p->scales;
    a.rows = p->rows;
    a.cols = p->cols;
    const bool vec = p->cols % 8 == 0 && aligned(p->x, 16) && aligned(p->out, 8);
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    auto run = [&](auto zero) {
        using XT = decltype(zero);
        return vec ? launch_quant<XT, true>(a, blocks, st) : launch_quant<XT, false>(a, blocks, st);
    };
    const cudaError_t e = p->x_dtype == COTTUS_F32   ? run(float{})
                          : p->x_dtype == COTTUS_F16 ? run(__half{})
                                                     : run(__nv_bfloat16{});
    return e == cudaSuccess ? COTTUS_OK : cuda_fail(e);
}

}  // extern "C"
