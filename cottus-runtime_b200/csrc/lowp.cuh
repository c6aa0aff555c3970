// Building blocks of the norm, 8-bit and sampling kernels: bf16 and e4m3
// conversions, group scales, host-side argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <string>
#include <type_traits>

#include "common.cuh"
#include "cottus_b200.h"

namespace cb200 {

int set_error(int code, const std::string& msg);

constexpr float kE4m3Max = 448.f;           // largest finite e4m3 value
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126: the scale of an all-zero group

template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x) { return from_f32<T>(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ uint32_t pack_bf2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
}

// Eight consecutive elements that this kernel reads once (no L1 allocation;
// a plain coherent load, so the buffer may be the kernel's output as well).
__device__ __forceinline__ uint4 ld_once(const void* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}
// (32-byte aligned: one access of 32 bytes per lane; two of 16, 32 bytes apart
// from lane to lane, pass through L1 twice)
__device__ __forceinline__ void load8_stream(const float* p, float (&v)[8]) {
    asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p));
}
__device__ __forceinline__ void load8_kept(const float* p, float (&v)[8]) {
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "l"(p));
}
__device__ __forceinline__ void store8_wide(float* p, const float (&v)[8]) {
    asm volatile("st.global.v8.f32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
                 "f"(v[5]), "f"(v[6]), "f"(v[7]), "l"(p)
                 : "memory");
}
__device__ __forceinline__ void load8_stream(const __half* p, float (&v)[8]) {
    const uint4 r = ld_once(p);
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = h2_to_f2(u[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void load8_stream(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 r = ld_once(p);
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a bf16 is the upper half of an fp32
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
}

// Maximum that keeps a NaN of either side.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = max_nan(m, fabsf(v[j]));
    return m;
}
// Eight elements in their own type.
template <typename XT>
struct Vec8 {
    union {
        uint4 u[sizeof(XT) / 2];
        uint16_t h[8 * sizeof(XT) / 2];
        uint32_t w[8 * sizeof(XT) / 4];
    };
    __device__ __forceinline__ Vec8() {}
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(XT) / 2; ++i) u[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const XT* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(XT) / 2; ++i) u[i] = ld_once(reinterpret_cast<const uint4*>(p) + i);
    }
    __device__ __forceinline__ void set(int j, XT x) {
        if constexpr (sizeof(XT) == 4) w[j] = __float_as_uint(to_f32(x));
        else h[j] = *reinterpret_cast<uint16_t*>(&x);
    }
    // Largest magnitude (NaN kept); two 16-bit values per operation.
    __device__ __forceinline__ float amax() const {
        if constexpr (sizeof(XT) == 4) {
            float v[8];
            get(v);
            return amax8(v);
        } else {
            const uint32_t m = max2_abs(max2_abs(w[0], w[1]), max2_abs(w[2], w[3]));
            return max_nan(fabsf(to_f32(half_of(m))), fabsf(to_f32(half_of(m >> 16))));
        }
    }
    __device__ __forceinline__ static XT half_of(uint32_t x) {
        const uint16_t b = (uint16_t)x;
        return *reinterpret_cast<const XT*>(&b);
    }
    // (with the product's sign)
    __device__ __forceinline__ static uint32_t max2_abs(uint32_t a, uint32_t b) {
        uint32_t r;
        if constexpr (std::is_same<XT, __half>::value) asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (sizeof(XT) == 4) v[j] = __uint_as_float(w[j]);
            else v[j] = to_f32(*reinterpret_cast<const XT*>(&h[j]));
        }
    }
};

// Maximum over each half of the warp (all 32 lanes take part).
__device__ __forceinline__ float amax16(float m) {
#pragma unroll
    for (int o = 8; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
// max(amax / 448, 2^-126), the quotient correctly rounded as below (what a
// subnormal remainder would spoil is under the smallest scale anyway).
__device__ __forceinline__ float group_scale(float amax) {
    constexpr float r = 1.f / kE4m3Max;
    const float q0 = amax * r;
    const float q = fmaf(fmaf(-q0, kE4m3Max, amax), r, q0);
    return amax < INFINITY ? fmaxf(q, kMinScale) : amax;
}

// value / scale in e4m3, to nearest even, magnitudes above 448 to 448, NaN kept.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Division by a group's scale.  The quotients are correctly rounded: with
// r = RN(1/s), q0 = RN(v r) is within an ulp, and q0 + RN(v - q0 s) r is then
// RN(v / s) (Markstein, IBM J. Res. Dev. 34, 1990) while nothing underflows:
// v below 2^-10 s is 0 in e4m3 whatever its last bit, and for larger v the
// remainder stays a normal number where s >= 2^-90.  Smaller, infinite and NaN
// scales divide.  (With divisions the 28672 x 8200 bf16 weight took 272 us.)
struct Divisor {
    float s, r;
    bool plain;
    __device__ __forceinline__ explicit Divisor(float scale) : s(scale), r(0.f), plain(scale >= 0x1p-90f && scale < INFINITY) {
        if (plain) r = __frcp_rn(scale);
    }
};
__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], const Divisor& d) {
    float q[8];
    if (d.plain) {
        // (two at a time: the 28672 x 8200 weight takes 133 us, one by one 146)
        const float2 r2 = make_float2(d.r, d.r), ns2 = make_float2(-d.s, -d.s);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float2 x = make_float2(v[j], v[j + 1]);
            const float2 q0 = fmul2(x, r2);
            const float2 q1 = ffma2(ffma2(q0, ns2, x), r2, q0);
            q[j] = q1.x;
            q[j + 1] = q1.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = __fdiv_rn(v[j], d.s);
    }
    uint2 o;
    o.x = e4m3x2(q[0], q[1]) | (e4m3x2(q[2], q[3]) << 16);
    o.y = e4m3x2(q[4], q[5]) | (e4m3x2(q[6], q[7]) << 16);
    return o;
}
// Four or eight values times the reciprocal of their group's scale: for values that
// are rounded themselves, as a norm's are, where the quotient's last fp32 bit
// is below their own error.
__device__ __forceinline__ uint32_t e4m3x4_times(const float (&v)[4], const Divisor& d) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = d.plain ? v[j] * d.r : __fdiv_rn(v[j], d.s);
    return e4m3x2(q[0], q[1]) | (e4m3x2(q[2], q[3]) << 16);
}
__device__ __forceinline__ uint2 e4m3x8_times(const float (&v)[8], const Divisor& d) {
    if (!d.plain) return e4m3x8(v, d);
    uint2 o;
    o.x = e4m3x2(v[0] * d.r, v[1] * d.r) | (e4m3x2(v[2] * d.r, v[3] * d.r) << 16);
    o.y = e4m3x2(v[4] * d.r, v[5] * d.r) | (e4m3x2(v[6] * d.r, v[7] * d.r) << 16);
    return o;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr int kMaxWidth = 1 << 30;  // of a matrix: the kernels round 32-bit columns up to whole tiles
inline bool lowp_input_dtype(int32_t t) { return t == COTTUS_F32 || t == COTTUS_F16 || t == COTTUS_BF16; }
inline int dtype_bytes(int32_t t) { return t == COTTUS_F32 ? 4 : (t == COTTUS_E4M3 ? 1 : 2); }
inline bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

struct Span {
    const void* p;
    size_t bytes;
};
inline bool overlap(const Span& a, const Span& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
}

// Launch that may start while the stream's preceding kernel drains: the
// kernel calls grid_dependency_wait() before it touches global memory, and
// only then grid_dependents_launch(), so that whatever follows starts after
// everything before this kernel is complete.  This kernel itself is not: what a
// follower does before its own wait is hints (prefetches into L2), no reads.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                              Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

}  // namespace cb200
