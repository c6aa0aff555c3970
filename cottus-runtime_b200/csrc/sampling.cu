// One token per row of logits: temperature, top-k, top-p and min-p, drawn
// with a given uniform number.  Replaces the device-to-host copy of the
// logits and the host argmax (engine.cpp:85-87).
//
// With the candidates ordered by (logit descending, index ascending) every
// filter keeps a prefix, so the kept set is { order key <= threshold } (and,
// for min-p, weight >= min_p, which is a prefix as well).  The order key of a
// logit is the 64-bit integer (descending image of its fp32 bits, index): all
// keys of a row differ, so ties need no special case.
//
// A row belongs to one thread-block cluster; each CTA holds a contiguous
// slice of it in shared memory and the row is read from HBM once.
//   1. the maximum, while the slice is loaded (greedy rows then look for its
//      first place and are done);
//   2. with top-k or top-p: a histogram (count, mass) of the distance to the
//      maximum, 128 bins per octave, merged over the cluster; the bin in
//      which the count or the mass passes its target; its few members are
//      gathered by the first CTA, sorted by key, and the threshold is read
//      off their prefix sums.  A bin with more members than the list holds is
//      first split by histograms of the key itself.  top_k up to 1024, and
//      top-p alone, start from a histogram of counts (an atomic per logit
//      where count and mass take four);
//   3. the kept mass per warp, each warp owning a contiguous run of indices,
//      then the one warp whose run holds uniform * mass walks it.
//
// Weights are 64-bit fixed point (43 to 47 fractional bits, so that a row's sum
// fits): integer sums do not depend on their order, so atomics leave no trace
// in the result.  exp is table-driven (P. Tang, ACM Trans. Math. Softw. 15,
// 1989): with y = (logit - max) log2(e) / T in two fp32 words and
// y = k + j / 256 + r, |r| <= 2^-9,  2^y = 2^k 2^(j/256) (1 + q(r)), the table
// exact to fixed point and the cubic q < 2^-9 in one fp32 word.  A weight is off
// by 2^-31 of itself (q's rounding to units of 2^-31 is half of that, the fp32
// roundings of r and q less than the other half) and by its last place, 2^-43
// or less of the largest.  (A vocabulary of 2^17 near-equal tokens then draws
// another token than exact arithmetic once in some 10^6 rows.)  exp in fp64
// took twice the time of everything else together; it serves the settings
// that fp32 words cannot hold (temperatures beyond 1e-6 or 1e6, infinities).
//
// Bounds: latency.  At one row (1 x 32000, all filters, 11 us) no phase has
// enough work to hide its own; by the clock of the first CTA: set-up and load
// 1.6 us with the first cluster barrier, the maximum 1.0, counting the distances
// and adding them up over the cluster 2.0, finding the bin 1.0, gathering 1.0,
// and by the first CTA alone two sorts 1.0 and the sums, cuts and the draw 1.9
// (four cluster barriers in all, 0.5 us each with its wait; top_k above 1024
// and top-p take more of them).  At many rows (256 x 50257 fp16, temperature
// alone, 39 us; 4 us of HBM) a CTA takes 14 us, 6 of them the exponentials
// beside those of the SM's other CTA, 2 the load, the rest the maximum, the sums
// and the walk; and the 512 CTAs are two waves of 296, the second part empty.
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
int device_sm_count(int device);

namespace {

using u64 = unsigned long long;

constexpr int kT = 512;        // threads per CTA
constexpr int kW = kT / 32;
constexpr int kBins = 1024;    // 8 octaves of distance to the maximum, 0.25 to 64
constexpr int kList = 2048;    // members of a bin that are sorted directly
constexpr int kMaxCluster = 8; // portable cluster size
constexpr u64 kNoKey = ~0ull;

struct SampleArgs {
    const void* logits;
    const float* uniforms;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* tokens;
    float* logprobs;
    uint32_t* status;
    int vocab, slice, raw_bytes, frac_bits;
};

constexpr int kDirect = 1024;  // largest top_k that one CTA finishes from the list
constexpr int kCountSort = 192;  // entries up to which a list is sorted by counting
constexpr int kTable = 256;    // 2^(j/256)

// Shared memory behind the slice.
struct Shared {
    u64 exp2_table[kTable];  // with 14 bits more than the weights
    uint32_t count[kBins];  // histogram: members,
    uint32_t limb[3][kBins];  // and their mass in limbs of limb_bits
    u64 list[kList];
    uint32_t mcnt[kBins];  // merged over the cluster
    u64 mmass[kBins];
    u64 wsum[kW];
    uint32_t wcnt[kW];
    u64 slot[3][kMaxCluster];  // one word from each CTA
    u64 res[4];                // broadcast by the first CTA
    u64 pick_mass;
    uint32_t pick_cnt, pick_in, pick_bin, list_n;
};

__device__ __forceinline__ void carrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cwait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void csync() {
    carrive();
    cwait();
}
__device__ __forceinline__ uint32_t mapa(const void* local, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(local)), "r"(rank));
    return a;
}
__device__ __forceinline__ void st_cluster(uint32_t a, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ld_cluster_u4(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t atom_add_cluster(uint32_t a, uint32_t v) {
    uint32_t r;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(a), "r"(v) : "memory");
    return r;
}
__device__ __forceinline__ u64 ld_cluster_u64(uint32_t a) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ u64 shfl_xor(u64 v, int o) { return __shfl_xor_sync(0xffffffffu, v, o); }
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ u64 warp_min(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const u64 w = shfl_xor(v, o);
        v = w < v ? w : v;
    }
    return v;
}
template <typename T>
__device__ __forceinline__ T warp_scan(T v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
    }
    return v;
}

// fp32 -> 32 bits whose unsigned order is descending value (-0 as +0), and back.
__device__ __forceinline__ uint32_t desc_bits(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return ~(b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u));
}
__device__ __forceinline__ float from_desc(uint32_t d) {
    const uint32_t k = ~d;
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ bool candidate(float x) { return x > -INFINITY; }  // false for -inf and NaN
__device__ __forceinline__ u64 order_key(float x, uint32_t index) { return ((u64)desc_bits(x) << 32) | index; }

// The weight of a logit, in units of 2^-frac.
struct Weight {
    float top;
    double inv_t;
    int frac;
    bool plain;       // fp32 words hold the exponent
    float c, cl;      // log2(e) / T in two words
    const u64* table;

    __device__ __forceinline__ void set(float max, float temperature, int frac_bits, const u64* exp2_table) {
        top = max;
        inv_t = 1.0 / (double)temperature;
        frac = frac_bits;
        const double cd = 1.4426950408889634 * inv_t;
        c = (float)cd;
        cl = (float)(cd - (double)c);
        plain = cd > 1e-6 && cd < 1e6 && fabsf(max) < 1e30f;
        table = exp2_table;
    }
    __device__ __forceinline__ double unit() const { return (double)(1ull << frac); }
    __device__ __forceinline__ double z(float x) const { return x == top ? 0.0 : ((double)x - (double)top) * inv_t; }
    __device__ __noinline__ u64 general(float x) const {
        if (x == top) return 1ull << frac;
        if (top == INFINITY || !candidate(x)) return 0;
        const double v = z(x);
        return v < -(frac + 2) * 0.6931471805599453 ? 0 : __double2ull_rn(exp(v) * unit());
    }
    __device__ __forceinline__ u64 operator()(float x) const { return plain ? fast(x) : general(x); }
    __device__ __forceinline__ u64 fast(float x) const { return fast(x, x).x; }
    // Of two logits (0 for -inf and NaN).  The arithmetic of both is packed, and
    // what is integer kept short: that pipe has half the rate, and bounds the
    // passes over all logits (25 such operations per logit before: 256 x 50257
    // fp16 without filters 44 us, so 38).
    struct Pair {
        u64 x, y;
    };
    __device__ __forceinline__ Pair fast(float x0, float x1) const {
        constexpr float magic = 12582912.f;  // 1.5 2^23: a float above it holds an integer in its low bits
        const float2 x = make_float2(x0, x1), one = make_float2(1.f, 1.f), minus = make_float2(-1.f, -1.f);
        const float2 tops = make_float2(top, top);
        // x - top = d + e exactly
        const float2 d = ffma2(tops, minus, x), b = ffma2(x, minus, d);
        const float2 e = ffma2(ffma2(b, one, tops), minus, ffma2(ffma2(b, minus, d), minus, x));
        // -y = -(d c) and what it leaves out
        const float2 cc = make_float2(c, c), ny = fmul2(d, make_float2(-c, -c));
        const float2 yl = ffma2(e, cc, ffma2(d, make_float2(cl, cl), ffma2(d, cc, ny)));
        // m = rint(256 y); from y = -64 on (or NaN) the shift below leaves nothing
        const float2 t = ffma2(make_float2(fminf(ny.x, 64.f), fminf(ny.y, 64.f)), make_float2(-256.f, -256.f),
                               make_float2(magic, magic));
        const float2 m = ffma2(t, one, make_float2(-magic, -magic));
        const float2 r = ffma2(ffma2(m, make_float2(1.f / 256.f, 1.f / 256.f), ny), minus, yl);
        // 2^r - 1 = sum (r ln 2)^i / i!, in units of 2^-31
        const float2 q = fmul2(r, ffma2(r, ffma2(r, make_float2(0.0555041087f, 0.0555041087f), make_float2(0.240226507f, 0.240226507f)),
                                        make_float2(0.693147181f, 0.693147181f)));
        const float2 qs = ffma2(q, make_float2(2147483648.f, 2147483648.f), make_float2(magic, magic));
        return {scaled(t.x, qs.x), scaled(t.y, qs.y)};
    }
    // 2^(m / 256) (1 + q) from the floats that hold m and q.
    __device__ __forceinline__ u64 scaled(float t, float qs) const {
        constexpr uint32_t magic = 0x4B400000u;
        const uint32_t m = __float_as_uint(t);
        const u64 p = table[m & (kTable - 1)];  // below 2^62, 13 bits more than 2^(j/256) has
        const u64 v = p + (u64)((long long)(int)(p >> 31) * (int)(__float_as_uint(qs) - magic));
        u64 w;  // (a shift by 64 or more is 0)
        asm("shr.u64 %0, %1, %2;" : "=l"(w) : "l"(v), "r"((14 + (magic >> 8)) - (m >> 8)));
        return w;
    }
};

// Level-one bin: monotone in the distance to the maximum.
__device__ __forceinline__ int distance_bin(float top, float x) {
    if (x == top) return 0;
    const int b = (int)(__float_as_uint(top - x) >> 16) - (125 << 7);
    return b < 0 ? 0 : (b < kBins ? b : kBins - 1);
}

// The bin's distances: at least near_edge, below far_edge (comparisons of
// the distance alone, for passes over all logits).
__device__ __forceinline__ float near_edge(int bin) { return bin <= 0 ? -INFINITY : __uint_as_float((uint32_t)(bin + (125 << 7)) << 16); }
__device__ __forceinline__ float far_edge(int bin) {
    return bin >= kBins - 1 ? INFINITY : __uint_as_float((uint32_t)(bin + 1 + (125 << 7)) << 16);
}
__device__ __forceinline__ float distance(float top, float x) { return x == top ? 0.f : top - x; }

template <typename XT>
struct Row {
    static constexpr int E = 16 / (int)sizeof(XT);  // logits per 16-byte vector
    Shared& s;
    const uint4* vec;  // the slice in shared memory, -inf before and behind it
    int lo, n;         // index of the first vector's first element; vectors
    int rank, size;    // of this CTA in the cluster
    int limb_bits;     // a slice's limbs add up within 32 bits
    Weight weight;

    __device__ __forceinline__ static void unpack(const uint4& u, float (&v)[E]) {
        const XT* x = reinterpret_cast<const XT*>(&u);
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] = to_f32(x[k]);
    }
    // f(logit, index) for every candidate of the slice
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int j = threadIdx.x; j < n; j += kT) {
            float v[E];
            unpack(vec[j], v);
#pragma unroll
            for (int k = 0; k < E; ++k)
                if (candidate(v[k])) f(v[k], lo + j * E + k);
        }
    }

    __device__ void clear_hist() const {
        for (int i = threadIdx.x; i < kBins; i += kT) {
            s.count[i] = 0;
            s.limb[0][i] = s.limb[1][i] = s.limb[2][i] = 0;
        }
        __syncthreads();
    }
    __device__ __forceinline__ void add(int bin, float v, bool mass) const {
        atomicAdd(&s.count[bin], 1u);
        if (mass) {
            const u64 w = weight(v);
            const uint32_t mask = (1u << limb_bits) - 1;
            atomicAdd(&s.limb[0][bin], (uint32_t)w & mask);
            atomicAdd(&s.limb[1][bin], (uint32_t)(w >> limb_bits) & mask);
            const uint32_t high = (uint32_t)(w >> (2 * limb_bits));
            if (high) atomicAdd(&s.limb[2][bin], high);  // (the likeliest few)
        }
    }
    // Adds the cluster's histograms up, every CTA for itself, into its mcnt /
    // mmass (four bins per thread).  The histogram may be cleared, or its words
    // used, after the next cluster barrier.  (Code that runs once costs its
    // way through the instruction caches first: with the loads of all CTAs
    // unrolled this took 20k cycles, so 10k.)
    __device__ void merge_hist() const {
        csync();
        constexpr int Q = kBins / 4;  // runs of four bins
        static_assert(2 * Q == kT, "half of the threads add counts and low limbs, half the others");
        const int b = (threadIdx.x % Q) * 4;
        const bool low = threadIdx.x < Q;
        const uint32_t* a0 = low ? &s.count[b] : &s.limb[1][b];
        const uint32_t* a1 = low ? &s.limb[0][b] : &s.limb[2][b];
        u64 cx[4] = {0, 0, 0, 0}, cy[4] = {0, 0, 0, 0};
#pragma unroll 2
        for (int q = 0; q < size; ++q) {
            const uint4 x = ld_cluster_u4(mapa(a0, q)), y = ld_cluster_u4(mapa(a1, q));
            cx[0] += x.x, cx[1] += x.y, cx[2] += x.z, cx[3] += x.w;
            cy[0] += y.x, cy[1] += y.y, cy[2] += y.z, cy[3] += y.w;
        }
        if (low) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s.mcnt[b + j] = (uint32_t)cx[j];
                s.mmass[b + j] = cy[j];
            }
        }
        __syncthreads();
        if (!low) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s.mmass[b + j] += (cx[j] << limb_bits) + (cy[j] << (2 * limb_bits));
        }
        __syncthreads();
    }

    struct Pick {
        int bin;  // kBins: none
        uint32_t before_cnt, in_cnt;
        u64 before_mass;
    };
    // The bin in which the running count reaches k (by_mass false) or the
    // running mass, on top of mass0, reaches t.
    __device__ Pick pick_bin(bool by_mass, uint32_t k, u64 mass0, double t) const {
        return pick_bin(by_mass, k, mass0, t, [&](int b) { return s.mcnt[b]; }, [&](int b) { return s.mmass[b]; });
    }
    template <typename FC, typename FM>
    __device__ __forceinline__ Pick pick_bin(bool by_mass, uint32_t k, u64 mass0, double t, FC cnt_of, FM mass_of) const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        constexpr int PER = kBins / kT;
        uint32_t c[PER], ctot = 0;
        u64 m[PER], mtot = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            ctot += c[j] = cnt_of(threadIdx.x * PER + j);
            mtot += m[j] = mass_of(threadIdx.x * PER + j);
        }
        uint32_t cb = warp_scan(ctot, lane);
        u64 mb = warp_scan(mtot, lane);
        __syncthreads();  // (earlier readers of these words are done)
        if (lane == 31) {
            s.wcnt[warp] = cb;
            s.wsum[warp] = mb;
        }
        if (threadIdx.x == 0) {
            s.pick_bin = kBins;
            s.pick_cnt = s.pick_in = 0;
            s.pick_mass = 0;
        }
        __syncthreads();
        const uint32_t cw = s.wcnt[lane % kW];
        const u64 mw = s.wsum[lane % kW];
        cb += __shfl_sync(0xffffffffu, warp_scan(cw, lane) - cw, warp) - ctot;
        mb += __shfl_sync(0xffffffffu, warp_scan(mw, lane) - mw, warp) - mtot + mass0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            // sums only grow, so one bin takes them past the target
            const bool here = by_mass ? (double)mb < t && (double)(mb + m[j]) >= t : cb < k && cb + c[j] >= k;
            if (here) {
                s.pick_bin = threadIdx.x * PER + j;
                s.pick_cnt = cb;
                s.pick_in = c[j];
                s.pick_mass = mb - mass0;
            }
            cb += c[j];
            mb += m[j];
        }
        __syncthreads();
        return {(int)s.pick_bin, s.pick_cnt, s.pick_in, s.pick_mass};
    }

    // Every CTA's count of each distance, added up by every CTA for itself into
    // its mcnt.  with_mass: mmass gets what the counts say of the masses, a
    // token weighing what the middle of its bin weighs (the maximum itself 1).
    __device__ void count_distances(bool with_mass) const {
        each([&](float v, int) { atomicAdd(&s.count[distance_bin(weight.top, v)], 1u); });
        csync();
#pragma unroll 1
        for (int b = threadIdx.x; b < kBins; b += kT) {
            uint32_t sum = 0;
#pragma unroll 4
            for (int q = 0; q < size; ++q) sum += ld_cluster(mapa(&s.count[b], q));
            s.mcnt[b] = sum;
            u64 m = 0;
            if (with_mass) {
                const float mid = b == 0 ? 0.125f : (b == kBins - 1 ? near_edge(b) : 0.5f * (near_edge(b) + far_edge(b)));
                const u64 w = weight.fast(weight.top - mid);
                m = b == 0 ? (u64)(sum - 1) * w + (1ull << weight.frac) : sum * w;
            }
            s.mmass[b] = m;
        }
        __syncthreads();
    }
    // The bins in which the running mass reaches (p - eps) and (p + eps) times
    // its end (0 and the last one, where it never does).
    __device__ void mass_range(float p, float eps, int& lo, int& hi) const {
        constexpr int PER = kBins / kT;
        u64 m[PER], own = 0, total;
#pragma unroll
        for (int j = 0; j < PER; ++j) own += m[j] = s.mmass[threadIdx.x * PER + j];
        if (threadIdx.x == 0) {
            s.pick_bin = 0;
            s.pick_in = kBins - 1;
        }
        u64 run = block_before(own, total);
        const double t0 = ((double)p - eps) * (double)total, t1 = ((double)p + eps) * (double)total;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const double a = (double)run, b = (double)(run + m[j]);
            if (a < t0 && b >= t0) s.pick_bin = threadIdx.x * PER + j;
            if (a < t1 && b >= t1) s.pick_in = threadIdx.x * PER + j;
            run += m[j];
        }
        __syncthreads();
        lo = (int)s.pick_bin;
        hi = (int)s.pick_in;
    }

    // Level one: the histogram of the distance to the maximum.
    __device__ void build_l1(bool mass) const {
        clear_hist();
        each([&](float v, int) { add(distance_bin(weight.top, v), v, mass); });
        merge_hist();
    }
    // The mass of all candidates, from the level-one histogram.
    __device__ u64 l1_mass() const {
        u64 m = 0;
        for (int b = threadIdx.x; b < kBins; b += kT) m += s.mmass[b];
        m = warp_sum(m);
        if ((threadIdx.x & 31) == 0) s.wsum[threadIdx.x >> 5] = m;
        __syncthreads();
        m = 0;
#pragma unroll 1
        for (int w = 0; w < kW; ++w) m += s.wsum[w];
        __syncthreads();
        return m;
    }

    // Sorts the first m entries of this CTA's list (all different), ascending.
    __device__ void sort_list(int m) const {
        if (m <= kCountSort) {
            // an entry's place is the number of smaller ones, counted by
            // kT / (m rounded up to a power of two) threads: no barrier until
            // the end (145 entries: 2k cycles, the bitonic network's 36 steps
            // 4k; the reads grow with m times the block, so 356 took 18k)
            int lg = 4;  // log2 of threads per entry, at most 16
            while (lg > 0 && (m << lg) > kT) --lg;
            const int e = threadIdx.x >> lg, part = threadIdx.x & ((1 << lg) - 1);
            const u64 key = e < m ? s.list[e] : kNoKey;
            uint32_t rank = 0;
#pragma unroll 4
            for (int j = part; j < m; j += 1 << lg) rank += s.list[j] < key;
            for (int o = 1; o < 1 << lg; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
            __syncthreads();
            if (e < m && part == 0) s.list[rank] = key;
            __syncthreads();
            return;
        }
        int pow2 = 2;
        while (pow2 < m) pow2 <<= 1;
        if (m <= kT) {
            // bitonic, an entry per thread; steps within a warp need no barrier
            u64 key = threadIdx.x < m ? s.list[threadIdx.x] : kNoKey;
            for (int w = 2; w <= pow2; w <<= 1)
                for (int j = w >> 1; j; j >>= 1) {
                    u64 other;
                    if (j < 32) {
                        other = shfl_xor(key, j);
                    } else {
                        __syncthreads();
                        s.list[threadIdx.x] = key;
                        __syncthreads();
                        other = s.list[threadIdx.x ^ j];
                    }
                    const bool small = ((threadIdx.x & j) == 0) == ((threadIdx.x & w) == 0);
                    key = small == (key < other) ? key : other;
                }
            __syncthreads();
            s.list[threadIdx.x] = key;
            __syncthreads();
            return;
        }
        for (int i = m + threadIdx.x; i < pow2; i += kT) s.list[i] = kNoKey;
        __syncthreads();
        for (int w = 2; w <= pow2; w <<= 1)
            for (int j = w >> 1; j; j >>= 1) {
                for (int i = threadIdx.x; i < pow2 / 2; i += kT) {
                    const int p0 = ((i & ~(j - 1)) << 1) | (i & (j - 1)), p1 = p0 | j;
                    const u64 u = s.list[p0], v = s.list[p1];
                    if ((u > v) == ((p0 & w) == 0)) {
                        s.list[p0] = v;
                        s.list[p1] = u;
                    }
                }
                __syncthreads();
            }
    }
    // Brings the entries of every CTA's list into this one's, behind its own
    // (kList in all at most); their number.
    __device__ int collect_lists() const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const uint32_t mine = lane < size ? ld_cluster(mapa(&s.list_n, lane)) : 0;
        const uint32_t upto = warp_scan(mine, lane);
        const uint32_t total = __shfl_sync(0xffffffffu, upto, 31);
        if (warp > 0 && warp < size) {  // (warp q copies CTA q's)
            const uint32_t m = __shfl_sync(0xffffffffu, mine, warp), at = __shfl_sync(0xffffffffu, upto, warp) - m;
            const uint32_t from = mapa(&s.list[0], warp);
#pragma unroll 4
            for (uint32_t i = lane; i < m; i += 32)
                if (at + i < (uint32_t)kList) s.list[at + i] = ld_cluster_u64(from + i * 8);
        }
        __syncthreads();
        return (int)(total < (uint32_t)kList ? total : (uint32_t)kList);
    }
    // Keeps the entries of this CTA's list of m among which the running count
    // (from before_cnt) reaches k, or the running mass (from before_mass) t;
    // their number.  A histogram of the keys, as in select, but of this list
    // alone (in the words of the merged one, which is lost): sorting 1300
    // entries took 13k cycles.
    __device__ int narrow_list(int m, bool by_mass, uint32_t k, double t, uint32_t& before_cnt, u64& before_mass,
                               bool need_mass) const {
        constexpr int PER = kList / kT;
        uint32_t *cnt = s.count, *l0 = s.mcnt, *l1 = reinterpret_cast<uint32_t*>(s.mmass), *l2 = l1 + kBins;
        u64 key[PER], mn = kNoKey, mx = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x + j * kT;
            key[j] = i < m ? s.list[i] : kNoKey;
            if (i < m) {
                mn = key[j] < mn ? key[j] : mn;
                mx = key[j] > mx ? key[j] : mx;
            }
        }
        mn = block_min64(mn);
        mx = ~block_min64(~mx);
        int sh = 0;
        while (((mx - mn) >> sh) >= (u64)kBins) ++sh;
        for (int b = threadIdx.x; b < kBins; b += kT) cnt[b] = l0[b] = l1[b] = l2[b] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (threadIdx.x + j * kT < m) {
                const int b = (int)((key[j] - mn) >> sh);
                atomicAdd(&cnt[b], 1u);
                if (need_mass) {  // (at most 2048 entries: limbs of 16 bits add up within 32)
                    const u64 w = weight(from_desc((uint32_t)(key[j] >> 32)));
                    atomicAdd(&l0[b], (uint32_t)w & 0xFFFFu);
                    atomicAdd(&l1[b], (uint32_t)(w >> 16) & 0xFFFFu);
                    atomicAdd(&l2[b], (uint32_t)(w >> 32));
                }
            }
        if (threadIdx.x == 0) s.list_n = 0;
        __syncthreads();
        const Pick p = pick_bin(by_mass, k - before_cnt, before_mass, t, [&](int b) { return cnt[b]; },
                                [&](int b) { return (u64)l0[b] + ((u64)l1[b] << 16) + ((u64)l2[b] << 32); });
        before_cnt += p.before_cnt;
        before_mass += p.before_mass;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (threadIdx.x + j * kT < m && (int)((key[j] - mn) >> sh) == p.bin) s.list[atomicAdd(&s.list_n, 1u)] = key[j];
        __syncthreads();
        m = (int)s.list_n;
        __syncthreads();
        return m;
    }
    // Smallest v of the block's threads, in every thread.
    __device__ u64 block_min64(u64 v) const {
        v = warp_min(v);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s.wsum[threadIdx.x >> 5] = v;
        __syncthreads();
        return warp_min(s.wsum[threadIdx.x % kW]);
    }
    // Sum of `own` over the threads before this one; `total` over all.
    __device__ u64 block_before(u64 own, u64& total) const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const u64 incl = warp_scan(own, lane);
        __syncthreads();  // (earlier readers of wsum are done)
        if (lane == 31) s.wsum[warp] = incl;
        __syncthreads();
        const u64 upto = warp_scan(s.wsum[lane % kW], lane);  // (in lanes below kW)
        total = __shfl_sync(0xffffffffu, upto, kW - 1);
        return __shfl_sync(0xffffffffu, upto, warp) - s.wsum[warp] + incl - own;
    }
    // Smallest value of the block's threads, in every thread.
    __device__ uint32_t block_min(uint32_t v) const {
        __syncthreads();
        if (threadIdx.x == 0) s.pick_bin = 0xFFFFFFFFu;
        __syncthreads();
        v = __reduce_min_sync(0xffffffffu, v);
        if ((threadIdx.x & 31) == 0) atomicMin(&s.pick_bin, v);
        __syncthreads();
        return s.pick_bin;
    }

    // The whole choice among the m <= kList keys of this CTA's list, which
    // hold the row's first top_k candidates: filters, then the draw.
    __device__ void solve_row(int m, int top_k, float top_p, float min_p, float u, int32_t* token, float* logprob) const {
        sort_list(m);
        if (m > top_k) m = top_k;
        constexpr int PER = kList / kT;
        const int per = (m + kT - 1) / kT, at = threadIdx.x * per;  // this thread's run of entries
        u64 own = 0, total;
#pragma unroll 1
        for (int i = at; i < at + per && i < m; ++i) own += weight(from_desc((uint32_t)(s.list[i] >> 32)));
        u64 run = block_before(own, total);
        // entries that stay: up to the one at which the mass reaches its
        // share, and with at least the least weight; both cut the order off
        const double t = (double)top_p * (double)total;
        const u64 least = min_p > 0.f ? __double2ull_ru((double)min_p * weight.unit()) : 0;
        uint32_t cut = (uint32_t)m;
#pragma unroll 1
        for (int i = at; i < at + per && i < m; ++i) {
            const u64 w = weight(from_desc((uint32_t)(s.list[i] >> 32)));
            run += w;
            if (w < least) cut = min(cut, (uint32_t)i);
            if (top_p < 1.f && (double)run >= t) cut = min(cut, (uint32_t)(i + 1));
        }
        const int kept = (int)block_min(cut);
        // the draw, in index order: (index, logit) keys, sorted
        u64 again[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const u64 key = j < per && at + j < kept ? s.list[at + j] : kNoKey;
            again[j] = (key << 32) | (key >> 32);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j < per && at + j < kept) s.list[at + j] = again[j];
        __syncthreads();
        sort_list(kept);
        own = 0;
#pragma unroll 1
        for (int i = at; i < at + per && i < kept; ++i) own += weight(from_desc((uint32_t)s.list[i]));
        run = block_before(own, total);
        const double draw = (double)u * (double)total;
        if ((double)(run + own) > draw && !((double)run > draw)) {
#pragma unroll 1
            for (int i = at;; ++i) {
                const float x = from_desc((uint32_t)s.list[i]);
                run += weight(x);
                if ((double)run > draw) {
                    *token = (int32_t)(s.list[i] >> 32);
                    if (logprob) *logprob = (float)(weight.z(x) - log((double)total / weight.unit()));
                    break;
                }
            }
        }
    }

    // The threshold key at which the running count reaches k, or the running
    // mass reaches t, among the keys up to `limit`; `limit` where it does not.
    // gathered: the lists hold the keys among which it does, behind mass_to.
    // l1: the merged arrays hold the level-one histogram (with masses, where
    // need_mass); false on return if they no longer do.  mass_to (need_mass):
    // the mass of everything up to the threshold.
    __device__ __forceinline__ u64 select(bool by_mass, uint32_t k, double t, u64 limit, bool need_mass, bool gathered, bool& l1,
                                          u64& mass_to) const {
        uint32_t before_cnt = 0;
        u64 before_mass = mass_to;
        if (!gathered && !gather(by_mass, k, t, limit, need_mass, l1, before_cnt, before_mass)) {
            mass_to = before_mass;
            return limit;
        }
        csync();
        if (rank == 0) {
            int m = collect_lists();
            while (m > kCountSort) m = narrow_list(m, by_mass, k, t, before_cnt, before_mass, need_mass);
            sort_list(m);
            // prefix masses of the sorted members, in runs of `per` per thread
            const int per = (m + kT - 1) / kT;
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            u64 own = 0;
            if (need_mass)
#pragma unroll 1
                for (int j = 0; j < per; ++j) {
                    const int i = threadIdx.x * per + j;
                    if (i < m) own += weight(from_desc((uint32_t)(s.list[i] >> 32)));
                }
            const u64 incl = warp_scan(own, lane);
            if (lane == 31) s.wsum[warp] = incl;
            if (threadIdx.x == 0) s.pick_bin = 0x7fffffffu;
            __syncthreads();
            u64 run = before_mass + incl - own;
#pragma unroll 1
            for (int w = 0; w < warp; ++w) run += s.wsum[w];
            const u64 run0 = run;
#pragma unroll 1
            for (int j = 0; j < per; ++j) {
                const int i = threadIdx.x * per + j;
                if (i >= m) break;
                if (need_mass) run += weight(from_desc((uint32_t)(s.list[i] >> 32)));
                const bool hit = i == m - 1 || (by_mass ? (double)run >= t : before_cnt + (uint32_t)i + 1 >= k);
                if (hit) {
                    atomicMin(&s.pick_bin, (uint32_t)i);
                    break;
                }
            }
            __syncthreads();
            const int hit = (int)s.pick_bin;
            if (m == 0) {  // (a picked bin has members)
                if (threadIdx.x < size) {
                    st_cluster(mapa(&s.res[0], threadIdx.x), limit);
                    st_cluster(mapa(&s.res[1], threadIdx.x), before_mass);
                }
            } else if (threadIdx.x == hit / per) {
                u64 r = run0;
                if (need_mass)
#pragma unroll 1
                    for (int i = threadIdx.x * per; i <= hit; ++i)
                        r += weight(from_desc((uint32_t)(s.list[i] >> 32)));
                const u64 key = s.list[hit];
#pragma unroll 1
                for (int q = 0; q < size; ++q) {
                    st_cluster(mapa(&s.res[0], q), key);
                    st_cluster(mapa(&s.res[1], q), r);
                }
            }
        }
        csync();
        l1 = false;  // (the first CTA's merged words may have served its list)
        mass_to = s.res[1];
        const u64 thr = s.res[0];
        __syncthreads();
        return thr;
    }

    // select's first part: the members of the bin of the threshold into the
    // lists; false (with the mass of all candidates) where none is reached.
    __device__ __forceinline__ bool gather(bool by_mass, uint32_t k, double t, u64 limit, bool need_mass, bool& l1,
                                           uint32_t& before_cnt, u64& before_mass) const {
        if (!l1) build_l1(need_mass);
        l1 = true;
        Pick p = pick_bin(by_mass, k, 0, t);
        if (p.bin == kBins) {  // fewer candidates than k
            before_mass = need_mass ? l1_mass() : 0;
            return false;
        }
        const int level_bin = p.bin;
        u64 kmin = 0, kmax = limit;  // members: keys in this range (and, at first, of the picked bin)
        bool by_bin = true;
        before_cnt = p.before_cnt;
        before_mass = p.before_mass;
        auto member = [&](float v, u64 key) {
            return by_bin ? distance_bin(weight.top, v) == level_bin && key <= limit : key >= kmin && key <= kmax;
        };
        while (p.in_cnt > (uint32_t)kList) {
            // split the bin: its members' key range in kBins equal parts
            u64 mn = kNoKey, mx = 0;
            each([&](float v, int i) {
                const u64 key = order_key(v, (uint32_t)i);
                if (!member(v, key)) return;
                mn = key < mn ? key : mn;
                mx = key > mx ? key : mx;
            });
            mn = cluster_min(mn, 0);
            mx = ~cluster_min(~mx, 1);
            int sh = 0;
            while (((mx - mn) >> sh) >= (u64)kBins) ++sh;
            clear_hist();
            each([&](float v, int i) {
                const u64 key = order_key(v, (uint32_t)i);
                if (member(v, key)) add((int)((key - mn) >> sh), v, need_mass);
            });
            merge_hist();
            l1 = false;
            p = pick_bin(by_mass, k - before_cnt, before_mass, t);
            before_cnt += p.before_cnt;
            before_mass += p.before_mass;
            by_bin = false;
            kmin = mn + ((u64)p.bin << sh);
            kmax = kmin + (((u64)1 << sh) - 1);
            if (kmax > mx) kmax = mx;
        }
        // gather the members in the first CTA
        if (threadIdx.x == 0) s.list_n = 0;
        __syncthreads();
        const float d0 = near_edge(level_bin), d1 = far_edge(level_bin);
        each([&](float v, int i) {
            const float d = distance(weight.top, v);
            if (d < d0 || !(d < d1 || d1 == INFINITY)) return;  // not of the picked bin, split up or not
            const u64 key = order_key(v, (uint32_t)i);
            if (member(v, key)) s.list[atomicAdd(&s.list_n, 1u)] = key;
        });
        return true;
    }

    // Smallest v of the cluster's threads, in every thread.  `use` names the
    // words that carry it: not those of the call before, which other CTAs may
    // still be reading.
    __device__ u64 cluster_min(u64 v, int use) const {
        v = warp_min(v);
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        __syncthreads();  // (earlier readers of wsum are done)
        if (lane == 0) s.wsum[warp] = v;
        __syncthreads();
        if (warp == 0) {
            v = warp_min(lane < kW ? s.wsum[lane] : kNoKey);
            if (lane < size) st_cluster(mapa(&s.slot[use][rank], lane), v);
        }
        csync();
        return warp_min(s.slot[use][lane % size]);
    }
};

template <typename XT>
__global__ void __launch_bounds__(kT, 2) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem + a.raw_bytes);
    uint32_t rank_u, size_u;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank_u));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size_u));
    const int rank = (int)rank_u, size = (int)size_u;
    const int row = blockIdx.x / size;
    const int lane = threadIdx.x & 31;
    // this CTA's logits [i0, i1), in whole 16-byte vectors from the boundary
    // at or before the first one
    constexpr int E = Row<XT>::E;
    const int i0 = rank * a.slice < a.vocab ? rank * a.slice : a.vocab;
    const int i1 = a.vocab - i0 < a.slice ? a.vocab : i0 + a.slice;
    const XT* g = reinterpret_cast<const XT*>(a.logits) + (size_t)row * a.vocab + i0;
    const int pad = (int)(reinterpret_cast<uintptr_t>(g) & 15) / (int)sizeof(XT);
    const int vecs = i1 > i0 ? (pad + i1 - i0 + E - 1) / E : 0;
    uint4* vec = reinterpret_cast<uint4*>(smem);
    carrive();  // (awaited below: no CTA's shared memory is written before it has started)
    for (int i = threadIdx.x; i < kBins; i += kT) s.count[i] = 0;
    if (threadIdx.x == 0) s.list_n = 0;
    if (threadIdx.x < kTable) {
        const double unit = (double)(1ull << (a.frac_bits + 1));
        s.exp2_table[threadIdx.x] = __double2ull_rn(exp2(threadIdx.x * (1.0 / kTable)) * unit) << 13;
    }
    grid_dependency_wait();
    grid_dependents_launch();
    float top = -INFINITY;  // (fmaxf passes NaN over)
    {
        const uint4* src = reinterpret_cast<const uint4*>(g - pad);
        const int whole0 = pad ? 1 : 0, whole1 = (pad + i1 - i0) / E;  // vectors that lie within the row
#pragma unroll 4
        for (int j = whole0 + threadIdx.x; j < whole1; j += kT) {
            const uint4 u = ld_once(src + j);
            vec[j] = u;
            float v[E];
            Row<XT>::unpack(u, v);
#pragma unroll
            for (int k = 0; k < E; ++k) top = fmaxf(top, v[k]);
        }
        // the first and the last vector, where they reach past the row
        if (threadIdx.x < 2 * E) {
            const int j = threadIdx.x < E ? 0 : vecs - 1, k = threadIdx.x % E, i = j * E + k - pad;
            if (vecs > 0 && (j < whole0 || j >= whole1)) {
                const bool in = i >= 0 && i < i1 - i0;
                const XT v = in ? g[i] : from_float<XT>(-INFINITY);
                reinterpret_cast<XT*>(vec)[j * E + k] = v;
                if (in) top = fmaxf(top, to_f32(v));
            }
        }
    }
    float temp = a.temperature ? a.temperature[row] : 1.f;
    const float u_in = a.uniforms[row];
    const int top_k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.f;
    const float min_p = a.min_p ? a.min_p[row] : 0.f;
    cwait();

    Row<XT> r{s, vec, i0 - pad, vecs, rank, size, a.slice <= 32768 ? 17 : 16, {}};
    const u64 best = r.cluster_min((u64)desc_bits(top), 0);
    top = from_desc((uint32_t)best);
    const bool none = !(top > -INFINITY);
    if (none || !(temp > 0.f) || top_k == 1 || top_p <= 0.f || min_p > 1.f) {
        // nothing to choose from, or the front candidate alone
        u64 first = kNoKey;
        if (!none) r.each([&](float v, int i) { first = v == top && (u64)i < first ? (u64)i : first; });
        first = r.cluster_min(first, 1);
        if (rank == 0 && threadIdx.x == 0) {
            a.tokens[row] = none ? -1 : (int32_t)first;
            if (a.logprobs) a.logprobs[row] = none ? -INFINITY : 0.f;
            if (none) report(a.status, COTTUS_STATUS_NO_TOKEN);
        }
        return;
    }
    r.weight.set(top, temp, a.frac_bits, s.exp2_table);

    u64 thr = kNoKey;
    const bool by_p = top_p < 1.f;  // (false for NaN)
    const bool by_k = top_k > 0 && top_k < a.vocab;
    // uniform in [0, 1): 1 - 2^-24 is the largest fp32 below 1 (NaN counts as 0)
    const float u = u_in > 0.f ? fminf(u_in, 0.99999994f) : 0.f;
    if (by_k && top_k <= kDirect) {
        // few candidates: their histogram by count alone, every CTA adding up
        // the cluster's; the first CTA gets all up to the bin in which the
        // count reaches top_k, and does the rest by itself
        r.count_distances(false);
        const auto p = r.pick_bin(false, (uint32_t)top_k, 0, 0.0);
        if (p.before_cnt + p.in_cnt <= (uint32_t)kList) {  // (no bin picked: top_k candidates or fewer)
            const uint32_t counter = mapa(&s.list_n, 0), list0 = mapa(&s.list[0], 0);
            const float d1 = far_edge(p.bin);
            r.each([&](float v, int i) {
                const float d = distance(top, v);
                if (d < d1 || d1 == INFINITY)
                    st_cluster(list0 + atom_add_cluster(counter, 1) * 8, order_key(v, (uint32_t)i));
            });
            csync();
            if (rank == 0) r.solve_row((int)s.list_n, top_k, top_p, min_p, u, a.tokens + row, a.logprobs ? a.logprobs + row : nullptr);
            return;
        }
        csync();  // (the histogram is about to be cleared)
    }
    // each thread owns a contiguous run of vectors (an odd number, so that the
    // lanes of a warp read from different banks)
    const int run = (vecs + kT - 1) / kT | 1;
    const int v0 = threadIdx.x * run < vecs ? threadIdx.x * run : vecs, v1 = v0 + run < vecs ? v0 + run : vecs;
    // min-p in the weights' units (0: off, as for NaN; the largest weight, 1, always stays)
    const u64 least_w = min_p > 0.f ? __double2ull_ru((double)min_p * r.weight.unit()) : 0;

    bool near = false;  // the members around top-p's threshold are in the lists
    u64 mass = 0, own = 0;
    u64 mine[kList / kT];  // this thread's of them
    double t_mass = 0.0;
    if (by_p && !by_k && r.weight.plain) {
        // top-p alone: the counts of the distances say about where its
        // threshold is.  One pass then takes exact sums, of everything and of
        // what lies before that place, and lists the tokens around it.  Where
        // the sums show it to be among those, the rest is work on the lists;
        // else nothing is lost but the pass.  (Masses of all bins are four
        // atomics per token: 64 x 128256 fp32 took 140 us, so 108.)
        r.count_distances(true);
        int b0, b1;
        // (as wide as the lists bear where a share of the mass has up to
        // sixteen times its share of the tokens)
        r.mass_range(top_p, fminf(0.01f, (float)size * (kList / 16) / (float)a.vocab), b0, b1);
        const float d0 = near_edge(b0), d1 = far_edge(b1);
        u64 all = 0;
        for (int j = v0; j < v1; ++j) {
            float v[E];
            Row<XT>::unpack(vec[j], v);
#pragma unroll
            for (int k = 0; k < E; k += 2) {
                const auto w = r.weight.fast(v[k], v[k + 1]);
                all += w.x + w.y;
                own += (top - v[k] < d0 ? w.x : 0) + (top - v[k + 1] < d0 ? w.y : 0);
            }
#pragma unroll
            for (int k = 0; k < E; ++k) {
                const float d = top - v[k];  // (neither -inf nor NaN passes d < d1)
                if (d >= d0 && d < d1) {
                    const uint32_t at = atomicAdd(&s.list_n, 1u);
                    if (at < (uint32_t)kList) s.list[at] = order_key(v[k], (uint32_t)(r.lo + j * E + k));
                }
            }
        }
        u64 cta_all, cta_before;
        r.block_before(all, cta_all);
        r.block_before(own, cta_before);
        const bool full = s.list_n > (uint32_t)kList;
        if (threadIdx.x < size) {
            st_cluster(mapa(&s.slot[0][rank], threadIdx.x), cta_all);
            st_cluster(mapa(&s.slot[1][rank], threadIdx.x), cta_before | (full ? 1ull << 63 : 0));
        }
        csync();
        u64 before = 0;
        for (int q = 0; q < size; ++q) {
            mass += s.slot[0][q];
            before |= s.slot[1][q] & (1ull << 63);
            before += s.slot[1][q] & ~(1ull << 63);
        }
        t_mass = (double)top_p * (double)mass;
        if (!(before >> 63) && (double)before < t_mass) {
            // a histogram of the listed ones, and the members of its bin
            const uint32_t lo_bits = b0 ? __float_as_uint(d0) : 0, span = __float_as_uint(d1) - lo_bits;
            int sh = 0;
            while (((span - 1) >> sh) >= (uint32_t)kBins) ++sh;
            const int m = (int)s.list_n;
            r.clear_hist();
            auto bin_of = [&](u64 key) {
                return (int)((__float_as_uint(top - from_desc((uint32_t)(key >> 32))) - lo_bits) >> sh);
            };
#pragma unroll
            for (int j = 0; j < kList / kT; ++j) {
                const int i = threadIdx.x + j * kT;
                mine[j] = i < m ? s.list[i] : kNoKey;
                if (i < m) r.add(bin_of(mine[j]), from_desc((uint32_t)(mine[j] >> 32)), true);
            }
            __syncthreads();
            if (threadIdx.x == 0) s.list_n = 0;
            r.merge_hist();
            const auto p = r.pick_bin(true, 0, before, t_mass);
            near = p.bin < kBins && p.in_cnt <= (uint32_t)kList;
            if (near) {
#pragma unroll
                for (int j = 0; j < kList / kT; ++j)
                    if (mine[j] != kNoKey && bin_of(mine[j]) == p.bin) s.list[atomicAdd(&s.list_n, 1u)] = mine[j];
                mass = before + p.before_mass;
            } else {
                csync();  // (the histogram is about to be cleared)
            }
        }
    }
    // first by count, then by mass
    bool l1 = false;
    for (int by_mass = by_k ? 0 : 1; by_mass < (by_p ? 2 : 1); ++by_mass) {
        if (by_mass && !by_k && !near) {  // the whole mass first: one histogram serves both
            r.build_l1(true);
            l1 = true;
            mass = r.l1_mass();
        }
        if (!near) t_mass = (double)top_p * (double)mass;
        thr = r.select(by_mass != 0, (uint32_t)top_k, t_mass, thr, by_p, near, l1, mass);
    }

    // the kept mass
    const float thr_v = thr == kNoKey ? -INFINITY : from_desc((uint32_t)(thr >> 32));
    const int thr_i = (int)(uint32_t)thr;
    auto kept = [&](float v, int i, u64 w) -> u64 {  // w, or 0 behind the threshold or below min-p
        return (v > thr_v || (v == thr_v && i <= thr_i)) && w >= least_w ? w : 0;
    };
    if (near && least_w == 0) {
        // what lies before the listed ones is summed up already; of those, the
        // ones up to the threshold go to their runs (in the merged masses' words)
        s.mmass[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kList / kT; ++j)
            if (mine[j] != kNoKey && mine[j] <= thr)
                atomicAdd(&s.mmass[((uint32_t)mine[j] - r.lo) / E / run], r.weight.fast(from_desc((uint32_t)(mine[j] >> 32))));
        __syncthreads();
        own += s.mmass[threadIdx.x];
    } else if (own = 0; r.weight.plain) {
        auto pairs = [&](auto f) {
            for (int j = v0; j < v1; ++j) {
                float v[E];
                Row<XT>::unpack(vec[j], v);
#pragma unroll
                for (int k = 0; k < E; k += 2) own += f(v[k], v[k + 1], r.lo + j * E + k, r.weight.fast(v[k], v[k + 1]));
            }
        };
        if (thr == kNoKey && least_w == 0) pairs([&](float, float, int, auto w) { return w.x + w.y; });
        else pairs([&](float x, float y, int i, auto w) { return kept(x, i, w.x) + kept(y, i + 1, w.y); });
    } else {
        for (int i = v0 * E; i < v1 * E; ++i) {
            const float v = to_f32(reinterpret_cast<const XT*>(vec)[i]);
            own += kept(v, r.lo + i, r.weight.general(v));
        }
    }
    u64 cta;
    u64 base = r.block_before(own, cta);
    if (threadIdx.x < size) st_cluster(mapa(&s.slot[2][rank], threadIdx.x), cta);
    csync();
    u64 total = 0;
    for (int q = 0; q < size; ++q) {
        if (q < rank) base += s.slot[2][q];
        total += s.slot[2][q];
    }
    const double t = (double)u * (double)total;
    // the thread in whose run the running sum first exceeds t; its warp
    // walks the run, a logit per lane
    const uint32_t owner = __ballot_sync(0xffffffffu, (double)(base + own) > t && !((double)base > t));
    if (owner) {
        const int who = __ffs(owner) - 1;
        u64 before = __shfl_sync(0xffffffffu, base, who);
        const int e0 = __shfl_sync(0xffffffffu, v0, who) * E, e1 = __shfl_sync(0xffffffffu, v1, who) * E;
        for (int i0 = e0; i0 < e1; i0 += 32) {
            const int i = i0 + lane;
            const float v = i < e1 ? to_f32(reinterpret_cast<const XT*>(vec)[i]) : -INFINITY;
            const u64 m = kept(v, r.lo + i, r.weight(v));
            const u64 incl = before + warp_scan(m, lane);
            const uint32_t hit = __ballot_sync(0xffffffffu, (double)incl > t);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    a.tokens[row] = r.lo + i;
                    if (a.logprobs) a.logprobs[row] = (float)(r.weight.z(v) - log((double)total / r.weight.unit()));
                }
                break;
            }
            before = __shfl_sync(0xffffffffu, incl, 31);
        }
    }
}

// Dynamic shared memory of a CTA that holds `slice` logits.
size_t sample_smem(int slice, int es) { return ((size_t)slice * es + 46) / 16 * 16 + sizeof(Shared); }

template <typename XT>
cudaError_t launch_sample(SampleArgs a, int batch, int cluster, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};  // a bit per device
    auto kern = sample_kernel<XT>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready.fetch_or(uint64_t(1) << dev, std::memory_order_release);
    }
    a.slice = (a.vocab + cluster - 1) / cluster;
    const size_t smem = sample_smem(a.slice, sizeof(XT));
    a.raw_bytes = (int)(smem - sizeof(Shared));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)batch * cluster));
    cfg.blockDim = dim3(kT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

int fail(int code, const std::string& msg) { return set_error(code, msg); }

}  // namespace
}  // namespace cb200

extern "C" int cottus_sample_tokens(const cottus_sample_params* p, cottus_stream_t stream) {
    using namespace cb200;
    if (!p) return fail(COTTUS_ERR_INVALID_ARGUMENT, "params must not be NULL");
    if (p->batch < 0 || p->vocab <= 0) return fail(COTTUS_ERR_INVALID_ARGUMENT, "batch must be non-negative and vocab positive");
    if (!lowp_input_dtype(p->dtype)) return fail(COTTUS_ERR_INVALID_ARGUMENT, "unknown dtype");
    if (p->vocab > COTTUS_MAX_VOCAB)
        return fail(COTTUS_ERR_UNSUPPORTED, "vocab must be at most " + std::to_string(COTTUS_MAX_VOCAB));
    if (p->batch == 0) return COTTUS_OK;
    if (p->batch > (1 << 27)) return fail(COTTUS_ERR_UNSUPPORTED, "too many rows for one launch");
    if (!p->logits || !p->uniforms || !p->tokens) return fail(COTTUS_ERR_INVALID_ARGUMENT, "NULL pointer argument");
    const int es = dtype_bytes(p->dtype);
    if (!aligned(p->logits, es) || !aligned(p->uniforms, 4) || !aligned(p->temperature, 4) || !aligned(p->top_k, 4) ||
        !aligned(p->top_p, 4) || !aligned(p->min_p, 4) || !aligned(p->tokens, 4) || !aligned(p->logprobs, 4))
        return fail(COTTUS_ERR_INVALID_ARGUMENT, "a pointer is not aligned to its element");
    const size_t b4 = (size_t)p->batch * 4;
    const Span out[2] = {{p->tokens, b4}, {p->logprobs, p->logprobs ? b4 : 0}};
    const Span in[6] = {{p->logits, (size_t)p->batch * p->vocab * es}, {p->uniforms, b4},
                        {p->temperature, p->temperature ? b4 : 0}, {p->top_k, p->top_k ? b4 : 0},
                        {p->top_p, p->top_p ? b4 : 0}, {p->min_p, p->min_p ? b4 : 0}};
    bool clash = overlap(out[0], out[1]);
    for (const Span& o : out)
        for (const Span& i : in) clash = clash || overlap(o, i);
    if (clash) return fail(COTTUS_ERR_INVALID_ARGUMENT, "an output overlaps another buffer");
    SampleArgs a = {};
    a.logits = p->logits;
    a.uniforms = p->uniforms;
    a.temperature = p->temperature;
    a.top_k = p->top_k;
    a.top_p = p->top_p;
    a.min_p = p->min_p;
    a.tokens = p->tokens;
    a.logprobs = p->logprobs;
    a.status = p->status;
    a.vocab = p->vocab;
    int bits = 1;
    while ((int64_t(1) << bits) <= p->vocab) ++bits;
    a.frac_bits = 62 - bits < 47 ? 62 - bits : 47;  // a weight fits three 16-bit limbs, a row's sum 62 bits
    int dev = 0;
    cudaGetDevice(&dev);
    const int sms = device_sm_count(dev);
    // the smallest cluster that gives every SM work, and whose slices let two CTAs share an SM
    int cluster = 1;
    while (cluster < kMaxCluster &&
           ((long long)p->batch * cluster < sms || sample_smem((p->vocab + cluster - 1) / cluster, es) > 114 * 1024))
        cluster *= 2;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = p->dtype == COTTUS_F32   ? launch_sample<float>(a, p->batch, cluster, st)
                          : p->dtype == COTTUS_F16 ? launch_sample<__half>(a, p->batch, cluster, st)
                                                   : launch_sample<__nv_bfloat16>(a, p->batch, cluster, st);
    return e == cudaSuccess ? COTTUS_OK : fail(COTTUS_ERR_CUDA, std::string("CUDA error: ") + cudaGetErrorString(e));
}
