// lists_device.cuh — what the kernels over lists of candidates share on the device.
#pragma once

#include <cfloat>

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"
#include "lists.cuh"

namespace sb2 {

constexpr float kLog2E = 1.4426950408889634f;
constexpr uint32_t kFull = 0xffffffffu;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// A gradient leaves in the scores' own type (16-bit scores: one rounding, half a step at most).
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Entry `i` of an array of SB2_F32 / SB2_BF16 / SB2_F16 values.
__device__ __forceinline__ float load_typed(const void* p, int32_t type, uint64_t i) {
    if (type == SB2_F32) return static_cast<const float*>(p)[i];
    if (type == SB2_BF16) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
    return to_float(static_cast<const __half*>(p)[i]);
}

// List `i`: its first entry and its length. Boundaries come from the caller's device memory: whatever they hold, the
// range stays within the entries that the call named.
__device__ __forceinline__ void list_range(const ListsArgs& l, uint32_t i, uint64_t& first, uint32_t& n) {
    if (l.bounds == nullptr) {
        first = static_cast<uint64_t>(i) * l.stride;
        n = static_cast<uint32_t>(l.width);
        return;
    }
    const uint64_t b = l.bounds[i], e = l.bounds[i + 1];
    first = b < l.width ? b : l.width;
    const uint64_t end = e < l.width ? e : l.width;
    n = static_cast<uint32_t>(end > first ? end - first : 0);
}

// The order of alternatives as one ascending key: the score (-0 as 0, NaN above everything), then the lower index.
__device__ __forceinline__ uint32_t order_of(float z) {
    const uint32_t bits = __float_as_uint(__fadd_rn(z, 0.0f));
    return z != z ? 0xFFFFFFFFu : (bits >> 31) != 0 ? ~bits : (bits | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(float z, uint32_t index) {
    return (static_cast<unsigned long long>(order_of(z)) << 32) | (0xFFFFFFFFu - index);
}
// A score from its order (a NaN from a NaN's).
__device__ __forceinline__ float score_of(uint32_t order) {
    return __uint_as_float((order >> 31) != 0 ? order & 0x7FFFFFFFu : ~order);
}
__device__ __forceinline__ uint32_t index_of(unsigned long long key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }

// 2^x, at most 2 ulp off (ex2.approx); results below 2^-126 are 0.
__device__ __forceinline__ float pow2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// max that keeps a NaN of either side.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// exp((z - m) / T) is pow2(y) with y = exponent(z - m, c), c = log2(e) / T: the difference first, so the argument's
// error grows with the distance from the reference, where the terms are small, and not with the scores' size. A masked
// score's exponent is finite, so that 0 times it is 0.
__device__ __forceinline__ float exponent(float z, float m, float c) { return max_nan(__fmul_rn(__fsub_rn(z, m), c), -200.0f); }

// What stands for a masked entry where its exponent is multiplied: its weight is 0 beside any score that is not far.
constexpr float kMasked = -1.0e30f;

// A list as one thread block (or a cluster of them) walks it: scalars up to the first 16-byte boundary, vectors of
// kVec entries, scalars behind the last. kVec 1: entry by entry, so that sums do not depend on where a list starts.
template <class T, int kVec>
struct Walk {
    const T* z;
    uint32_t n, head, vectors;
    __device__ __forceinline__ Walk(const T* scores, uint32_t entries) : z(scores), n(entries) {
        head = 0;
        const uint32_t bytes = static_cast<uint32_t>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15);  // to the boundary
        if (kVec > 1) head = min(n, bytes / static_cast<uint32_t>(sizeof(T)));
        vectors = (n - head) / kVec;
    }
    // The first entry of vector v, and where the scalars behind the vectors start.
    __device__ __forceinline__ uint32_t at(uint32_t v) const { return head + v * kVec; }
    __device__ __forceinline__ uint32_t tail() const { return head + vectors * kVec; }
    // Scalars outside the vectors, fewer than 2 kVec: entry of scalar i, or n behind the last.
    __device__ __forceinline__ uint32_t edge(uint32_t i) const {
        if (i < head) return i;
        const uint32_t j = tail() + (i - head);
        return j < n ? j : n;
    }
};

// The packed entries of one vector.
template <class T, int kVec>
struct Pack {
    uint4 raw;
    __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const uint4*>(p)); }
    // Into shared memory, without a register (copies_done() waits for the thread's own).
    __device__ __forceinline__ void copy(const T* p) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(this))), "l"(p)
                     : "memory");
    }
    __device__ __forceinline__ void values(float (&f)[kVec]) const {
        if constexpr (sizeof(T) == 4) {
            f[0] = __uint_as_float(raw.x);
            f[1] = __uint_as_float(raw.y);
            f[2] = __uint_as_float(raw.z);
            f[3] = __uint_as_float(raw.w);
        } else {
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                    f[2 * i] = __uint_as_float(w[i] << 16);
                    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                } else {
                    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    f[2 * i] = v.x;
                    f[2 * i + 1] = v.y;
                }
            }
        }
    }
    // The largest entry (a NaN gives way).
    __device__ __forceinline__ float most() const {
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)), fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
        } else {
            const uint32_t m = larger(larger(raw.x, raw.y), larger(raw.z, raw.w));
            if constexpr (std::is_same_v<T, __nv_bfloat16>)
                return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&m));
            return fmaxf(v.x, v.y);
        }
    }
    // The entries, masked ones and those of no weight beside scores that are not far as kMasked.
    __device__ __forceinline__ void finite(float (&f)[kVec]) const {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            Pack p;
            p.raw = make_uint4(at_least(raw.x), at_least(raw.y), at_least(raw.z), at_least(raw.w));
            p.values(f);
        } else {
            values(f);
#pragma unroll
            for (int e = 0; e < kVec; ++e) f[e] = max_nan(f[e], kMasked);
        }
    }
    __device__ __forceinline__ static uint32_t at_least(uint32_t a) {
        const __nv_bfloat162 low = __floats2bfloat162_rn(kMasked, kMasked);
        const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), low);
        return *reinterpret_cast<const uint32_t*>(&m);
    }
    // The larger of each entry and its counterpart (a NaN gives way).
    __device__ __forceinline__ void raise(const Pack& o) {
        if constexpr (sizeof(T) == 4) {
            raw.x = __float_as_uint(fmaxf(__uint_as_float(raw.x), __uint_as_float(o.raw.x)));
            raw.y = __float_as_uint(fmaxf(__uint_as_float(raw.y), __uint_as_float(o.raw.y)));
            raw.z = __float_as_uint(fmaxf(__uint_as_float(raw.z), __uint_as_float(o.raw.z)));
            raw.w = __float_as_uint(fmaxf(__uint_as_float(raw.w), __uint_as_float(o.raw.w)));
        } else {
            raw.x = larger(raw.x, o.raw.x);
            raw.y = larger(raw.y, o.raw.y);
            raw.z = larger(raw.z, o.raw.z);
            raw.w = larger(raw.w, o.raw.w);
        }
    }
    __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
            return *reinterpret_cast<const uint32_t*>(&m);
        } else {
            const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
            return *reinterpret_cast<const uint32_t*>(&m);
        }
    }
    __device__ __forceinline__ void masked() {  // every entry -inf
        const uint32_t w = sizeof(T) == 4 ? 0xFF800000u : std::is_same_v<T, __nv_bfloat16> ? 0xFF80FF80u : 0xFC00FC00u;
        raw = make_uint4(w, w, w, w);
    }
};
template <class T>
struct Pack<T, 1> {
    T raw;
    __device__ __forceinline__ void load(const T* p) { raw = __ldg(p); }
    __device__ __forceinline__ void values(float (&f)[1]) const { f[0] = to_float(raw); }
    __device__ __forceinline__ float most() const { return to_float(raw); }
    __device__ __forceinline__ void finite(float (&f)[1]) const { f[0] = max_nan(to_float(raw), kMasked); }
    __device__ __forceinline__ void masked() { raw = from_float<T>(-CUDART_INF_F); }
};

// A softmax's statistics: the reference m, S = sum 2^y and V = sum 2^y y about it, y = (z - m) log2(e) / T.
struct Stats {
    float m, s, v;
};

// Statistics about another reference.
__device__ __forceinline__ void rebase(Stats& a, float m, float c) {
    const float y = exponent(a.m, m, c), f = pow2(y);
    a.v = f * (a.v + a.s * y);
    a.s *= f;
    a.m = m;
}

// Statistics about R = m c rounded, so that an exponent is one fma(z, c, -R).
struct Rounded {
    Stats a;  // a.m the reference, a.s and a.v about r
    float r;
};

// The statistics about m itself: the rounding of R is put back.
__device__ __forceinline__ Stats settled(const Rounded& x, float c) {
    if (x.a.s == 0.0f) return {x.a.m, 0.0f, 0.0f};
    const float y = -__fmaf_rn(x.a.m, c, -x.r), f = pow2(y);
    return {x.a.m, x.a.s * f, f * __fmaf_rn(x.a.s, y, x.a.v)};
}

// The statistics about a higher reference.
static __device__ __noinline__ Rounded moved(Rounded x, float m, float c) {
    Stats now = settled(x, c);
    rebase(now, m, c);
    const float r = __fmul_rn(m, c);
    const float y = __fmaf_rn(m, c, -r), f = pow2(y);
    return {{m, now.s * f, f * __fmaf_rn(now.s, y, now.v)}, r};
}

constexpr float kSlack = 4.0f;        // log2 units that an entry may lie above the reference before it moves
constexpr float kFar = 1048576.0f;    // |R| from which its rounding matters: exponents are then taken from z - m

// One thread's running statistics; kParts: V too.
template <bool kParts>
struct Reader {
    Rounded x;
    float c, limit;

    // About the maximum of the first entries (-inf: about the first unmasked entry that comes).
    __device__ __forceinline__ Reader(float m, float scale) : c(scale), limit(m + kSlack / scale) {
        x.a = {fmaxf(m, -FLT_MAX), 0.0f, 0.0f};
        x.r = m == -CUDART_INF_F ? 0.0f : __fmul_rn(m, scale);
    }
    __device__ __forceinline__ bool far() const { return !(fabsf(x.r) < kFar); }
    __device__ __forceinline__ Stats stats() const { return settled(x, c); }
    // For entries above the limit (`most` their maximum), before they are added.
    __device__ __forceinline__ void raise(float most) {
        x = moved(x, most, c);
        limit = most + kSlack / c;
    }
    // Adds entries up to the limit; kParts: none below kMasked, so that 0 times its exponent is 0.
    template <int kCount>
    __device__ __forceinline__ void add(const float (&z)[kCount]) {
        if constexpr (kCount == 1) {
            const float y = __fmaf_rn(z[0], c, -x.r), p = pow2(y);
            x.a.s += p;
            if (kParts) x.a.v = __fmaf_rn(p, y, x.a.v);
        } else {
            // Pairs in one instruction: issue bounds the kernels before memory. A vector's own sums, so that vectors do
            // not wait for one another.
            const float2 cc = make_float2(c, c), minus_r = make_float2(-x.r, -x.r);
            float2 sum = make_float2(0.0f, 0.0f), part = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int e = 0; e < kCount; e += 2) {
                const float2 y = __ffma2_rn(make_float2(z[e], z[e + 1]), cc, minus_r);
                const float2 p = make_float2(pow2(y.x), pow2(y.y));
                sum = __fadd2_rn(sum, p);
                if (kParts) part = __ffma2_rn(p, y, part);
            }
            x.a.s += sum.x + sum.y;
            if (kParts) x.a.v += part.x + part.y;
        }
    }
};

__device__ __forceinline__ void copies_begun() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

}  // namespace sb2
