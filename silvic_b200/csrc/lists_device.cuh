// lists_device.cuh — what the kernels over lists of candidates share on the device.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"
#include "lists.cuh"

namespace sb2 {

constexpr float kLog2E = 1.4426950408889634f;

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
__device__ __forceinline__ unsigned long long order_key(float z, uint32_t index) {
    const uint32_t bits = __float_as_uint(__fadd_rn(z, 0.0f));
    uint32_t order = (bits >> 31) != 0 ? ~bits : (bits | 0x80000000u);
    if (z != z) order = 0xFFFFFFFFu;
    return (static_cast<unsigned long long>(order) << 32) | (0xFFFFFFFFu - index);
}

// exp((z - m) / T) with c = log2(e) / T: the difference first, so the argument's error grows with the distance from
// the maximum, where the terms are small, and not with the scores' size.
__device__ __forceinline__ float exp_of(float d, float c) { return exp2f(__fmul_rn(d, c)); }

}  // namespace sb2
