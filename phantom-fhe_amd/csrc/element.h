// Element types of the clear operators' floating tensors, and reductions over
// a workgroup.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "internal.h"

namespace pfa {

// Storage types: arithmetic is in float, a store rounds to nearest even.
using bf16_t = __bf16;
using f16_t = _Float16;

// Calls f with a value of the type that the ABI's code `type` names.
template <class F>
void with_type(int type, F &&f) {
    switch (type) {
        case PFA_F32: f(float{}); return;
        case PFA_BF16: f(bf16_t{}); return;
        case PFA_F16: f(f16_t{}); return;
    }
    fail(PFA_ERR_INVALID_ARGUMENT, "unknown element type " + std::to_string(type));
}

inline size_t type_bytes(int type) {
    require(type == PFA_F32 || type == PFA_BF16 || type == PFA_F16, "unknown element type " + std::to_string(type));
    return type == PFA_F32 ? 4 : 2;
}

// Magnitudes as unsigned integers: ordered like the magnitudes, with every NaN
// above infinity, so one integer maximum carries a NaN through a reduction.
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = max(v, (uint32_t)__shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)v, d);
        v = o > v ? o : v;
    }
    return v;
}

}  // namespace pfa
