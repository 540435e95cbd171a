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

// V neighbouring elements as floats, from any address that is aligned to one element.
// The words between are vector types: a plain array would be taken apart into
// accesses of one element, while the memory takes 16 bytes at any alignment.
template <int BYTES>
struct WordsOf {
    using type = uint32_t __attribute__((ext_vector_type(BYTES / 4)));
};
template <int V, class T>
struct Elements {
    T e[V];
};
template <int V, class T>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[V]) {
    constexpr int kPart = sizeof(T) * V > 16 ? 16 : sizeof(T) * V, kEach = kPart / sizeof(T);
#pragma unroll
    for (int h = 0; h < V; h += kEach) {
        typename WordsOf<kPart>::type w;
        __builtin_memcpy(&w, p + h, kPart);
        using Part = Elements<kEach, T>;
        const auto t = __builtin_bit_cast(Part, w);
#pragma unroll
        for (int i = 0; i < kEach; i++) v[h + i] = (float)t.e[i];
    }
}
template <int V, class T>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[V]) {
    constexpr int kPart = sizeof(T) * V > 16 ? 16 : sizeof(T) * V, kEach = kPart / sizeof(T);
#pragma unroll
    for (int h = 0; h < V; h += kEach) {
        Elements<kEach, T> t;
#pragma unroll
        for (int i = 0; i < kEach; i++) t.e[i] = (T)v[h + i];
        using Words = typename WordsOf<kPart>::type;
        const auto w = __builtin_bit_cast(Words, t);
        __builtin_memcpy(p + h, &w, kPart);
    }
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
