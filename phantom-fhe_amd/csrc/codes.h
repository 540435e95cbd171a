// Rows of 8-bit codes, as the products of them read them.
#pragma once

#include "element.h"

namespace pfa {

namespace {

using i32x4 = int __attribute__((ext_vector_type(4)));

// 16 codes of a row from place k on, from any address; places past the row's end are 0
__device__ __forceinline__ i32x4 load16(const int8_t *row, uint32_t k) {
    i32x4 v;
    __builtin_memcpy(&v, row + k, 16);
    return v;
}
__device__ __forceinline__ i32x4 load16_end(const int8_t *row, uint32_t k, uint32_t K) {
    if (K < 16) {
        i32x4 v = {0, 0, 0, 0};
#pragma unroll 1
        for (uint32_t i = k; i < K; i++) {
            const int c = (int)((uint32_t)(uint8_t)row[i] << (i % 4 * 8));
            v[0] |= i / 4 == k / 4 ? c : 0;
            v[1] |= i / 4 == k / 4 + 1 ? c : 0;
            v[2] |= i / 4 == k / 4 + 2 ? c : 0;
            v[3] |= i / 4 == k / 4 + 3 ? c : 0;
        }
        return v;
    }
    // past the end: the row's last 16 codes, moved down by what is past
    const uint32_t at = min(k, K - 16), past = min(k - at, 16u);
    i32x4 v = load16(row, at);
    if (past & 8) v = {v[2], v[3], 0, 0};
    if (past & 4) v = {v[1], v[2], v[3], 0};
    const uint32_t bits = past % 4 * 8;
#pragma unroll
    for (int i = 0; i < 4; i++)
        v[i] = (int)__builtin_amdgcn_alignbit(i < 3 ? (uint32_t)v[i + 1] : 0u, (uint32_t)v[i], bits);
    return past & 16 ? i32x4{0, 0, 0, 0} : v;
}

}  // namespace

}  // namespace pfa
