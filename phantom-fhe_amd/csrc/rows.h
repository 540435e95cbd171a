// What the row-by-row kernels of the clear operators share: the grid of rows, vectors
// of a row, temperatures and masks of logits, and the checks of a call's rows.
#pragma once

#include <algorithm>
#include <string>

#include "element.h"

namespace pfa {

namespace {

// Rows go over x and y of the grid: a launch has at most 2^32 threads along one of them.
constexpr uint32_t kRowsX = 1u << 20;
__device__ __forceinline__ size_t row_of() { return (size_t)blockIdx.y * kRowsX + blockIdx.x; }
dim3 row_grid(size_t rows) {
    return dim3((uint32_t)std::min<size_t>(rows, kRowsX), (uint32_t)((rows + kRowsX - 1) / kRowsX));
}

constexpr int kVec = 8;  // elements a thread takes at once: 16 bytes of the 2-byte types, 8 codes

// Sum of squares of a row whose squares are lost in 32 bits, of values lifted by 2^100: in the
// row's threads, to be added up.  Rare, so one place at a time.
constexpr float kFewSquares = 0x1p-90f;
template <class T>
__device__ __forceinline__ float lifted_squares(const T *x, const T *residual, uint32_t width, uint32_t t,
                                                uint32_t threads) {
    float sum = 0.f;
#pragma unroll 1
    for (uint32_t i = t; i < width; i += threads) {
        const float y = ((float)x[i] + (residual ? (float)residual[i] : 0.f)) * 0x1p100f;
        sum = fmaf(y, y, sum);
    }
    return sum;
}

constexpr float kLog2e = 1.44269504088896341f;
__device__ __forceinline__ float infinity() { return __uint_as_float(kInfBits); }
__device__ __forceinline__ float not_a_number() { return __uint_as_float(0x7fc00000u); }

// e^((l - m) / t) = exp2((half l - half m) rate).  From t = 1 on the difference is formed halved, as one of two
// numbers of 32 bits may pass them and t brings it back; below 1 such a difference has weight 0 in any case.
struct Heat {
    float half, rate;
    __device__ __forceinline__ explicit Heat(float t) {
        half = t >= 1.f ? 0.5f : 1.f;
        // within float's range: a subnormal t must not make 0 rate a NaN
        rate = fminf(kLog2e / (half * t), 3e38f);
    }
    // The bound takes -infinity (also at an infinite t) to 0; m is finite.
    __device__ __forceinline__ float weight(float l, float m) const {
        return __builtin_amdgcn_exp2f(fmaxf(fmaf(l, half, -half * m) * rate, -200.f));
    }
};

// kVec logits from i on, -infinity where no token is allowed or the place is before `own`
template <class T>
__device__ __forceinline__ void allowed_logits(const T *logits, const uint8_t *mask, uint32_t i, uint32_t own,
                                               float (&v)[kVec]) {
    load_vec<kVec>(logits + i, v);
    if (mask) {
        const uint8_t *p = mask + i;
        uint32_t w[2];
        __builtin_memcpy(w, p, 8);
#pragma unroll
        for (int e = 0; e < kVec; e++) v[e] = (w[e / 4] >> (e % 4 * 8) & 0xff) ? v[e] : -infinity();
    }
#pragma unroll
    for (int e = 0; e < kVec; e++) v[e] = i + e >= own ? v[e] : -infinity();
}

// How a call is cut: chunks == 1 is one workgroup a row.
struct Cut {
    uint32_t chunk, chunks;
};

constexpr size_t kMostWidth = (size_t)1 << 30;

void aligned(const void *p, size_t bytes, const char *what) {
    require(((uintptr_t)p & (bytes - 1)) == 0, std::string(what) + " is not aligned to its elements");
}

// rows that are read may be one row over and over (stride 0), rows that are written may not
bool apart(size_t rows, size_t stride, size_t width, bool written = false) {
    return rows == 1 || stride >= width || (stride == 0 && !written);
}

void check_rows(size_t rows, size_t width, const char *what) {
    require(rows <= 0x7fffffffu, std::string(what) + ": more than 2^31 - 1 rows");
    require(width <= kMostWidth, std::string(what) + ": rows of more than 2^30 elements");
}

}  // namespace

}  // namespace pfa
