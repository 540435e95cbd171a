// Products of 8-bit integers with a scale for each row of both operands (a
// token of the activations, an output channel of the weights):
//   out[m][n] = (sum_k a[m][k] b[n][k]) sa[m] sb[n] + bias[n]
// Sums are exact in 32-bit integers for K <= 131071 (128^2 K < 2^31); the scales
// are applied in 32-bit floats, and one rounding leads to the output's type.
#include "element.h"

namespace pfa {

namespace {

using i32x4 = int __attribute__((ext_vector_type(4)));
using i32x16 = int __attribute__((ext_vector_type(16)));

struct MatmulArgs {
    const int8_t *a, *b;      // [M][K], [N][K], rows a_stride and b_stride bytes apart
    const float *sa, *sb;     // [M], [N]
    const float *bias;        // [N] or null
    void *out;                // [M][N], rows out_stride elements apart
    size_t a_stride, b_stride, out_stride;
    uint32_t M, N, K;
};

// 16 codes of a row from place k on; places past the row's end are 0
__device__ __forceinline__ i32x4 load16(const int8_t *row, uint32_t k, uint32_t K) {
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        __builtin_memcpy(&v, row + k, 16);
    } else {
        for (uint32_t i = 0; k + i < K; i++) reinterpret_cast<int8_t *>(&v)[i] = row[k + i];
    }
    return v;
}

// 64 x 64 outputs a workgroup, 32 x 32 a wave.  The matrix instruction takes b's rows
// as its first operand, so a lane holds 4 neighbouring n of one m.
constexpr int kTile = 64, kStep = 64, kPitch = kStep + 16;

template <class T>
__global__ void __launch_bounds__(256)
k_matmul(MatmulArgs g) {
    __shared__ __align__(16) int8_t sa[kTile * kPitch], sb[kTile * kPitch];
    const uint32_t across = (g.N + kTile - 1) / kTile;
    const uint32_t m0 = blockIdx.x / across * kTile, n0 = blockIdx.x % across * kTile;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t wm = wave / 2 * 32, wn = wave % 2 * 32;
    const uint32_t r = threadIdx.x / 4, c = threadIdx.x % 4 * 16;
    const int8_t *ra = g.a + (size_t)min(m0 + r, g.M - 1) * g.a_stride;
    const int8_t *rb = g.b + (size_t)min(n0 + r, g.N - 1) * g.b_stride;
    i32x16 acc = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    for (uint32_t k = 0; k < g.K; k += kStep) {
        const i32x4 va = load16(ra, k + c, g.K), vb = load16(rb, k + c, g.K);
        __syncthreads();
        *reinterpret_cast<i32x4 *>(sa + r * kPitch + c) = va;
        *reinterpret_cast<i32x4 *>(sb + r * kPitch + c) = vb;
        __syncthreads();
#pragma unroll
        for (int h = 0; h < kStep; h += 32) {
            const uint32_t at = lane % 32 * kPitch + h + lane / 32 * 16;
            const i32x4 fa = *reinterpret_cast<const i32x4 *>(sa + wm * kPitch + at);
            const i32x4 fb = *reinterpret_cast<const i32x4 *>(sb + wn * kPitch + at);
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb, fa, acc, 0, 0, 0);
        }
    }
    const uint32_t m = m0 + wm + lane % 32;
    if (m >= g.M) return;
    const float s = g.sa[m];
    T *out = static_cast<T *>(g.out) + (size_t)m * g.out_stride;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const uint32_t n = n0 + wn + i / 4 * 8 + lane / 32 * 4 + i % 4;
        if (n < g.N) out[n] = (T)((float)acc[i] * s * g.sb[n] + (g.bias ? g.bias[n] : 0.f));
    }
}

constexpr size_t kMostK = 131071;

}  // namespace

}  // namespace pfa

using namespace pfa;

extern "C" {

int pfa_int8_matmul(const int8_t *a, size_t a_stride, const float *a_scales, const int8_t *b, size_t b_stride,
                    const float *b_scales, const float *bias, size_t M, size_t N, size_t K, void *out, int type,
                    size_t out_stride, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        require(K <= kMostK, "pfa_int8_matmul: sums of more than 131071 products can pass 32 bits");
        require(M <= 0x7fffffffu && N <= 0x7fffffffu, "pfa_int8_matmul: more than 2^31 - 1 rows");
        require(!workspace_bytes || workspace, "null workspace");
        if (M == 0 || N == 0) return;
        require(a_scales && b_scales && out && (K == 0 || (a && b)), "null argument");
        require((M == 1 || ((a_stride == 0 || a_stride >= K) && out_stride >= N)) &&
                    (N == 1 || b_stride == 0 || b_stride >= K),
                "rows overlap");
        require((((uintptr_t)a_scales | (uintptr_t)b_scales | (uintptr_t)bias) & 3) == 0 &&
                    ((uintptr_t)out & (size - 1)) == 0,
                "pfa_int8_matmul: a tensor is not aligned to its elements");
        MatmulArgs g{a, b, a_scales, b_scales, bias, out, a_stride, b_stride, out_stride, (uint32_t)M, (uint32_t)N,
                     (uint32_t)K};
        const size_t tiles = ((M + kTile - 1) / kTile) * ((N + kTile - 1) / kTile);
        require(tiles < 1u << 24, "pfa_int8_matmul: more outputs than one launch can form");
        with_type(type, [&](auto t) {
            hipLaunchKernelGGL(k_matmul<decltype(t)>, dim3((uint32_t)tiles), dim3(256), 0, as_stream(stream), g);
        });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
