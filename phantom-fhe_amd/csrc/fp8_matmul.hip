// Products of 8-bit floating point codes (e4m3) with a scale for each 128 places of a row of a (a token of
// the activations) and for each 128 rows and 128 places of b (output channels of the weights):
//   out[m][n] = sum_j (sum_{k in block j} a[m][k] b[n][k]) sa[m][j] sb[n / 128][j] + bias[n]
// Sums of a block and of the blocks are held in 32-bit floats, and one rounding leads to the output's type.
//
// Products for 16-bit outputs are formed by the 8-bit matrix instruction: it adds eight neighbouring products at a
// time, aligned to the largest of them, and cuts what is below 2^-13 of that one (measured; towards 0, so without
// a drift), then adds in 32 bits.  The sum of a block is off by 2^-13 of its largest products at most 8 times over, near
// 2^-16 of the result's size on normal codes, where a 16-bit output is rounded at 2^-8 or 2^-11.  32-bit
// outputs show it, so their codes are widened to 16-bit floats (exact) and multiplied at half that rate, every sum in 32
// bits.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "codes.h"

namespace pfa {

namespace {

using i32x8 = int __attribute__((ext_vector_type(8)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using f16x2 = _Float16 __attribute__((ext_vector_type(2)));

constexpr uint32_t kBlock = 128;  // places, and rows of b, that share a scale

struct Fp8Args {
    const int8_t *a, *b;   // [M][K], [N][K], rows a_stride and b_stride bytes apart
    const float *sa, *sb;  // scale (r, j) at r * row + j * block
    const float *bias;     // [N] or null
    void *out;             // [M][N], rows out_stride elements apart
    size_t a_stride, b_stride, out_stride, sa_row, sa_block, sb_row, sb_block;
    uint32_t M, N, K;
};

// 16 x 16 sums of 128 products.  A lane holds 2 x 16 codes of row lane % 16 of either operand, the same places of both.
template <bool WIDE>
__device__ __forceinline__ f32x4 block_sums(const i32x4 (&a)[2], const i32x4 (&b)[2]) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (!WIDE) {
        const i32x8 fa = {a[0][0], a[0][1], a[0][2], a[0][3], a[1][0], a[1][1], a[1][2], a[1][3]};
        const i32x8 fb = {b[0][0], b[0][1], b[0][2], b[0][3], b[1][0], b[1][1], b[1][2], b[1][3]};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, fa, sum, 0, 0, 0, 0, 0, 0);
    }
    auto widened = [](const i32x4 (&v)[2], int i) {
        f16x2 h[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned w = (unsigned)v[i / 2][i % 2 * 2 + j / 2];
            h[j] = j % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)
                         : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
        }
        return f16x8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
    };
#pragma unroll
    for (int i = 0; i < 4; i++) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(widened(b, i), widened(a, i), sum, 0, 0, 0);
    return sum;
}

// 16 rows of a and 16 columns a workgroup: b is streamed, its waves take the blocks of K in turn and meet in LDS.
constexpr int kFewWaves = 8;

template <class T>
__global__ void __launch_bounds__(kFewWaves * 64)
k_fp8_few(Fp8Args g) {
    constexpr bool kWide = std::is_same_v<T, float>;
    __shared__ float sums[kFewWaves][16][17];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, at = lane / 16 * 32;
    const uint32_t n0 = blockIdx.x * 16, m0 = blockIdx.y * 16, am = min(m0 + lane % 16, g.M - 1);
    const int8_t *pa = g.a + (size_t)am * g.a_stride;
    const int8_t *pb = g.b + (size_t)min(n0 + lane % 16, g.N - 1) * g.b_stride;
    const float *sa = g.sa + am * g.sa_row, *sb = g.sb + n0 / kBlock * g.sb_row;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t j = wave; j * kBlock < g.K; j += kFewWaves) {
        const uint32_t c = j * kBlock + at;
        i32x4 fa[2], fb[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if ((j + 1) * kBlock <= g.K) {
                fb[h] = load16(pb, c + h * 16);
                fa[h] = load16(pa, c + h * 16);
            } else {
                fb[h] = load16_end(pb, c + h * 16, g.K);
                fa[h] = load16_end(pa, c + h * 16, g.K);
            }
        }
        const float scale = sa[j * g.sa_block] * sb[j * g.sb_block];
        const f32x4 p = block_sums<kWide>(fa, fb);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = fmaf(p[i], scale, acc[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) sums[wave][lane % 16][lane / 16 * 4 + i] = acc[i];
    __syncthreads();
    const uint32_t m = threadIdx.x / 16, n = threadIdx.x % 16;
    if (threadIdx.x >= 256 || m0 + m >= g.M || n0 + n >= g.N) return;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWaves; w++) v += sums[w][m][n];
    static_cast<T *>(g.out)[(size_t)(m0 + m) * g.out_stride + n0 + n] = (T)(v + (g.bias ? g.bias[n0 + n] : 0.f));
}

}  // namespace

}  // namespace pfa

using namespace pfa;

extern "C" {

int pfa_fp8_workspace(size_t M, size_t N, size_t K, int type, size_t *bytes) {
    return guarded([&] {
        require(bytes != nullptr, "null argument");
        type_bytes(type);
        require(M <= 0x7fffffffu && N <= 0x7fffffffu && K <= 0x7fffffffu, "pfa_fp8_workspace: more than 2^31 - 1 rows or places");
        *bytes = 0;
    });
}

int pfa_fp8_matmul(const uint8_t *a, size_t a_stride, const float *a_scales, size_t a_scales_row, size_t a_scales_block,
                   const uint8_t *b, size_t b_stride, const float *b_scales, size_t b_scales_row, size_t b_scales_block,
                   const float *bias, size_t M, size_t N, size_t K, void *out, int type, size_t out_stride,
                   void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        require(M <= 0x7fffffffu && N <= 0x7fffffffu && K <= 0x7fffffffu, "pfa_fp8_matmul: more than 2^31 - 1 rows or places");
        require(!workspace_bytes || workspace, "null workspace");
        if (M == 0 || N == 0) return;
        require(out && (K == 0 || (a && b && a_scales && b_scales)), "null argument");
        require((M == 1 || ((a_stride == 0 || a_stride >= K) && out_stride >= N)) &&
                    (N == 1 || b_stride == 0 || b_stride >= K),
                "rows overlap");
        require((((uintptr_t)a_scales | (uintptr_t)b_scales | (uintptr_t)bias) & 3) == 0 &&
                    ((uintptr_t)out & (size - 1)) == 0,
                "pfa_fp8_matmul: a tensor is not aligned to its elements");
        require(((uintptr_t)workspace & 15) == 0, "pfa_fp8_matmul: the workspace is not aligned to 16 bytes");
        const Fp8Args g{(const int8_t *)a, (const int8_t *)b, a_scales,     b_scales,       bias,         out,
                        a_stride,          b_stride,          out_stride,   a_scales_row,   a_scales_block,
                        b_scales_row,      b_scales_block,    (uint32_t)M,  (uint32_t)N,    (uint32_t)K};
        require((M + 15) / 16 <= 65535, "pfa_fp8_matmul: more rows than one launch can form");
        with_type(type, [&](auto t) {
            hipLaunchKernelGGL(k_fp8_few<decltype(t)>, dim3((uint32_t)((N + 15) / 16), (uint32_t)((M + 15) / 16)),
                               dim3(kFewWaves * 64), 0, as_stream(stream), g);
        });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
