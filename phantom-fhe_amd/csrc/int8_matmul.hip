// Products of 8-bit integers with a scale for each row of both operands (a
// token of the activations, an output channel of the weights):
//   out[m][n] = (sum_k a[m][k] b[n][k]) sa[m] sb[n] + bias[n]
// Sums are exact in 32-bit integers for K <= 131071 (128^2 K < 2^31); the scales
// are applied in 32-bit floats, and one rounding leads to the output's type.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "codes.h"

namespace pfa {

namespace {

using i32x16 = int __attribute__((ext_vector_type(16)));

struct MatmulArgs {
    const int8_t *a, *b;      // [M][K], [N][K], rows a_stride and b_stride bytes apart
    const float *sa, *sb;     // [M], [N]
    const float *bias;        // [N] or null
    void *out;                // [M][N], rows out_stride elements apart
    size_t a_stride, b_stride, out_stride;
    int *parts;               // [splits][M][N] sums, with more than one split of K
    uint32_t M, N, K, splits;
};

// Up to 16 rows of a: b is streamed once, so its bytes are the time.  A workgroup takes
// 16 columns and all rows, its waves take blocks of 128 codes of K in turn and meet in LDS,
// where integer additions have no order.  In a block a lane takes 32 neighbouring codes
// of one row: two matrix instructions, which may see K in any order as long as both
// operands agree, and every line of b is read whole.  One row, 16384 columns, K = 4096:
// 15.3 us (4.4 TB/s); 4096 columns: 6.2 us.  More rows or columns a wave were slower: a's
// fragments come through the vector cache, whose time then exceeds b's.
constexpr int kBlock = 128;
constexpr int kFewWaves = 8, kFewUnroll = 4;  // four blocks a wave in flight

template <class T>
__global__ void __launch_bounds__(kFewWaves * 64)
k_few_rows(MatmulArgs g) {
    __shared__ int sums[16][16];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t n0 = blockIdx.x * 16;
    if (threadIdx.x < 256) sums[0][threadIdx.x] = 0;
    const uint32_t at = lane / 16 * 32;
    const int8_t *pa = g.a + (size_t)min(lane % 16, g.M - 1) * g.a_stride;
    const int8_t *pb = g.b + (size_t)min(n0 + lane % 16, g.N - 1) * g.b_stride;
    i32x4 acc = {0, 0, 0, 0};
    const uint32_t blocks = g.K / kBlock;
    uint32_t k = wave;
    for (; k + (kFewUnroll - 1) * kFewWaves < blocks; k += kFewUnroll * kFewWaves) {
        i32x4 fa[kFewUnroll][2], fb[kFewUnroll][2];
#pragma unroll
        for (int u = 0; u < kFewUnroll; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t c = (k + u * kFewWaves) * kBlock + at + h * 16;
                fb[u][h] = load16(pb, c);
                fa[u][h] = load16(pa, c);
            }
#pragma unroll
        for (int u = 0; u < kFewUnroll; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[u][h], fa[u][h], acc, 0, 0, 0);
    }
    // what is left: whole blocks, and the wave whose turn it is takes the rows' end
    for (; k * kBlock < g.K; k += kFewWaves) {
        const uint32_t c = k * kBlock + at;
#pragma unroll
        for (int h = 0; h < 2; h++)
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(load16_end(pb, c + h * 16, g.K), load16_end(pa, c + h * 16, g.K),
                                                        acc, 0, 0, 0);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) atomicAdd(&sums[lane % 16][lane / 16 * 4 + i], acc[i]);
    __syncthreads();
    const uint32_t m = threadIdx.x / 16, n = n0 + threadIdx.x % 16;
    if (m < g.M && threadIdx.x < 256 && n < g.N)
        static_cast<T *>(g.out)[(size_t)m * g.out_stride + n] =
            (T)((float)sums[m][threadIdx.x % 16] * g.sa[m] * g.sb[n] + (g.bias ? g.bias[n] : 0.f));
}

// Many rows: BM x BN outputs a workgroup of WM x WN waves.  Blocks of 128 codes of K go
// through LDS in a ring of STAGES blocks: the loads write LDS themselves, and all blocks but
// one are on their way while that one is multiplied.  A block's rows are 128 bytes, 8 chunks of
// 16, and chunk c of row r stands in place c ^ (r mod 8), so that a wave's reading of one
// chunk of 8 rows touches every bank once.  MF is the matrix instruction: 32 x 32 outputs from 32
// codes, or 16 x 16 from 64, whose shorter sums keep small tiles' chains short.  Large products
// (4096 x 16384 x 4096: 252 us, 8192^3: 460 us, 2.2 and 2.4 POP/s) are bound by the blocks' way into the L2s, then by
// the matrix units (55 % busy); wide ones of few rows by reading b (20 x 131072 x 4096: 97 us, 5.6 TB/s);
// small ones by the blocks' latency (128 x 4096 x 4096: 9.1 us).
template <int MF>
struct Matrix;
template <>
struct Matrix<32> {
    using Sum = i32x16;
    static __device__ __forceinline__ Sum product(i32x4 a, i32x4 b, Sum c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
    }
};
template <>
struct Matrix<16> {
    using Sum = i32x4;
    static __device__ __forceinline__ Sum product(i32x4 a, i32x4 b, Sum c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
    }
};

template <class T, int MF, int BM, int BN, int WM, int WN, int STAGES>
__global__ void __launch_bounds__(WM * WN * 64)
k_tiles(MatmulArgs g) {
    constexpr int WAVES = WM * WN, TM = BM / WM / MF, TN = BN / WN / MF;
    constexpr int kRows = BM + BN, kStage = kRows * kBlock;
    constexpr int kLoads = kRows / 8 / WAVES;  // a wave's load is 8 rows, 1 KiB
    constexpr int kLanes = 64 / MF;            // lanes that share a row of a fragment
    static_assert(kRows % (8 * WAVES) == 0 && BM % 8 == 0, "whole loads");
    using M = Matrix<MF>;
    // The ring, and in its place behind the products the scales, offsets and a line of outputs a wave.  Part of the
    // kernel and not of the launch, where more than 64 KiB need a limit raised on every device.
    constexpr int kRing = kStage * STAGES, kLines = (BN * 2 + BM) * 4 + WAVES * MF * (BN / WN * 4 + 16);
    constexpr int kLds = kRing > kLines ? kRing : kLines;
    static_assert(kLds <= 160 * 1024, "a CU's LDS");
    __shared__ __align__(1024) int8_t held[kLds];
    // where it begins is not told to the compiler: the tile of 32 x 64 then moves its sums from one register to
    // another in every block (17 x 4096 x 4096 8.9 us, told 9.4)
    uint32_t start = 0;
    asm("" : "+s"(start));
    int8_t *ring = held + start;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t down = (g.M + BM - 1) / BM, across = (g.N + BN - 1) / BN;
    // workgroups are dealt to the 8 XCDs in turn: each XCD gets a run of tiles, in groups of
    // some tiles of rows, so that its L2 holds what its tiles share (tiles of 256 rows, 8192 x
    // 8192 x 4096, us: groups of 2, 4, 6, 8: 258, 266, 255, 266)
    constexpr uint32_t kGroup = BM >= 256 ? 6 : 8;
    const uint32_t jobs = down * across * g.splits, each = (jobs + 7) / 8;
    const uint32_t job = blockIdx.x % 8 * each + blockIdx.x / 8;
    if (job >= jobs || blockIdx.x / 8 >= each) return;
    const uint32_t split = job % g.splits, t = job / g.splits;
    const uint32_t group = t / (kGroup * across), height = min(kGroup, down - group * kGroup);
    const uint32_t m0 = (group * kGroup + t % (kGroup * across) % height) * BM, n0 = t % (kGroup * across) / height * BN;
    const uint32_t wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    // this workgroup's codes of K
    const uint32_t all = (g.K + kBlock - 1) / kBlock, share = (all + g.splits - 1) / g.splits;
    const uint32_t first = split * share, last = min(first + share, all);
    const uint32_t full = max(min(last, g.K / kBlock), first);  // all but a block with the rows' end

    const uint32_t chunk = (lane % 8 ^ lane / 8) * 16;
    const int8_t *from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const uint32_t r = (wave * kLoads + i) * 8 + lane / 8;
        from[i] = r < BM ? g.a + (size_t)min(m0 + r, g.M - 1) * g.a_stride
                         : g.b + (size_t)min(n0 + r - BM, g.N - 1) * g.b_stride;
    }
    // Rows a power of two apart start in the same memory channel.  Where tiles share no rows of b,
    // each begins with another block (20 x 131072 x 4096: 103 -> 97 us).
    const uint32_t whole = full - first, turn = down == 1 && whole ? t * 3 % whole : 0;
    auto request = [&](int8_t *stage, uint32_t block, int i) {
        block += turn;
        block -= block < full ? 0 : whole;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) uint32_t *)(from[i] + chunk + block * kBlock),
            (__attribute__((address_space(3))) uint32_t *)(stage + (wave * kLoads + i) * 1024), 16, 0, 0);
    };
    typename M::Sum acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; m++)
#pragma unroll
        for (int n = 0; n < TN; n++) acc[m][n] = {};

    // Fragments of step h are read while step h - 1 is multiplied, the next block's first ones
    // while the last step is: its barrier stands before that step.
    constexpr int kSteps = kBlock / 16 / kLanes, kFrags = TM + TN, kProducts = TM * TN;
    const uint32_t ra = (wm + lane % MF) * kBlock, rb = (BM + wn + lane % MF) * kBlock;
    i32x4 f[2][kFrags];
    auto fragment = [&](const int8_t *stage, int h, int i) {
        const uint32_t c = ((h * kLanes + lane / MF) ^ (lane % 8)) * 16;
        const uint32_t row = i < TN ? rb + i * MF * kBlock : ra + (i - TN) * MF * kBlock;
        f[h % 2][i] = *reinterpret_cast<const i32x4 *>(stage + row + c);
    };
    // every wave's part of the awaited block has landed, and all are done with the one before
    auto landed = [&](bool more) {
        constexpr int kLeft = STAGES > 2 ? kLoads * (STAGES - 2) : 0;  // loads of the blocks behind it
        static_assert(kLeft < 64, "the counter's range");
        asm volatile("" ::: "memory");
        if (more)
            __builtin_amdgcn_s_waitcnt(0x0070 | (kLeft & 15) | kLeft >> 4 << 14);
        else
            __builtin_amdgcn_s_waitcnt(0x0070);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // requests go out in a block's first steps, a few products apart
    constexpr int kSpread = kSteps > 1 ? (kSteps - 1) * kProducts : kProducts;
    auto multiply = [&](const int8_t *now, const int8_t *next, int8_t *to, uint32_t ahead, auto asks, auto ends) {
#pragma unroll
        for (int h = 0; h < kSteps; h++) {
            if (h == kSteps - 1 && !ends) landed(asks);
#pragma unroll
            for (int j = 0; j < kProducts; j++) {
#pragma unroll
                for (int i = 0; i < kFrags; i++)
                    if (i * kProducts / kFrags == j) {
                        if (h + 1 < kSteps)
                            fragment(now, h + 1, i);
                        else if (!ends)
                            fragment(next, 0, i);
                    }
                if (asks)
#pragma unroll
                    for (int i = 0; i < kLoads; i++)
                        if (i * kSpread / kLoads == h * kProducts + j) request(to, ahead, i);
                acc[j / TN][j % TN] = M::product(f[h % 2][j % TN], f[h % 2][TN + j / TN], acc[j / TN][j % TN]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    uint32_t at = 0, b = first;
    if (first < full) {
#pragma unroll
        for (int p = 0; p < STAGES - 1; p++)
            if (first + p < full)
#pragma unroll
                for (int i = 0; i < kLoads; i++) request(ring + p * kStage, first + p, i);
        landed(full - first >= STAGES - 1);
#pragma unroll
        for (int i = 0; i < kFrags; i++) fragment(ring, 0, i);
        for (; b + STAGES - 1 < full; b++) {
            const uint32_t next = at + 1 == STAGES ? 0 : at + 1, to = at == 0 ? STAGES - 1 : at - 1;
            multiply(ring + at * kStage, ring + next * kStage, ring + to * kStage, b + STAGES - 1, yes, no);
            at = next;
        }
    }
    // The block with the rows' end comes through registers, read while the last whole ones are
    // multiplied and put into the ring behind them.
    i32x4 end[kLoads];
    auto put = [&](int8_t *stage) {
#pragma unroll
        for (int i = 0; i < kLoads; i++)
            *reinterpret_cast<i32x4 *>(stage + (wave * kLoads + i) * 1024 + lane * 16) = end[i];
    };
    if (full < last) {
#pragma unroll
        for (int i = 0; i < kLoads; i++) end[i] = load16_end(from[i], full * kBlock + chunk, g.K);
        if (first == full) {
            put(ring);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kFrags; i++) fragment(ring, 0, i);
        }
    }
    for (; b + 1 < last; b++) {
        const uint32_t next = at + 1 == STAGES ? 0 : at + 1;
        if (b + 1 == full) put(ring + next * kStage);
        multiply(ring + at * kStage, ring + next * kStage, nullptr, 0, no, no);
        at = next;
    }
    if (first < last) multiply(ring + at * kStage, nullptr, nullptr, 0, no, yes);

    // A lane holds groups of 4 neighbouring columns of one row: through LDS, MF rows of a wave at
    // a time, they become whole lines.
    __syncthreads();
    float *scale_b = reinterpret_cast<float *>(ring), *offset = scale_b + BN, *scale_a = offset + BN;
    int8_t *rest = reinterpret_cast<int8_t *>(scale_a + BM);
    for (uint32_t i = threadIdx.x; i < BN; i += WAVES * 64) {
        const uint32_t n = min(n0 + i, g.N - 1);
        scale_b[i] = g.sb[n];
        offset[i] = g.bias ? g.bias[n] : 0.f;
    }
    for (uint32_t i = threadIdx.x; i < BM; i += WAVES * 64) scale_a[i] = g.sa[min(m0 + i, g.M - 1)];
    __syncthreads();
    auto write = [&](auto *out0, size_t stride, auto value) {
        using O = std::remove_reference_t<decltype(*out0)>;
        constexpr int kCols = BN / WN, kPitch = kCols * (int)sizeof(O) + 16;
        constexpr int kPer = 16 / (int)sizeof(O), kLine = kCols / kPer;  // elements a lane, lanes a row
        int8_t *mine = rest + wave * (MF * kPitch);
        // A wave's lanes exchange values: its LDS accesses happen in their order, and the compiler may not change
        // it.  It looks at one lane, so the place that a lane reads from is kept from it: it must take every
        // reading for one of what was written.  (Fences between them also make it read the scales again for
        // every m: 300 x 20000 x 512 10.5 us, with fences 11.0.)
        uint32_t back = 0;
        asm("" : "+s"(back));
        const int8_t *lines = mine + back;
#pragma unroll
        for (int m = 0; m < TM; m++) {
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int q = 0; q < MF * MF / 256; q++) {
                    const uint32_t col = n * MF + q * 4 * kLanes + lane / MF * 4;
                    O v[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = value(acc[m][n][q * 4 + i], m * MF + lane % MF, col + i);
                    __builtin_memcpy(__builtin_assume_aligned(mine + lane % MF * kPitch + col * sizeof(O), 4 * sizeof(O)),
                                     v, sizeof(v));
                }
#pragma unroll
            for (int i = 0; i < (MF * kLine + 63) / 64; i++) {
                const uint32_t at = i * 64 + lane, r = at / kLine, c = at % kLine * kPer;
                if (MF * kLine % 64 && r >= MF) continue;
                const i32x4 v = *reinterpret_cast<const i32x4 *>(lines + r * kPitch + c * sizeof(O));
                const uint32_t row = m0 + wm + m * MF + r, col = n0 + wn + c;
                O *out = out0 + (size_t)row * stride + col;
                if (row < g.M && col + kPer <= g.N) {
                    __builtin_memcpy(out, &v, 16);
                } else if (row < g.M) {
                    using Part = Elements<kPer, O>;
                    const auto e = __builtin_bit_cast(Part, v);
#pragma unroll
                    for (int j = 0; j < kPer; j++)
                        if (col + j < g.N) out[j] = e.e[j];
                }
            }
        }
    };
    if (g.splits > 1)
        write(g.parts + (size_t)split * g.M * g.N, g.N, [&](int v, uint32_t, uint32_t) { return v; });
    else
        write(static_cast<T *>(g.out), g.out_stride, [&](int v, uint32_t r, uint32_t c) {
            return (T)((float)v * scale_a[wm + r] * scale_b[wn + c] + offset[wn + c]);
        });
}

// The sums of all splits, scaled: four columns a thread.  The partial sums are still in the
// caches, so a launch's 3 us are most of its time (64 x 2048 x 8192 in 4 parts: 11 us in all).
template <class T>
__global__ void __launch_bounds__(256)
k_join(MatmulArgs g) {
    const size_t quads = (g.N + 3) / 4, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t m = (uint32_t)(i / quads), n = (uint32_t)(i % quads) * 4;
    if (m >= g.M) return;
    const uint32_t count = min(4u, g.N - n);
    int sum[4] = {0, 0, 0, 0};
    const int *part = g.parts + (size_t)m * g.N + n;
    for (uint32_t s = 0; s < g.splits; s++, part += (size_t)g.M * g.N) {
        if (count == 4) {
            i32x4 v;
            __builtin_memcpy(&v, part, 16);
#pragma unroll
            for (int j = 0; j < 4; j++) sum[j] += v[j];
        } else {
            for (uint32_t j = 0; j < count; j++) sum[j] += part[j];
        }
    }
    T *out = static_cast<T *>(g.out) + (size_t)m * g.out_stride + n;
    const float sa = g.sa[m];
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (j < (int)count) out[j] = (T)((float)sum[j] * sa * g.sb[n + j] + (g.bias ? g.bias[n + j] : 0.f));
}

constexpr size_t kMostK = 131071;

// The shapes of k_tiles and what one block of K costs them, in us (measured, gfx950, over K from 512
// to 8192): `alone` with one tile a CU, `pair` with two, `each` for every one of more.
struct Shape {
    uint32_t rows, cols;
    float alone, pair, each;
};
enum { kSmall, kSquare, kWide, kLarge, kBroad, kHuge, kTall, kShapes };
constexpr Shape shapes[kShapes] = {
    {32, 64, .19f, .25f, .12f}, {64, 64, .30f, .48f, .23f}, {64, 128, .47f, .70f, .35f},
    {128, 128, .56f, 1.12f, .56f}, {128, 192, .66f, 1.32f, .66f}, {128, 256, .80f, 1.60f, .80f}, {256, 128, .80f, 1.55f, .76f}};

// How a product is formed: `few` by k_few_rows, else by tiles of `shape`, K in `splits` parts.
struct Plan {
    bool few;
    int shape;
    uint32_t splits;
};

// The plan of least estimated time: that of the products, or of reading b, a little more for every
// row of tiles that reads it again.  The estimates order the plans; the launch, the rows' end and odd strides, which
// all plans of a size pay, are not in them (777 x 5003 x 2050: 11 us estimated, 20 measured).  Few rows and few columns go to k_few_rows (1 x 8192 x 2048: 6.3 us,
// tiles 6.7; 1 x 32768 x 2048: 16 us, tiles 14).  K is split where tiles are too few for the card and the sums are
// long enough to pay for the second launch and the partial sums (64 x 2048 x 8192: 15 us whole, 11 us in 4).
Plan plan_matmul(size_t M, size_t N, size_t K) {
    if (M <= 16 && N <= 16384) return {true, 0, 1};
    const float blocks = (float)((K + kBlock - 1) / kBlock), memory = 5e6f;  // bytes a us
    Plan best{false, 0, 1};
    float least = INFINITY;
    for (int i = 0; i < kShapes; i++) {
        const Shape &s = shapes[i];
        if (s.rows > 32 && M <= s.rows / 2) continue;  // half a tile or more of nothing
        const size_t down = (M + s.rows - 1) / s.rows, tiles = down * ((N + s.cols - 1) / s.cols);
        const float reading = ((float)N * K * (1 + .15f * (down - 1)) + (float)M * K) / memory;
        for (uint32_t splits = 1; splits <= 8; splits *= 2) {
            if (splits > 1 && (tiles * splits > 512 || blocks < 8 * splits)) break;
            const size_t on_cu = (tiles * splits + 255) / 256;
            const float block = on_cu <= 1 ? s.alone : on_cu == 2 ? s.pair : on_cu * s.each;
            const float join = splits == 1 ? 0.f : 4.f + (float)splits * M * N * 8 / memory;
            const float time = std::max(block * blocks / splits, reading) + join;
            if (time < least) {
                least = time;
                best = {false, i, splits};
            }
        }
    }
    return best;
}

template <class T, int MF, int BM, int BN, int WM, int WN, int STAGES>
void launch_tiles(const MatmulArgs &g, hipStream_t s) {
    const auto kernel = &k_tiles<T, MF, BM, BN, WM, WN, STAGES>;
    const size_t jobs = (size_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN) * g.splits;
    require(jobs < 1u << 22, "pfa_int8_matmul: more outputs than one launch can form");
    hipLaunchKernelGGL(kernel, dim3((uint32_t)((jobs + 7) / 8 * 8)), dim3(WM * WN * 64), 0, s, g);
    if (g.splits > 1)
        hipLaunchKernelGGL(k_join<T>, dim3((uint32_t)(((size_t)g.M * ((g.N + 3) / 4) + 255) / 256)), dim3(256), 0, s, g);
}

template <class T>
void matmul(const MatmulArgs &g, const Plan &p, hipStream_t s) {
    if (p.few) {
        hipLaunchKernelGGL(k_few_rows<T>, dim3((g.N + 15) / 16), dim3(kFewWaves * 64), 0, s, g);
        return;
    }
    switch (p.shape) {
        case kSmall: return launch_tiles<T, 16, 32, 64, 2, 2, 6>(g, s);
        case kSquare: return launch_tiles<T, 16, 64, 64, 2, 2, 4>(g, s);
        case kWide: return launch_tiles<T, 16, 64, 128, 1, 4, 3>(g, s);
        case kLarge: return launch_tiles<T, 32, 128, 128, 2, 2, 3>(g, s);
        case kBroad: return launch_tiles<T, 16, 128, 192, 2, 4, 3>(g, s);
        case kHuge: return launch_tiles<T, 16, 128, 256, 2, 4, 3>(g, s);
        default: return launch_tiles<T, 16, 256, 128, 4, 2, 3>(g, s);
    }
}

}  // namespace

}  // namespace pfa

using namespace pfa;

extern "C" {

int pfa_matmul_workspace(size_t M, size_t N, size_t K, size_t *bytes) {
    return guarded([&] {
        require(bytes != nullptr, "null argument");
        require(K <= kMostK, "pfa_matmul_workspace: sums of more than 131071 products can pass 32 bits");
        require(M <= 0x7fffffffu && N <= 0x7fffffffu, "pfa_matmul_workspace: more than 2^31 - 1 rows");
        const Plan p = plan_matmul(M, N, K);
        *bytes = p.splits > 1 && M && N ? p.splits * M * N * 4 : 0;
    });
}

int pfa_matmul_plan(size_t M, size_t N, size_t K, size_t *tile_rows, size_t *tile_cols, size_t *splits) {
    return guarded([&] {
        require(tile_rows && tile_cols && splits, "null argument");
        require(K <= kMostK, "pfa_matmul_plan: sums of more than 131071 products can pass 32 bits");
        require(M <= 0x7fffffffu && N <= 0x7fffffffu, "pfa_matmul_plan: more than 2^31 - 1 rows");
        const Plan p = plan_matmul(M, N, K);
        *tile_rows = p.few ? 0 : shapes[p.shape].rows;
        *tile_cols = p.few ? 16 : shapes[p.shape].cols;
        *splits = p.splits;
    });
}

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
        const Plan p = plan_matmul(M, N, K);
        const size_t need = p.splits > 1 ? p.splits * M * N * 4 : 0;
        require(workspace_bytes >= need, "pfa_int8_matmul: the workspace needs " + std::to_string(need) + " bytes");
        require(((uintptr_t)workspace & 15) == 0, "pfa_int8_matmul: the workspace is not aligned to 16 bytes");
        const MatmulArgs g{a, b, a_scales, b_scales, bias, out, a_stride, b_stride, out_stride, (int *)workspace,
                           (uint32_t)M, (uint32_t)N, (uint32_t)K, p.splits};
        with_type(type, [&](auto t) { matmul<decltype(t)>(g, p, as_stream(stream)); });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
