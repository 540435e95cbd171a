// Products of 8-bit floating point codes (e4m3) with a scale for each 128 places of a row of a (a token of
// the activations) and for each 128 rows and 128 places of b (output channels of the weights):
//   out[m][n] = sum_j (sum_{k in block j} a[m][k] b[n][k]) sa[m][j] sb[n / 128][j] + bias[n]
// Sums of a block and of the blocks are held in 32-bit floats, and one rounding leads to the output's type.
//
// Products for 16-bit outputs are formed by the 8-bit matrix instruction.  It takes eight neighbouring products at a
// time and aligns them by the products of their codes' powers of two (a code below 2^-6 counts as 2^-6 there; products
// that are 0 do not count): with P the largest of these, each is cut towards 0 to a multiple of 2^-13 P.  Then it adds in
// 32 bits.  (Measured, number by number.)  Seven of eight lose less than 2^-13 P each: 1.53 2^-13 of the result at most, in
// the mean square over signs; 1.5 10^-5 on normal codes, 8 10^-5 where some places of a are 200 times the others, sums of one
// sign come out 2.6 10^-6 low.  A 16-bit output is rounded at 2^-8 or 2^-11, 1.7 10^-3 or 2.1 10^-4 in the mean square.
// Where large products cancel, what was cut beside them is missing.  32-bit outputs show it, so
// their codes are widened to 16-bit floats (exact) and multiplied at half that rate, every product whole and every sum in 32
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
    float *parts;          // [splits][M][N] sums, with more than one split of K
    uint32_t M, N, K, splits;
};

// 32 codes of a row: places 16 i and 64 + 16 i of a block, or 32 neighbouring ones; the same of either operand
struct Codes {
    i32x4 v[2];
};
// the same as 16-bit floats, eight at a time
struct Widened {
    f16x8 v[4];
    __device__ __forceinline__ Widened() {}
    __device__ __forceinline__ explicit Widened(const Codes &c) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f16x2 h[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned w = (unsigned)c.v[i / 2][i % 2 * 2 + j / 2];
                h[j] = j % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)
                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
            }
            v[i] = f16x8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
        }
    }
};

// 16 x 16 sums of 128 products.  A lane holds codes of row lane % 16 of either operand, and of the sums row
// lane % 16 of a and 4 neighbouring rows of b.
__device__ __forceinline__ f32x4 block_sums(const Codes &a, const Codes &b) {
    const i32x8 fa = {a.v[0][0], a.v[0][1], a.v[0][2], a.v[0][3], a.v[1][0], a.v[1][1], a.v[1][2], a.v[1][3]};
    const i32x8 fb = {b.v[0][0], b.v[0][1], b.v[0][2], b.v[0][3], b.v[1][0], b.v[1][1], b.v[1][2], b.v[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb, fa, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 block_sums(const Widened &a, const Widened &b) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; i++) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(b.v[i], a.v[i], sum, 0, 0, 0);
    return sum;
}

// BYTES of memory a lane to a wave's 64 BYTES places in LDS: from p (scalar), `from` (scalar) and `own`, the latter two 32
// bits in all.  Loads by such offsets are told apart from LDS accesses by the compiler's waits; by addresses of 64 bits
// they are not, and the products of a block then wait for all operands of the next.
template <int BYTES>
__device__ __forceinline__ void load_to_lds(const void *p, uint32_t from, uint32_t own, int8_t *lds) {
    static_assert(BYTES == 4 || BYTES == 16, "a load's sizes");
#ifdef __HIP_DEVICE_COMPILE__  // the host's pass does not know the type of a buffer's description
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, -1, 0x20000);
    const auto to = (__attribute__((address_space(3))) uint32_t *)lds;
    if (BYTES == 16)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, to, 16, own, from, 0, 0);
    else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, to, 4, own, from, 0, 0);
#endif
}

// A wave's 16 x 16 sums in LDS, where the waves' are added in their order.  A lane has row lane % 16 of a, 4 columns.
constexpr int kFewWaves = 8;
using FewSums = float[kFewWaves][16][17];

template <class T>
__device__ __forceinline__ void few_outputs(const Fp8Args &g, FewSums &sums, const f32x4 &acc, uint32_t m0, uint32_t n0) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
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

// 16 x 16 outputs a workgroup: b is streamed, its waves take the blocks of K in turn.  Lanes side by side read a row's
// chunks and the matrix instruction wants them to have rows side by side, so blocks go through LDS, two of a wave's
// own on their way at once, and no wave waits for another.  (More on their way leave LDS for one workgroup a CU instead
// of two: 1 x 131072 x 4096 109 us with three.)  ROWS of a (8 or 16) are loaded; the sums of rows behind the matrix are
// dropped.  Bound by memory: 1 x 131072 x 4096 92 us, to float32 88 (6.1 TB/s); 1 x 4096 x 14336 12.1 us (4.9 TB/s),
// 1 x 4096 x 4096 5.6 us from memory.  Where b is small by the launch and one trip to memory: 1 x 128 x 4096 3.1 us.
constexpr int kFewRing = 2;

template <class T, int ROWS>
__global__ void __launch_bounds__(kFewWaves * 64)
k_fp8_few(Fp8Args g) {
    using Operand = std::conditional_t<std::is_same_v<T, float>, Widened, Codes>;
    // a block's 16 rows of b, its rows of a, each as in k_fp8_tiles, a's scales and b's
    constexpr int kA = 16 * kBlock, kScales = kA + ROWS * kBlock, kSlot = kScales + 512, kLoads = 2 + ROWS / 8 + 2;
    constexpr int kLds = kFewWaves * kFewRing * kSlot;
    static_assert(kLds <= 160 * 1024 && kLds >= (int)sizeof(FewSums), "a CU's LDS");
    __shared__ __align__(1024) int8_t held[kLds];
    uint32_t start = 0;
    asm("" : "+s"(start));
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    int8_t *mine = held + start + wave * (kFewRing * kSlot);
    const uint32_t n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
    const int8_t *rows_a = g.a + m0 * g.a_stride, *rows_b = g.b + n0 * g.b_stride;
    const float *sa = g.sa + m0 * g.sa_row, *sb = g.sb + n0 / kBlock * g.sb_row;
    // a load is 8 rows, behind the matrix its last one
    const uint32_t chunk = (lane % 8 ^ lane / 8) * 16, last_a = g.M - 1 - m0, last_b = g.N - 1 - n0;
    uint32_t own_a[ROWS / 8], own_b[2];
#pragma unroll
    for (int i = 0; i < ROWS / 8; i++) own_a[i] = min(lane / 8 + i * 8, last_a) * (uint32_t)g.a_stride + chunk;
#pragma unroll
    for (int i = 0; i < 2; i++) own_b[i] = min(lane / 8 + i * 8, last_b) * (uint32_t)g.b_stride + chunk;
    const uint32_t own_scale = min(lane % 16, last_a) * (uint32_t)g.sa_row * 4;
    auto request = [&](int8_t *slot, uint32_t block) {
#pragma unroll
        for (int i = 0; i < 2; i++) load_to_lds<16>(rows_b, block * kBlock, own_b[i], slot + i * 1024);
#pragma unroll
        for (int i = 0; i < ROWS / 8; i++) load_to_lds<16>(rows_a, block * kBlock, own_a[i], slot + kA + i * 1024);
        load_to_lds<4>(sa + block * g.sa_block, 0, own_scale, slot + kScales);
        load_to_lds<4>(sb + block * g.sb_block, 0, 0, slot + kScales + 256);  // by registers it waits for all loads
    };
    const uint32_t in_row = (lane / 16 ^ lane % 8) * 16, other = in_row ^ 64;
    auto read = [&](const int8_t *row) {
        Codes c;
        c.v[0] = *reinterpret_cast<const i32x4 *>(row + in_row);
        c.v[1] = *reinterpret_cast<const i32x4 *>(row + other);
        return c;
    };
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](const Codes &fa, const Codes &fb, float scale) {
        const f32x4 p = block_sums(Operand(fa), Operand(fb));
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = fmaf(p[i], scale, acc[i]);
    };
    const uint32_t whole = g.K / kBlock;
    auto fence = [] { asm volatile("" ::: "memory"); };
#pragma unroll
    for (int p = 0; p < kFewRing; p++)
        if (wave + p * kFewWaves < whole) request(mine + p * kSlot, wave + p * kFewWaves);
    // the wave whose turn it is takes the rows' end, while its blocks are on their way
    if (const uint32_t j = whole; j * kBlock < g.K && j % kFewWaves == wave) {
        const uint32_t at = lane / 16 * 16;
        const int8_t *pa = rows_a + min(lane % 16, last_a) * g.a_stride, *pb = rows_b + min(lane % 16, last_b) * g.b_stride;
        Codes fa, fb;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            fb.v[h] = load16_end(pb, j * kBlock + at + h * 64, g.K);
            fa.v[h] = load16_end(pa, j * kBlock + at + h * 64, g.K);
        }
        add(fa, fb, sa[min(lane % 16, last_a) * g.sa_row + j * g.sa_block] * sb[j * g.sb_block]);
    }
    int8_t *slot = mine;
    for (uint32_t j = wave; j < whole; j += kFewWaves) {
        // this block has landed: of the loads behind it all may be on their way, or at the end none
        fence();
        if (j + (kFewRing - 1) * kFewWaves < whole)
            __builtin_amdgcn_s_waitcnt(0x0f70 | (kLoads * (kFewRing - 1) & 15) | kLoads * (kFewRing - 1) >> 4 << 14);
        else
            __builtin_amdgcn_s_waitcnt(0x0f70);
        fence();
        const Codes fa = read(slot + kA + lane % ROWS * kBlock), fb = read(slot + lane % 16 * kBlock);
        const float *scales = reinterpret_cast<const float *>(slot + kScales);
        const float scale = scales[lane] * scales[64];
        // and has been read, before its place is another's
        fence();
        __builtin_amdgcn_s_waitcnt(0xc07f);
        fence();
        if (j + kFewRing * kFewWaves < whole) request(slot, j + kFewRing * kFewWaves);
        slot = slot == mine + (kFewRing - 1) * kSlot ? mine : slot + kSlot;
        add(fa, fb, scale);
    }
    __syncthreads();
    few_outputs<T>(g, *reinterpret_cast<FewSums *>(held + start), acc, m0, n0);
}

// The same by registers, for rows so far apart that 32 bits do not hold the offsets of 16: a load of 16 rows by lanes
// side by side takes 64 clocks where whole lines take 16 (1 x 4096 x 4096 from memory 7.8 us).
constexpr int kFarUnroll = 4;

template <class T>
__global__ void __launch_bounds__(kFewWaves * 64)
k_fp8_far(Fp8Args g) {
    using Operand = std::conditional_t<std::is_same_v<T, float>, Widened, Codes>;
    __shared__ FewSums sums;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, at = lane / 16 * 32;
    const uint32_t n0 = blockIdx.x * 16, m0 = blockIdx.y * 16, am = min(m0 + lane % 16, g.M - 1);
    const int8_t *pa = g.a + am * g.a_stride, *pb = g.b + min(n0 + lane % 16, g.N - 1) * g.b_stride;
    const float *sa = g.sa + am * g.sa_row, *sb = g.sb + n0 / kBlock * g.sb_row;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](const Codes &fa, const Codes &fb, float scale) {
        const f32x4 p = block_sums(Operand(fa), Operand(fb));
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = fmaf(p[i], scale, acc[i]);
    };
    const uint32_t blocks = g.K / kBlock;
    uint32_t j = wave;
    for (; j + (kFarUnroll - 1) * kFewWaves < blocks; j += kFarUnroll * kFewWaves) {
        Codes fa[kFarUnroll], fb[kFarUnroll];
        float sj[kFarUnroll], tj[kFarUnroll];
#pragma unroll
        for (int u = 0; u < kFarUnroll; u++) {
            const uint32_t k = j + u * kFewWaves;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                fb[u].v[h] = load16(pb, k * kBlock + at + h * 16);
                fa[u].v[h] = load16(pa, k * kBlock + at + h * 16);
            }
            sj[u] = sa[k * g.sa_block];
            tj[u] = sb[k * g.sb_block];
        }
#pragma unroll
        for (int u = 0; u < kFarUnroll; u++) add(fa[u], fb[u], sj[u] * tj[u]);
    }
    // what is left: whole blocks, and the wave whose turn it is takes the rows' end
    for (; j * kBlock < g.K; j += kFewWaves) {
        Codes fa, fb;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            fb.v[h] = load16_end(pb, j * kBlock + at + h * 16, g.K);
            fa.v[h] = load16_end(pa, j * kBlock + at + h * 16, g.K);
        }
        add(fa, fb, sa[j * g.sa_block] * sb[j * g.sb_block]);
    }
    few_outputs<T>(g, sums, acc, m0, n0);
}

// The order of a wave's TM x TN products of a block: its first columns one by one, then the last `kRest` row by row.
// b's operands take kHeld registers' places in turn and are read kRest columns ahead; a's have their last product one
// row after the other, so the reading of the next block's is spread over the last columns' products.
template <int TM, int TN>
struct Order {
    static constexpr int kRest = TN > 3 ? 3 : TN > 1 ? TN - 1 : 1, kHeld = TN > 1 ? kRest + 1 : 1;
    static constexpr int kTurn = TM * (TN - kRest);  // products in columns
    static_assert(TN % kHeld == 0, "b's operands come back to their places");
    int m[TM * TN] = {}, n[TM * TN] = {};
    constexpr Order() {
        for (int j = 0; j < TM * TN; j++) {
            m[j] = j < kTurn ? j % TM : (j - kTurn) / kRest;
            n[j] = j < kTurn ? j / TM : TN - kRest + (j - kTurn) % kRest;
        }
    }
};

// Many rows: BM x BN outputs a workgroup of WM x WN waves.  Blocks of 128 places of K go through LDS in a ring of
// STAGES blocks by loads that write LDS themselves.  A block's rows are 128 bytes, 8 chunks of 16, and chunk c of
// row r stands in place c ^ (r mod 8), so that a wave's reading of one chunk of 8 rows touches every bank once; behind
// them stand the block's scales, one load of 64 numbers a wave.
//
// A block is one matrix instruction deep (four of the widened codes), and its sums are added up with their scale kLag
// products later, in the vector unit's time beside the matrix unit's.  A wave forms its first columns one after the
// other and the last ones row by row (Order): a's operands are held, b's read ahead.  A block's barrier stands behind
// the last product in columns, when all of the block is in registers; the row-wise products, whose operands are there,
// cover it, the requests of the block that goes to this one's place, and the reading of the next block's operands.
//
// Measured: 4096 x 16384 x 4096 250-257 us (2.2 PFLOP/s), 8192^3 471 us (2.33), where a library's product without
// scales by blocks takes 229 and 420.  A block of 256 x 256 takes 1.6 us, of it .93 the matrix instructions: LDS
// gives a wave's reading 167 bytes a clock and takes the loads' 64, one after the other, .95 us in all, and the clock
// falls under the load.  Without the scaling 220 us.  32-bit outputs: 8192^3 890 us (1.24 PFLOP/s), bound by the
// vector unit, two conversions of 4 clocks for each matrix instruction of 16.  Few rows: by reading b (20 x 131072 x
// 4096: 95 us to 16 bits, 102 to 32, 5.3 TB/s).  Odd sizes and odd strides: 777 x 5003 x 2050 21-24 us, of it 2.5
// the rows' end and 3.3 rows that begin anywhere (two cache lines a row of a block); 2048 places in whole lines 15.
template <class T, int BM, int BN, int WM, int WN, int STAGES>
__global__ void __launch_bounds__(WM * WN * 64)
k_fp8_tiles(Fp8Args g) {
    constexpr bool kWide = std::is_same_v<T, float>;
    constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, kProducts = TM * TN;
    constexpr int kRows = BM + BN, kCodes = kRows * kBlock;
    constexpr int kStage = kCodes + WAVES * 256, kScaleB = (BM + 63) / 64 * 64;  // a's scales, then b's
    constexpr int kLoads = kRows / 8 / WAVES;  // a wave's load is 8 rows, 1 KiB
    static_assert(kRows % (8 * WAVES) == 0 && BM % 8 == 0, "whole loads");
    static_assert(kScaleB < WAVES * 64, "a load of scales each wave");
    static_assert(BN % 64 == 0 && 128 % (BN / WN) == 0 && 256 % BN == 0, "a wave's columns share their scales");
    // the ring, and in its place behind the products a line of outputs a wave
    constexpr int kRing = kStage * STAGES, kLines = WAVES * 16 * (BN / WN * 4 + 16);
    constexpr int kLds = kRing > kLines ? kRing : kLines;
    static_assert(kLds <= 160 * 1024, "a CU's LDS");
    __shared__ __align__(1024) int8_t held[kLds];
    uint32_t start = 0;
    asm("" : "+s"(start));  // where the ring begins is not told to the compiler: it moves sums between registers otherwise
    int8_t *ring = held + start;
    // a wave's number is said to be uniform: addresses of loads and places in the ring are then scalar
    const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t down = (g.M + BM - 1) / BM, across = (g.N + BN - 1) / BN;
    // workgroups are dealt to the 8 XCDs in turn: each XCD gets a run of tiles, in groups of some tiles of rows, so that
    // its L2 holds what its tiles share
    constexpr uint32_t kGroup = BM >= 256 ? 6 : 8;
    const uint32_t jobs = down * across * g.splits, each = (jobs + 7) / 8;
    const uint32_t job = blockIdx.x % 8 * each + blockIdx.x / 8;
    if (job >= jobs || blockIdx.x / 8 >= each) return;
    const uint32_t split = job % g.splits, t = job / g.splits;
    const uint32_t group = t / (kGroup * across), height = min(kGroup, down - group * kGroup);
    const uint32_t m0 = (group * kGroup + t % (kGroup * across) % height) * BM, n0 = t % (kGroup * across) / height * BN;
    const uint32_t wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    // this workgroup's blocks of K
    const uint32_t all = (g.K + kBlock - 1) / kBlock, share = (all + g.splits - 1) / g.splits;
    const uint32_t first = min(split * share, all), last = min(first + share, all);
    const uint32_t full = max(min(last, g.K / kBlock), first);  // all but a block with the rows' end

    // A load is 8 rows of a or of b; behind the last row of the matrix, that one again.  Addresses are a tile's first row
    // (scalar), a load's first row and the block (scalar) and a lane's own row and chunk, the latter two 32 bits in all.
    const uint32_t chunk = (lane % 8 ^ lane / 8) * 16;
    const int8_t *const rows_a = g.a + m0 * g.a_stride, *const rows_b = g.b + n0 * g.b_stride;
    uint32_t stride_a = (uint32_t)g.a_stride, stride_b = (uint32_t)g.b_stride;
    asm("" : "+s"(stride_a), "+s"(stride_b));  // in registers: read from the launch's arguments they wait for LDS, too
    constexpr bool kTight = kProducts >= 32;  // the largest tiles: 128 sums a lane
    uint32_t from[kLoads], more_rows[kLoads], held_own[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const uint32_t r = (wave * kLoads + i) * 8;
        const bool of_a = r < BM;
        const uint32_t stride = of_a ? stride_a : stride_b, end = of_a ? g.M - 1 - m0 : g.N - 1 - n0;
        const uint32_t row = min(of_a ? r : r - BM, end);
        from[i] = row * stride;
        more_rows[i] = min(end - row, 7u);
        held_own[i] = min(lane / 8, end - row) * stride + chunk;
    }
    auto own = [&](int i) {  // formed anew where the registers are short; a stride has 24 bits
        if (!kTight) return held_own[i];
        uint32_t l = lane;
        asm volatile("" : "+v"(l));
        return __umul24(min(l / 8, more_rows[i]), (wave * kLoads + i) * 8 < BM ? stride_a : stride_b) +
               (l % 8 ^ l / 8) * 16;
    };
    // Scales: a load is 64 of a's rows, or one for each 64 columns
    const bool scale_of_a = wave * 64 < kScaleB;
    const float *scale_from = scale_of_a ? g.sa + m0 * g.sa_row : g.sb + n0 / kBlock * g.sb_row;
    const size_t scale_step = scale_of_a ? g.sa_block : g.sb_block;
    const uint32_t scale_own =
        scale_of_a ? min(wave * 64 + lane, g.M - 1 - m0) * (uint32_t)g.sa_row * 4
                   : (min(n0 + min(lane, (uint32_t)(BN - 1) / 64) * 64, g.N - 1) / kBlock - n0 / kBlock) *
                         (uint32_t)g.sb_row * 4;
    // Rows a power of two apart start in the same memory channel.  Where tiles share no rows of b, each begins with
    // another block.
    const uint32_t whole = full - first, turn = down == 1 && whole ? t * 3 % whole : 0;
    auto turned = [&](uint32_t block) {
        block += turn;
        return block - (block < full ? 0 : whole);
    };
    auto request = [&](int8_t *stage, uint32_t block, int i) {  // i == kLoads: the scales
        if (i < kLoads)
            load_to_lds<16>((wave * kLoads + i) * 8 < BM ? rows_a : rows_b, from[i] + block * kBlock, own(i),
                            stage + (wave * kLoads + i) * 1024);
        else
            load_to_lds<4>(scale_from + block * scale_step, 0, scale_own, stage + kCodes + wave * 256);
    };
    constexpr int kAsks = kLoads + 1;

    f32x4 acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; m++)
#pragma unroll
        for (int n = 0; n < TN; n++) acc[m][n] = {0.f, 0.f, 0.f, 0.f};
    using Products = Order<TM, TN>;
    Codes fa[TM], fb[Products::kHeld];
    float sa[TM], sb = 0.f;
    // a lane's places in a stage: chunks lane / 16 and 4 + lane / 16 of row lane % 16 of its wave's first 16 rows
    const uint32_t in_row = (lane / 16 ^ lane % 8) * 16, other = in_row ^ 64;
    const uint32_t of_a = (wm + lane % 16) * kBlock, of_b = (BM + wn + lane % 16) * kBlock;
    auto read = [&](const int8_t *place, int i) {
        Codes c;
        c.v[0] = *reinterpret_cast<const i32x4 *>(place + in_row + i * 16 * kBlock);
        c.v[1] = *reinterpret_cast<const i32x4 *>(place + other + i * 16 * kBlock);
        return c;
    };
    auto read_a = [&](const int8_t *stage, int m) {
        fa[m] = read(stage + of_a, m);
        sa[m] = reinterpret_cast<const float *>(stage + kCodes)[wm + lane % 16 + m * 16];
    };
    auto read_b = [&](const int8_t *stage, int n) {
        fb[n % Products::kHeld] = read(stage + of_b, n);
        if (n == 0) sb = reinterpret_cast<const float *>(stage + kCodes)[kScaleB + wn / 64];
    };
    // every wave's part of the next block has landed, and all are done with reading this one
    auto landed = [&](bool more) {
        constexpr int kLeft = STAGES > 2 ? kAsks * (STAGES - 2) : 0;  // loads of the blocks behind it
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
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    // The products of a block whose first operands are in registers.  `ends`: there is no next block.  `asks`: block
    // `ahead` goes to this block's own place.
    auto multiply = [&](int8_t *mine, const int8_t *next, uint32_t ahead, bool more, auto asks, auto ends, auto before) {
        constexpr Products order;
        constexpr int kHeld = Products::kHeld, kLag = kTight ? 4 : kProducts > 3 ? 3 : kProducts - 1;
        constexpr int kFirst = Products::kTurn > 0 ? Products::kTurn - 1 : 0;  // the product that the barrier stands behind
        f32x4 sum[kLag + 1];
        float scale[TM];
        const float scale_b = sb;
        std::conditional_t<kWide, Widened, Codes> wa[TM], wb[kHeld];
        auto add = [&](int j) {
            f32x4 &to = acc[order.m[j]][order.n[j]];
#pragma unroll
            for (int i = 0; i < 4; i++) to[i] = fmaf(sum[j % (kLag + 1)][i], scale[order.m[j]], to[i]);
        };
#pragma unroll
        for (int j = 0; j < kProducts; j++) {
            const int m = order.m[j], n = order.n[j], at_b = n % kHeld;
            if (n == 0) scale[m] = sa[m] * scale_b;
            if constexpr (kWide) {
                if (n == 0) wa[m] = Widened(fa[m]);
                if (m == 0) wb[at_b] = Widened(fb[at_b]);
                sum[j % (kLag + 1)] = block_sums(wa[m], wb[at_b]);
            } else {
                sum[j % (kLag + 1)] = block_sums(fa[m], fb[at_b]);
            }
            // a column that comes later, in the place of the one before this
            if (m == 0 && n > 0 && n + kHeld - 1 < TN && j < Products::kTurn) read_b(mine, n + kHeld - 1);
            if (j == kFirst && !ends) {
                before();
                landed(more);
            }
            if (!ends) {
                if (j == kFirst && (TN > kHeld || TN == 1)) read_b(next, 0);
                if (TN == kHeld && TN > 1 && n == 0 && m + 1 == TM) read_b(next, 0);
                if (n + 1 == TN) read_a(next, m);
                if (m + 1 == TM && n > 0 && j >= Products::kTurn) read_b(next, n - (TN - kHeld));
            }
            if (asks && j >= kFirst) {
                constexpr int kPlaces = kProducts - kFirst;
#pragma unroll
                for (int i = 0; i < kAsks; i++)
                    if (i * kPlaces / kAsks == j - kFirst) request(mine, ahead, i);
            }
            if (j >= kLag) add(j - kLag);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = kProducts - kLag; j < kProducts; j++) add(j);
    };
    auto nothing = [] {};
    uint32_t at = 0, b = first;
    auto stage = [&](uint32_t i) { return ring + i * kStage; };
    // The block with the rows' end comes through registers, read while the last whole ones are multiplied.  The largest
    // tiles have none to spare, and take whole blocks only.
    i32x4 end[kLoads];
    float end_scale;
    auto take_end = [&] {
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const bool of_a = (wave * kLoads + i) * 8 < BM;
            const int8_t *row = (of_a ? rows_a : rows_b) + from[i] + (own(i) - chunk);
            end[i] = load16_end(row, full * kBlock + chunk, g.K);
        }
        end_scale = *reinterpret_cast<const float *>(reinterpret_cast<const int8_t *>(scale_from + full * scale_step) + scale_own);
    };
    auto put_end = [&](int8_t *to) {
#pragma unroll
        for (int i = 0; i < kLoads; i++)
            *reinterpret_cast<i32x4 *>(to + (wave * kLoads + i) * 1024 + lane * 16) = end[i];
        *reinterpret_cast<float *>(to + kCodes + threadIdx.x * 4) = end_scale;
    };
    auto read_all = [&](const int8_t *from_stage) {
#pragma unroll
        for (int m = 0; m < TM; m++) read_a(from_stage, m);
#pragma unroll
        for (int n = 0; n < Products::kHeld; n++) read_b(from_stage, n);
    };
    if (first < full) {
#pragma unroll
        for (int p = 0; p < STAGES; p++)
            if (first + p < full)
#pragma unroll
                for (int i = 0; i < kAsks; i++) request(stage(p), turned(first + p), i);
        if (whole >= STAGES) {
            constexpr int kLeft = kAsks * (STAGES - 1);
            static_assert(kLeft < 64, "the counter's range");
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0x0070 | (kLeft & 15) | kLeft >> 4 << 14);
        } else {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0x0070);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read_all(stage(0));
        // Nothing of LDS is on its way where the loop begins, so the compiler's waits in it are for what each
        // product needs and not for all that was read before the loop in another order.
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);
        asm volatile("" ::: "memory");
        for (; b + STAGES < full; b++) {
            const uint32_t next = at + 1 == STAGES ? 0 : at + 1;
            multiply(stage(at), stage(next), turned(b + STAGES), true, yes, no, nothing);
            at = next;
        }
    }
    if (!kTight && full < last) {
        take_end();
        if (first == full) {
            put_end(ring);
            __syncthreads();
            read_all(ring);
        }
    }
    for (; b + 1 < last; b++) {
        const uint32_t next = at + 1 == STAGES ? 0 : at + 1;
        multiply(stage(at), stage(next), 0, b + STAGES - 1 < full, no, no, [&] {
            if (!kTight && b + 1 == full) put_end(stage(next));
        });
        at = next;
    }
    if (first < last) multiply(stage(at), nullptr, 0, false, no, yes, nothing);

    // A lane holds groups of 4 neighbouring columns of one row: through LDS, 16 rows of a wave at a time, they become
    // whole lines.
    __syncthreads();
    auto write = [&](auto *out0, size_t stride, const float *bias) {
        using O = std::remove_reference_t<decltype(*out0)>;
        constexpr int kCols = BN / WN, kPitch = kCols * (int)sizeof(O) + 16;
        constexpr int kPer = 16 / (int)sizeof(O), kLine = kCols / kPer;  // elements a lane, lanes a row
        int8_t *mine = ring + wave * (16 * kPitch);
        // A wave's lanes exchange values: its LDS accesses happen in their order, and the compiler, which looks at one
        // lane, must take every reading for one of what was written.
        uint32_t back = 0;
        asm("" : "+s"(back));
        const int8_t *lines = mine + back;
        if (bias) {
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float add = bias[min(n0 + wn + n * 16 + lane / 16 * 4 + i, g.N - 1)];
#pragma unroll
                    for (int m = 0; m < TM; m++) acc[m][n][i] += add;
                }
        }
#pragma unroll
        for (int m = 0; m < TM; m++) {
#pragma unroll
            for (int n = 0; n < TN; n++) {
                O v[4];
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = (O)acc[m][n][i];
                __builtin_memcpy(__builtin_assume_aligned(mine + lane % 16 * kPitch + (n * 16 + lane / 16 * 4) * sizeof(O), 4 * sizeof(O)),
                                 v, sizeof(v));
            }
#pragma unroll
            for (int i = 0; i < (16 * kLine + 63) / 64; i++) {
                const uint32_t place = i * 64 + lane, r = place / kLine, c = place % kLine * kPer;
                if (16 * kLine % 64 && r >= 16) continue;
                const i32x4 v = *reinterpret_cast<const i32x4 *>(lines + r * kPitch + c * sizeof(O));
                const uint32_t row = m0 + wm + m * 16 + r, col = n0 + wn + c;
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
        write(g.parts + (size_t)split * g.M * g.N, g.N, (const float *)nullptr);
    else
        write(static_cast<T *>(g.out), g.out_stride, g.bias);
}

// The sums of all splits, in their order, and the bias: four columns a thread.  They come from the caches (320 x 4096
// in 4: 5 us with its launch).
template <class T>
__global__ void __launch_bounds__(256)
k_fp8_join(Fp8Args g) {
    const size_t quads = (g.N + 3) / 4, i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t m = i / quads;
    const uint32_t n = (uint32_t)(i % quads) * 4;
    if (m >= g.M) return;
    const uint32_t count = min(4u, g.N - n);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const float *part = g.parts + m * g.N + n;
    for (uint32_t s = 0; s < g.splits; s++, part += (size_t)g.M * g.N) {
        if (count == 4) {
            float v[4];
            __builtin_memcpy(v, part, 16);
#pragma unroll
            for (int j = 0; j < 4; j++) sum[j] += v[j];
        } else {
            for (uint32_t j = 0; j < count; j++) sum[j] += part[j];
        }
    }
    T *out = static_cast<T *>(g.out) + m * g.out_stride + n;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (j < (int)count) out[j] = (T)(sum[j] + (g.bias ? g.bias[n + j] : 0.f));
}

// The shapes of k_fp8_tiles and what they cost a CU, in us (measured, gfx950, over K from 512 to 8192): a block of K
// `alone` with one tile a CU, `pair` with two, `each` for every one of more, and `end` for a tile's start and outputs;
// of 16-bit outputs, then of 32-bit ones, which the largest shape is not built for.
struct Cost {
    float alone, pair, each, end;
};
struct Shape {
    uint32_t rows, cols;
    Cost narrow, wide;
};
enum { kSmall, kSquare, kBroad, kLarge, kHigh, kHuge, kTall, kVast, kShapes };
constexpr Shape shapes[kShapes] = {{32, 64, {.21f, .28f, .15f, .3f}, {.38f, .52f, .24f, .3f}},
                                   {64, 64, {.26f, .42f, .21f, .5f}, {.43f, .71f, .35f, .5f}},
                                   {64, 128, {.42f, .68f, .32f, 1.f}, {.65f, 1.1f, .55f, 1.f}},
                                   {128, 128, {.55f, 1.12f, .57f, 2.f}, {.94f, 1.87f, .96f, 3.f}},
                                   {192, 128, {.73f, 1.48f, .73f, 3.5f}, {1.27f, 2.55f, 1.35f, 3.5f}},
                                   {128, 256, {.91f, 1.83f, .90f, 4.f}, {1.53f, 3.4f, 1.66f, 5.f}},
                                   {256, 128, {.90f, 1.84f, .90f, 4.f}, {1.53f, 3.4f, 1.67f, 5.f}},
                                   {256, 256, {1.6f, 3.3f, 1.66f, 6.5f}, {}}};

// How a product is formed: `few` by k_fp8_few, else by tiles of `shape`, K in `splits` parts.
struct Plan {
    bool few;
    int shape;
    uint32_t splits;
    bool far = false;  // by k_fp8_far
};

constexpr size_t kFewColumns = (size_t)1 << 26;  // a launch of k_fp8_few has 2^32 threads at twice as many
constexpr size_t kMostTiles = (size_t)1 << 22;   // a launch of 512 threads a tile has 2^32 at twice as many

// What k_fp8_few takes, measured in us against the best tile: up to two workgroups a CU, four for 32-bit outputs (16-bit:
// 1 x 4096 x 4096 5.6 / 9.8, 64 x 2048 x 4096 5.8 / 9.5, 16 x 8192 x 4096 8.6 / 11.0, 16 x 12288 x 4096 13.3 / 11.9; 32-bit:
// 16 x 12288 x 4096 12.6 / 16.3), one where sums are longer (64 x 1024 x 14336 10.6 / 13.0, 32 x 4096 x 14336 21.9 / 17.2);
// and whatever b it is where a tile's rows are mostly empty (1 x 131072 x 4096 92 / 94 and 88 / 96, 4 x 57344 x 8192 80 /
// 86 and 75 / 89).  The longest sums are split by tiles only (1 x 4096 x 32768 34 / 29, 16 x 1024 x 65536 42 / 23).
bool by_few(size_t M, size_t N, size_t K, int type) {
    const size_t groups = (M + 15) / 16 * ((N + 15) / 16);
    if (K > 24576 || N >= kFewColumns) return false;
    return M <= (type == PFA_F32 ? 16 : 8) || groups <= 256 || (K <= 8192 && groups <= (type == PFA_F32 ? 1024 : 512));
}

// The plan of least estimated time: that of the products and the tiles' ends, or of reading b, a little more for every
// row of tiles that reads it again.  K is split where tiles are too few for the card and the sums are long enough to
// pay for the second launch and the partial sums (128 x 4096 x 16384: 59.8 us whole, 26.4 in 4).
Plan plan_matmul(size_t M, size_t N, size_t K, int type) {
    if (by_few(M, N, K, type)) return {true, 0, 1};
    const float blocks = (float)((K + kBlock - 1) / kBlock), memory = 5e6f;  // bytes a us
    Plan best{false, -1, 1};
    float least = INFINITY;
    auto look = [&](bool half_empty) {
        for (int i = 0; i < kShapes; i++) {
            const Shape &s = shapes[i];
            if (s.rows > 32 && M <= s.rows / 2 && !half_empty) continue;  // half a tile or more of nothing
            if (i == kVast && (type == PFA_F32 || K % kBlock)) continue;  // takes whole blocks only
            const Cost &c = type == PFA_F32 ? s.wide : s.narrow;
            const size_t down = (M + s.rows - 1) / s.rows, tiles = down * ((N + s.cols - 1) / s.cols);
            if (tiles >= kMostTiles) continue;
            const float reading = ((float)N * K * (1 + .15f * (down - 1)) + (float)M * K) / memory;
            for (uint32_t splits = 1; splits <= 8; splits *= 2) {
                if (splits > 1 && (tiles * splits > 512 || blocks < 8 * splits)) break;
                const size_t on_cu = (tiles * splits + 255) / 256;
                const float block = on_cu <= 1 ? c.alone : on_cu == 2 ? c.pair : on_cu * c.each;
                const float join = splits == 1 ? 0.f : 4.f + (float)splits * M * N * 8 / memory;
                const float time = std::max(block * blocks / splits + on_cu * c.end, reading) + join;
                if (time < least) {
                    least = time;
                    best = {false, i, splits};
                }
            }
        }
    };
    look(false);
    if (best.shape < 0) look(true);  // a few rows of more columns than low tiles cover
    require(best.shape >= 0, "pfa_fp8_matmul: more outputs than one launch can form");
    return best;
}

template <class T, int BM, int BN, int WM, int WN, int STAGES>
void launch_tiles(const Fp8Args &g, hipStream_t s) {
    const size_t jobs = (size_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN) * g.splits;  // below kMostTiles
    hipLaunchKernelGGL((k_fp8_tiles<T, BM, BN, WM, WN, STAGES>), dim3((uint32_t)((jobs + 7) / 8 * 8)), dim3(WM * WN * 64), 0,
                       s, g);
    if (g.splits > 1)
        hipLaunchKernelGGL(k_fp8_join<T>, dim3((uint32_t)(((size_t)g.M * ((g.N + 3) / 4) + 255) / 256)), dim3(256), 0, s,
                           g);
}

template <class T>
void matmul(const Fp8Args &g, const Plan &p, hipStream_t s) {
    if (p.few) {
        const dim3 grid((g.N + 15) / 16, (g.M + 15) / 16), threads(kFewWaves * 64);
        if (p.far)
            hipLaunchKernelGGL(k_fp8_far<T>, grid, threads, 0, s, g);
        else if (g.M <= 8)
            hipLaunchKernelGGL((k_fp8_few<T, 8>), grid, threads, 0, s, g);
        else
            hipLaunchKernelGGL((k_fp8_few<T, 16>), grid, threads, 0, s, g);
        return;
    }
    switch (p.shape) {
        case kSmall: return launch_tiles<T, 32, 64, 2, 2, 6>(g, s);
        case kSquare: return launch_tiles<T, 64, 64, 2, 2, 4>(g, s);
        case kBroad: return launch_tiles<T, 64, 128, 2, 2, 3>(g, s);
        case kLarge: return launch_tiles<T, 128, 128, 2, 4, 4>(g, s);
        case kHigh: return launch_tiles<T, 192, 128, 4, 2, 3>(g, s);
        case kHuge: return launch_tiles<T, 128, 256, 2, 4, 3>(g, s);
        case kTall: return launch_tiles<T, 256, 128, 4, 2, 3>(g, s);
    }
    if constexpr (!std::is_same_v<T, float>)
        if (p.shape == kVast) return launch_tiles<T, 256, 256, 4, 2, 2>(g, s);
}

size_t parts_bytes(size_t M, size_t N, const Plan &p) {
    return !p.few && p.splits > 1 && M && N ? p.splits * M * N * sizeof(float) : 0;
}

void check_sizes(size_t M, size_t N, size_t K, const char *what) {
    require(M <= 0x7fffffffu && N <= 0x7fffffffu && K <= 0x7fffffffu,
            std::string(what) + ": more than 2^31 - 1 rows or places");
}

}  // namespace

}  // namespace pfa

using namespace pfa;

extern "C" {

int pfa_fp8_workspace(size_t M, size_t N, size_t K, int type, size_t *bytes) {
    return guarded([&] {
        require(bytes != nullptr, "null argument");
        type_bytes(type);
        check_sizes(M, N, K, "pfa_fp8_workspace");
        *bytes = parts_bytes(M, N, plan_matmul(M, N, K, type));
    });
}

int pfa_fp8_plan(size_t M, size_t N, size_t K, int type, size_t *tile_rows, size_t *tile_cols, size_t *splits) {
    return guarded([&] {
        require(tile_rows && tile_cols && splits, "null argument");
        type_bytes(type);
        check_sizes(M, N, K, "pfa_fp8_plan");
        const Plan p = plan_matmul(M, N, K, type);
        *tile_rows = p.few ? 0 : shapes[p.shape].rows;
        *tile_cols = p.few ? 16 : shapes[p.shape].cols;
        *splits = p.splits;
    });
}

int pfa_fp8_matmul(const uint8_t *a, size_t a_stride, const float *a_scales, size_t a_scales_row, size_t a_scales_block,
                   const uint8_t *b, size_t b_stride, const float *b_scales, size_t b_scales_row, size_t b_scales_block,
                   const float *bias, size_t M, size_t N, size_t K, void *out, int type, size_t out_stride,
                   void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        check_sizes(M, N, K, "pfa_fp8_matmul");
        require(!workspace_bytes || workspace, "null workspace");
        if (M == 0 || N == 0) return;
        require(out && (K == 0 || (a && b && a_scales && b_scales)), "null argument");
        require((M == 1 || ((a_stride == 0 || a_stride >= K) && out_stride >= N)) &&
                    (N == 1 || b_stride == 0 || b_stride >= K),
                "rows overlap");
        require((((uintptr_t)a_scales | (uintptr_t)b_scales | (uintptr_t)bias) & 3) == 0 &&
                    ((uintptr_t)out & (size - 1)) == 0,
                "pfa_fp8_matmul: a tensor is not aligned to its elements");
        Plan p = plan_matmul(M, N, K, type);
        // the tiles' offsets from their first rows have 32 bits: 256 rows 2^23 bytes apart, their scales 2^20 numbers
        const size_t far = (size_t)1 << 23;
        if ((M > 1 && (a_stride > far || a_scales_row > far / 8)) || (N > 1 && b_stride > far) ||
            (N > kBlock && b_scales_row > far))
            p = {true, 0, 1, true};
        require(!p.few || (M <= 65535 * 16 && N < kFewColumns),
                "pfa_fp8_matmul: rows this far apart: at most 1048560 of a and 2^26 - 1 of b");
        const size_t need = parts_bytes(M, N, p);
        require(workspace_bytes >= need, "pfa_fp8_matmul: the workspace needs " + std::to_string(need) + " bytes");
        require(((uintptr_t)workspace & 15) == 0, "pfa_fp8_matmul: the workspace is not aligned to 16 bytes");
        const Fp8Args g{(const int8_t *)a, (const int8_t *)b, a_scales,           b_scales,      bias,           out,
                        a_stride,          b_stride,          out_stride,         a_scales_row,  a_scales_block, b_scales_row,
                        b_scales_block,    (float *)workspace, (uint32_t)M,       (uint32_t)N,   (uint32_t)K,    p.splits};
        with_type(type, [&](auto t) { matmul<decltype(t)>(g, p, as_stream(stream)); });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
