// Codes of 8-bit floating point (e4m3: 4 significant bits, largest 448) with a scale for each
// block of 128 places of a row, or of 128 rows and 128 places: quantization, and the root-mean-square
// norm that ends in such codes.  The products of them are in fp8_matmul.hip.
//
// The scale of a block is the least power of two that takes its largest magnitude to 448 or less (2^-126 at
// least, so that its inverse is a number too).  A floating code has its 4 bits wherever it stands
// below 448, so a scale between two powers would gain nothing; the quotient by a power is exact, and the one rounding
// is the code's.
#include <algorithm>
#include <cmath>

#include "rows.h"

namespace pfa {

namespace {

constexpr uint32_t kSpan = 128;            // places of a row, and rows, that share a scale
constexpr int kSpanLanes = kSpan / kVec;   // lanes that share a block of one row
constexpr uint32_t kNan = 0x7fc00000u;

// largest of 16 neighbouring lanes, in each of them
__device__ __forceinline__ uint32_t span_max(uint32_t v) {
#define PFA_STEP(control) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, control, 0xf, 0xf, false))
    PFA_STEP(0xb1);   // the neighbour
    PFA_STEP(0x4e);   // the other pair of four
    PFA_STEP(0x141);  // the other four of eight
    PFA_STEP(0x140);  // the other eight
#undef PFA_STEP
    return v;
}

// Scale of a block from its largest magnitude: 448 is 1.75 2^8.
struct Step {
    uint32_t scale, inverse;  // powers of two, as the bits of 32-bit floats
    bool bad;                 // a NaN or an infinity: a NaN scale, codes of 0
    __device__ __forceinline__ explicit Step(uint32_t top) {
        const int e = max((int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), 1);
        bad = top >= kInfBits;
        scale = bad ? kNan : top ? (uint32_t)e << 23 : 0u;
        inverse = (uint32_t)(254 - min(e, 253)) << 23;
    }
};

// codes of kVec values, the first in the lowest byte
__device__ __forceinline__ uint2 codes_of(const float (&v)[kVec], const Step &s) {
    const float k = __uint_as_float(s.inverse);
    uint2 w;
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * k, v[1] * k, 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * k, v[3] * k, lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * k, v[5] * k, 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * k, v[7] * k, hi, true);
    w.x = s.bad ? 0u : (uint32_t)lo;
    w.y = s.bad ? 0u : (uint32_t)hi;
    return w;
}

// A thread's kVec places of a row of `width`, the first at `own`.  The row's last vector starts early, so no load
// stands behind a branch and all of a thread's are in flight at once; what it reads before `own` (or all of it,
// behind the row's end) is another thread's and becomes 0.  Rows of fewer than kVec places are read one by one.
// EVEN: whole vectors only.  What is read behind the end is then the last vector again, of the row's last block, and
// changes no largest: nothing is cleared.
template <bool EVEN>
struct Part {
    uint32_t own, at, width;
    __device__ __forceinline__ Part(uint32_t own, uint32_t width)
        : own(own), at(width >= kVec ? min(own, width - kVec) : 0u), width(width) {}
    __device__ __forceinline__ bool mine(int e) const { return at + e >= own && (width >= kVec || at + e < width); }
    __device__ __forceinline__ bool inside() const { return own < width; }
    template <class T>
    __device__ __forceinline__ void load(const T *x, float (&v)[kVec]) const {
        if (EVEN || width >= kVec) {
            load_vec<kVec>(x + at, v);
        } else {
#pragma unroll
            for (int e = 0; e < kVec; e++) v[e] = mine(e) ? (float)x[e] : 0.f;
        }
    }
    __device__ __forceinline__ void clear(float (&v)[kVec]) const {
        if (EVEN) return;
#pragma unroll
        for (int e = 0; e < kVec; e++) v[e] = mine(e) ? v[e] : 0.f;
    }
    // 2- and 4-byte values; where the vector starts early it holds the neighbour's own values too
    template <class T>
    __device__ __forceinline__ void store(T *x, const float (&v)[kVec]) const {
        if (EVEN || width >= kVec) {
            if (own < width) store_vec<kVec>(x + at, v);
        } else {
#pragma unroll
            for (int e = 0; e < kVec; e++)
                if (mine(e)) x[e] = (T)v[e];
        }
    }
    __device__ __forceinline__ void store_codes(uint8_t *codes, uint2 w) const {
        if (EVEN ? inside() : own + kVec <= width) {
            __builtin_memcpy(codes + own, &w, kVec);
        } else if (!EVEN) {
#pragma unroll
            for (int e = 0; e < kVec; e++)
                if (mine(e)) codes[at + e] = (uint8_t)((e < 4 ? w.x : w.y) >> (e % 4 * 8));
        }
    }
};
__device__ __forceinline__ uint32_t top_of(const float (&v)[kVec]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < kVec; e++) top = max(top, mag_bits(v[e]));
    return top;
}

struct BlockArgs {
    const void *x;
    uint8_t *codes;
    float *scales;
    size_t rows, x_stride, codes_stride, scales_row, scales_block;
    uint32_t width, across;  // workgroups along a row
};

// A scale for each 128 places of a row.  16 lanes take a block of a row, a workgroup 16 rows and 4
// blocks, all of a thread's loads in flight at once; the scales of its 16 rows stand together in memory.
// Bound by memory: 4096 x 8192 bf16 17.4 us (5.8 TB/s), float32 28.4 (5.9 TB/s); rows that begin anywhere, 777 x 5119
// fp16, 6.1 us.
constexpr int kBlockRows = 16, kBlockSteps = 4;

template <class T, bool EVEN>
__global__ void __launch_bounds__(256)
k_fp8_rows(BlockArgs a) {
    const size_t job = row_of(), row = job / a.across * kBlockRows + threadIdx.x / kSpanLanes;
    if (row >= a.rows) return;
    const uint32_t first = (uint32_t)(job % a.across) * kBlockSteps, lane = threadIdx.x % kSpanLanes;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    uint8_t *codes = a.codes + row * a.codes_stride;
    float v[kBlockSteps][kVec];
#pragma unroll
    for (int j = 0; j < kBlockSteps; j++) Part<EVEN>((first + j) * kSpan + lane * kVec, a.width).load(x, v[j]);
#pragma unroll
    for (int j = 0; j < kBlockSteps; j++) {
        const uint32_t block = first + j;
        const Part<EVEN> p(block * kSpan + lane * kVec, a.width);
        p.clear(v[j]);
        const Step s(span_max(top_of(v[j])));
        p.store_codes(codes, codes_of(v[j], s));
        if (lane == 0 && block * kSpan < a.width)
            a.scales[row * a.scales_row + block * a.scales_block] = __uint_as_float(s.scale);
    }
}

// A scale for each 128 rows and 128 places: a workgroup takes a block, 8 vectors a thread in flight at once, so that
// the block is read once.  Bound by memory: 16384 x 4096 bf16 35 us (5.8 TB/s), float32 60 us (5.6 TB/s).
template <class T, bool EVEN>
__global__ void __launch_bounds__(256)
k_fp8_squares(BlockArgs a) {
    __shared__ uint32_t part[4];
    const size_t job = row_of(), down = job / a.across;
    if (down * kSpan >= a.rows) return;
    const uint32_t block = (uint32_t)(job % a.across);
    const Part<EVEN> p(block * kSpan + threadIdx.x % kSpanLanes * kVec, a.width);
    constexpr int kSteps = kSpan / (256 / kSpanLanes);
    float v[kSteps][kVec];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < kSteps; j++) {
        // behind the last row: that one again, which changes no maximum
        const size_t row = min(down * kSpan + j * (256 / kSpanLanes) + threadIdx.x / kSpanLanes, a.rows - 1);
        p.load(static_cast<const T *>(a.x) + row * a.x_stride, v[j]);
    }
#pragma unroll
    for (int j = 0; j < kSteps; j++) {
        p.clear(v[j]);
        top = max(top, top_of(v[j]));
    }
    top = wave_max(top);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = top;
    __syncthreads();
    const Step s(max(max(part[0], part[1]), max(part[2], part[3])));
#pragma unroll
    for (int j = 0; j < kSteps; j++) {
        const size_t row = down * kSpan + j * (256 / kSpanLanes) + threadIdx.x / kSpanLanes;
        if (row < a.rows) p.store_codes(a.codes + row * a.codes_stride, codes_of(v[j], s));
    }
    if (threadIdx.x == 0) a.scales[down * a.scales_row + block * a.scales_block] = __uint_as_float(s.scale);
}

template <class T, bool EVEN>
void quantize_blocks(BlockArgs a, size_t block_rows, hipStream_t s) {
    if (block_rows == 1) {
        a.across = (a.across + kBlockSteps - 1) / kBlockSteps;
        hipLaunchKernelGGL((k_fp8_rows<T, EVEN>), row_grid((a.rows + kBlockRows - 1) / kBlockRows * a.across), dim3(256), 0, s,
                           a);
    } else {
        hipLaunchKernelGGL((k_fp8_squares<T, EVEN>), row_grid((a.rows + kSpan - 1) / kSpan * a.across), dim3(256), 0, s, a);
    }
}

struct NormArgs {
    const void *x, *residual, *weight;
    void *total;
    uint8_t *codes;
    float *scales;
    size_t rows, x_stride, residual_stride, total_stride, codes_stride, scales_row, scales_block;
    uint32_t width;
    double eps;
};

// y = x + residual and v = y weight of a thread's places, the squares of y, total on the way
template <class T, bool EVEN>
__device__ __forceinline__ void norm_values(const NormArgs &a, const T *x, const T *residual, T *total, const Part<EVEN> &p,
                                            float &sum, float (&v)[kVec]) {
    float w[kVec];
    p.load(x, v);
    p.load(static_cast<const T *>(a.weight), w);
    if (residual) {
        float r[kVec];
        p.load(residual, r);
#pragma unroll
        for (int e = 0; e < kVec; e++) v[e] += r[e];
        if (total) p.store(total, v);
    }
    p.clear(v);
    p.clear(w);
    float squares = 0.f;
#pragma unroll
    for (int e = 0; e < kVec; e++) {
        squares = fmaf(v[e], v[e], squares);
        v[e] *= w[e];
    }
    sum += p.inside() ? squares : 0.f;
}

// The norm's factor 1 / sqrt(mean + eps) is common to a row: codes and powers of two are those of the blocks of y
// weight, and the factor goes into the scales.  So the row is read once and stays in registers, STEPS x kVec a thread,
// while its squares are summed.  THREADS = 64: four rows a workgroup, one a wave, no barrier.  STEPS = 0:
// rows too long for the registers are read twice.  Bound by memory: 4096 x 8192 bf16 with residual 44-47 us (5.0-5.4
// TB/s), float32 84 us (5.2 TB/s); one row of 4096 3.3 us.
template <class T, bool EVEN, int THREADS, int STEPS>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS)
k_fp8_norm(NormArgs a) {
    constexpr bool kWave = THREADS == 64;
    constexpr int kHold = STEPS ? STEPS : 1;
    const uint32_t t = threadIdx.x % THREADS;
    const size_t row = kWave ? row_of() * 4 + threadIdx.x / 64 : row_of();
    if (row >= a.rows) return;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *residual = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    T *total = residual ? static_cast<T *>(a.total) + row * a.total_stride : nullptr;
    uint8_t *codes = a.codes + row * a.codes_stride;
    float *scales = a.scales + row * a.scales_row;
    float v[kHold][kVec], sum = 0.f;
    uint32_t any = 0;  // of the row's magnitudes
    if (STEPS) {
#pragma unroll
        for (int j = 0; j < kHold; j++) norm_values(a, x, residual, total, Part<EVEN>((j * THREADS + t) * kVec, a.width), sum, v[j]);
#pragma unroll
        for (int j = 0; j < kHold; j++) any = max(any, top_of(v[j]));
    } else {
        for (uint32_t i = t * kVec; i < a.width; i += THREADS * kVec) {
            norm_values(a, x, residual, total, Part<EVEN>(i, a.width), sum, v[0]);
            any = max(any, top_of(v[0]));
        }
    }
    sum = wave_sum(sum);
    any = wave_max(any);
    if (!kWave) {
        __shared__ float part_sum[THREADS / 64];
        __shared__ uint32_t part_any[THREADS / 64];
        if (t % 64 == 0) {
            part_sum[t / 64] = sum;
            part_any[t / 64] = any;
        }
        __syncthreads();
        sum = 0.f;
        any = 0u;
#pragma unroll
        for (int w = 0; w < THREADS / 64; w++) {
            sum += part_sum[w];
            any = max(any, part_any[w]);
        }
    }
    // Codes first: they do not wait for the factor.
    const bool lost = !(sum < __uint_as_float(kInfBits));
    auto put_codes = [&](uint32_t i, const float (&u)[kVec]) {
        Step s(span_max(top_of(u)));
        s.bad |= lost;
        if (i < a.width) Part<EVEN>(i, a.width).store_codes(codes, codes_of(u, s));
        return s.bad ? kNan : s.scale;
    };
    uint32_t power[kHold];
    if (STEPS) {
#pragma unroll
        for (int j = 0; j < kHold; j++) power[j] = put_codes((j * THREADS + t) * kVec, v[j]);
    }
    // Squares below 2^-126 lose bits, below 2^-149 all of them.  Where they could matter, in a sum below
    // 2^-90 that eps does not outweigh, they are summed again.
    float lifted = 0.f;
    const bool few = any && sum < kFewSquares && a.eps < 0x1p-60;
    if (few) {
        lifted = wave_sum(lifted_squares(x, residual, a.width, t, THREADS));
        if (!kWave) {
            __shared__ float part[THREADS / 64];
            if (t % 64 == 0) part[t / 64] = lifted;
            __syncthreads();
            lifted = 0.f;
#pragma unroll
            for (int w = 0; w < THREADS / 64; w++) lifted += part[w];
        }
    }
    const double total_sum = few ? (double)lifted * 0x1p-200 : (double)sum;
    const double factor = few || a.eps > 0x1p100 ? rsqrt(total_sum / a.width + a.eps)
                                                 : (double)rsqrtf(sum / (float)a.width + (float)a.eps);
    auto put_scale = [&](uint32_t i, uint32_t bits) {
        if (t % kSpanLanes == 0 && i < a.width)  // 0 stays 0 at eps = 0
            scales[i / kSpan * a.scales_block] = bits ? (float)((double)__uint_as_float(bits) * factor) : 0.f;
    };
    if (STEPS) {
#pragma unroll
        for (int j = 0; j < kHold; j++) put_scale((j * THREADS + t) * kVec, power[j]);
    } else {
        float again = 0.f;
        // all lanes of a block go round together
        for (uint32_t i = t * kVec; i - t % kSpanLanes * kVec < a.width; i += THREADS * kVec) {
            norm_values(a, x, residual, (T *)nullptr, Part<EVEN>(i, a.width), again, v[0]);
            put_scale(i, put_codes(i, v[0]));
        }
    }
}

template <class T, bool EVEN>
void norm_rows(const NormArgs &a, hipStream_t s) {
    const uint32_t vecs = (a.width + kVec - 1) / kVec;
#define PFA_LAUNCH(threads, steps)                                                                                \
    hipLaunchKernelGGL((k_fp8_norm<T, EVEN, threads, steps>), row_grid(threads == 64 ? (a.rows + 3) / 4 : a.rows),      \
                       dim3(threads < 256 ? 256 : threads), 0, s, a)
    if (vecs <= 64)
        PFA_LAUNCH(64, 1);
    else if (vecs <= 256)
        PFA_LAUNCH(256, 1);
    else if (vecs <= 512)
        PFA_LAUNCH(256, 2);
    else if (vecs <= 1024)
        PFA_LAUNCH(256, 4);
    else if (vecs <= 2048)
        PFA_LAUNCH(256, 8);
    else if (vecs <= 4096)
        PFA_LAUNCH(1024, 4);
    else
        PFA_LAUNCH(1024, 0);
#undef PFA_LAUNCH
}

}  // namespace

}  // namespace pfa

using namespace pfa;

extern "C" {

int pfa_quantize_fp8(const void *x, size_t x_stride, int type, size_t rows, size_t width, size_t block_rows,
                     uint8_t *codes, size_t codes_stride, float *scales, size_t scales_row, size_t scales_block,
                     void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        require(block_rows == 1 || block_rows == kSpan, "pfa_quantize_fp8: blocks have 1 or 128 rows");
        check_rows(rows, width, "pfa_quantize_fp8");
        if (rows == 0 || width == 0) return;
        require(x && codes && scales, "null argument");
        require(apart(rows, x_stride, width) && apart(rows, codes_stride, width, true), "rows overlap");
        const size_t down = (rows + block_rows - 1) / block_rows, across = (width + kSpan - 1) / kSpan;
        require((down == 1 || scales_row) && (across == 1 || scales_block), "pfa_quantize_fp8: scales overlap");
        aligned(x, size, "x");
        aligned(scales, 4, "scales");
        const BlockArgs a{x,        codes,        scales,     rows,         x_stride,
                    codes_stride, scales_row, scales_block, (uint32_t)width, (uint32_t)across};
        with_type(type, [&](auto t) {
            if (width % kVec)
                quantize_blocks<decltype(t), false>(a, block_rows, as_stream(stream));
            else
                quantize_blocks<decltype(t), true>(a, block_rows, as_stream(stream));
        });
        PFA_HIP(hipGetLastError());
    });
}

int pfa_rms_norm_fp8(const void *x, size_t x_stride, const void *residual, size_t residual_stride, const void *weight,
                     int type, size_t rows, size_t width, double eps, void *total, size_t total_stride, uint8_t *codes,
                     size_t codes_stride, float *scales, size_t scales_row, size_t scales_block, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        check_rows(rows, width, "pfa_rms_norm_fp8");
        require(eps >= 0 && eps < INFINITY, "pfa_rms_norm_fp8: eps must be finite and 0 or more");
        if (rows == 0) return;
        require(width >= 1, "pfa_rms_norm_fp8: the mean of an empty row");
        require(x && weight && codes && scales && (!residual || total), "null argument");
        require(apart(rows, x_stride, width) && apart(rows, codes_stride, width, true) &&
                    (!residual ||
                     (apart(rows, residual_stride, width) && apart(rows, total_stride, width, true))),
                "rows overlap");
        require((rows == 1 || scales_row) && (width <= kSpan || scales_block), "pfa_rms_norm_fp8: scales overlap");
        aligned(x, size, "x");
        aligned(residual, size, "residual");
        aligned(weight, size, "weight");
        aligned(total, size, "total");
        aligned(scales, 4, "scales");
        const NormArgs a{x,        residual,        weight,       total,        codes,      scales,       rows,
                         x_stride, residual_stride, total_stride, codes_stride, scales_row, scales_block, (uint32_t)width,
                         eps};
        with_type(type, [&](auto t) {
            if (width % kVec)
                norm_rows<decltype(t), false>(a, as_stream(stream));
            else
                norm_rows<decltype(t), true>(a, as_stream(stream));
        });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
