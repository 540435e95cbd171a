// The clear end of an encrypted generation step, row by row: root-mean-square
// norm and quantization to 8-bit codes, probabilities of tokens, and the check
// of drafted tokens.  No counterpart in the reference, whose client side does
// these on the CPU; the products between them are in int8_matmul.hip.
//
// All of them are bound by memory: a few operations for each element that is
// read.  Statistics are held in 32 bits throughout.
#include <algorithm>
#include <cmath>

#include "rows.h"

namespace pfa {

namespace {

constexpr int kRowThreads = 256;

// Codes of one row: 127 v / max|v| to the nearest.  The norm's factor rsqrt(mean + eps) is
// common to the row and cancels, so the sum of squares and the maximum come from the same pass.
struct RowStat {
    float sum;     // of squares
    uint32_t top;  // largest |y w|, as mag_bits
};

struct RowArgs {
    const void *x, *residual, *weight;
    void *total;
    int8_t *codes;
    float *scales;
    size_t rows, x_stride, residual_stride, total_stride, codes_stride;
    uint32_t width;
    double eps;
};

// v = (x + residual) weight of kVec places from i on (quantization: x itself), total and
// the statistics on the way.  Places before `own` belong to another thread.
template <class T, bool NORM>
__device__ __forceinline__ void row_values(const RowArgs &a, const T *x, const T *residual, T *total, uint32_t i,
                                           uint32_t own, RowStat &s, float (&v)[kVec]) {
    load_vec<kVec>(x + i, v);
    if (NORM) {
        float w[kVec];
        if (residual) {
            load_vec<kVec>(residual + i, w);
#pragma unroll
            for (int e = 0; e < kVec; e++) v[e] += w[e];
            if (total && own < a.width) store_vec<kVec>(total + i, v);
        }
        load_vec<kVec>(static_cast<const T *>(a.weight) + i, w);
#pragma unroll
        for (int e = 0; e < kVec; e++) {
            const float y = i + e >= own ? v[e] : 0.f;
            s.sum = fmaf(y, y, s.sum);
            v[e] *= w[e];
        }
    }
#pragma unroll
    for (int e = 0; e < kVec; e++) s.top = max(s.top, mag_bits(v[e]));
}

// rows of fewer than kVec places
template <class T, bool NORM>
__device__ __forceinline__ void short_row_values(const RowArgs &a, const T *x, const T *residual, T *total,
                                                 RowStat &s, float (&v)[kVec]) {
#pragma unroll
    for (int e = 0; e < kVec; e++) {
        v[e] = 0.f;
        if (e < (int)a.width) {
            v[e] = (float)x[e];
            if (NORM) {
                if (residual) {
                    v[e] += (float)residual[e];
                    total[e] = (T)v[e];
                }
                s.sum = fmaf(v[e], v[e], s.sum);
                v[e] *= (float)static_cast<const T *>(a.weight)[e];
            }
            s.top = max(s.top, mag_bits(v[e]));
        }
    }
}

// A code from the value and k = 127 / max|v|, in the low byte: 127 v / max|v| to the nearest, ties to
// even, for every v.  What is no tie is 2^-33 or more from one (v and max|v| have 24 bits), and k's
// rounding moves a product by 2^-46: rounded at 2^-40 (the unit of 6144), ties are ties again, and 1.5 2^52
// then leaves the code in the sum's last bits.  Two operations of 64 bits, at the rate of 32; with a factor of
// 24 bits one value in 10^5 would get the neighbouring code.
__device__ __forceinline__ uint32_t code_of(float v, double k) {
    return (uint32_t)__double2loint(fma((double)v, k, 6144.) + (6755399441055744. - 6144.));
}
__device__ __forceinline__ void store_codes(int8_t *codes, const float (&v)[kVec], double k, uint32_t keep) {
    uint32_t w[kVec / 4];
#pragma unroll
    for (int e = 0; e < kVec; e += 4) {
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; i++) c[i] = code_of(v[e + i], k);
        const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0c);
        w[e / 4] = (lo | hi) & keep;
    }
    __builtin_memcpy(codes, w, kVec);
}

// A row is read once: its values stay in registers, STEPS x kVec a thread, between the
// reduction and the codes.  The row's last kVec places are one thread's even where the
// width is no multiple of kVec (its vector then starts early, and threads past the end
// read it too), so no load stands behind a branch and all of them are in flight at once.
// THREADS = 64: four rows a workgroup, one a wave, no barrier.  STEPS = 0: rows too
// long for the registers are read twice.  Bound by memory: 2048 x 16384 bf16 in 18.2 us (5.5 TB/s), float32 29 us
// (5.8 TB/s); with norm and residual 4096 x 8192 bf16 in 46 us (5.1 TB/s), float32 83 us (5.2 TB/s); one row of
// 4096 in 3.1 us, a launch and one trip to memory.
template <class T, bool NORM, int THREADS, int STEPS>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS)
k_quantize_rows(RowArgs a) {
    constexpr bool kWave = THREADS == 64;
    constexpr int kHold = STEPS ? STEPS : 1;
    const uint32_t t = threadIdx.x % THREADS;
    const size_t row = kWave ? row_of() * 4 + threadIdx.x / 64 : row_of();
    if (row >= a.rows) return;
    const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
    const T *residual = a.residual ? static_cast<const T *>(a.residual) + row * a.residual_stride : nullptr;
    T *total = residual ? static_cast<T *>(a.total) + row * a.total_stride : nullptr;
    int8_t *codes = a.codes + row * a.codes_stride;
    const bool brief = kWave && a.width < kVec;
    const uint32_t last = a.width - kVec;
    float v[kHold][kVec];
    RowStat s{0.f, 0u};
    if (brief) {
        if (t == 0) short_row_values<T, NORM>(a, x, residual, total, s, v[0]);
    } else if (STEPS) {
#pragma unroll
        for (int j = 0; j < kHold; j++) {
            const uint32_t own = (j * THREADS + t) * kVec;
            row_values<T, NORM>(a, x, residual, total, min(own, last), own, s, v[j]);
        }
    } else {
        for (uint32_t own = t * kVec; own < a.width; own += THREADS * kVec)
            row_values<T, NORM>(a, x, residual, total, min(own, last), own, s, v[0]);
    }
    s.sum = NORM ? wave_sum(s.sum) : 0.f;
    s.top = wave_max(s.top);
    if (!kWave) {
        __shared__ float part_sum[THREADS / 64];
        __shared__ uint32_t part_top[THREADS / 64];
        if (t % 64 == 0) {
            part_sum[t / 64] = s.sum;
            part_top[t / 64] = s.top;
        }
        __syncthreads();
        s = {0.f, 0u};
#pragma unroll
        for (int w = 0; w < THREADS / 64; w++) {
            s.sum += part_sum[w];
            s.top = max(s.top, part_top[w]);
        }
    }
    // a NaN, an infinity or a sum past float's range: a NaN scale, codes of 0
    const bool bad = s.top >= kInfBits || !(s.sum < __uint_as_float(kInfBits));
    const float top = __uint_as_float(s.top);
    const double k = s.top ? 127. / (double)top : 0.;
    const uint32_t keep = bad ? 0u : ~0u;
    if (brief) {
        if (t == 0)
#pragma unroll
            for (int e = 0; e < kVec; e++)
                if (e < (int)a.width) codes[e] = (int8_t)(code_of(v[0][e], k) & keep);
    } else if (STEPS) {
#pragma unroll
        for (int j = 0; j < kHold; j++) {
            const uint32_t own = (j * THREADS + t) * kVec;
            if (own < a.width) store_codes(codes + min(own, last), v[j], k, keep);
        }
    } else {
        RowStat again{0.f, 0u};
        for (uint32_t own = t * kVec; own < a.width; own += THREADS * kVec) {
            row_values<T, NORM>(a, x, residual, nullptr, min(own, last), own, again, v[0]);
            store_codes(codes + min(own, last), v[0], k, keep);
        }
    }
    // The scale, behind the codes, which do not wait for it (in front 4096 x 8192 took 0.5 us more).
    // Squares below 2^-126 lose bits, below 2^-149 all of them.  Where they could matter, in a sum below
    // 2^-90 (2^30 of them make 2^-119) that eps does not outweigh, they are summed again.
    float lifted = 0.f;
    const bool few = NORM && s.top && s.sum < kFewSquares && a.eps < 0x1p-60;
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
    if (t == 0) {
        float scale = top / 127.f;
        if (NORM && s.top) {  // 0 stays 0 at eps = 0; the factor may be past 32 bits, and `top` subnormal
            const double sum = few ? (double)lifted * 0x1p-200 : (double)s.sum;
            const double factor = few || a.eps > 0x1p100 ? rsqrt(sum / a.width + a.eps)
                                                         : (double)rsqrtf(s.sum / (float)a.width + (float)a.eps);
            scale = (float)((double)top * (1. / 127.) * factor);
        }
        a.scales[row] = bad ? __uint_as_float(0x7fc00000u) : scale;
    }
}

template <class T, bool NORM, int THREADS, int STEPS>
void launch_rows(const RowArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((k_quantize_rows<T, NORM, THREADS, STEPS>),
                       row_grid(THREADS == 64 ? (a.rows + 3) / 4 : a.rows), dim3(THREADS < 256 ? 256 : THREADS), 0, s,
                       a);
}

template <class T, bool NORM>
void quantize_rows(const RowArgs &a, hipStream_t s) {
    const uint32_t vecs = (a.width + kVec - 1) / kVec;
    if (vecs <= 64) return launch_rows<T, NORM, 64, 1>(a, s);
    if (vecs <= 256) return launch_rows<T, NORM, 256, 1>(a, s);
    if (vecs <= 512) return launch_rows<T, NORM, 256, 2>(a, s);
    if (vecs <= 1024) return launch_rows<T, NORM, 256, 4>(a, s);
    if (vecs <= 2048) return launch_rows<T, NORM, 256, 8>(a, s);
    if (vecs <= 4096) return launch_rows<T, NORM, 1024, 4>(a, s);
    // the norm's three inputs of 8 steps would pass 128 registers, 1024 threads' share
    if (!NORM && vecs <= 8192) return launch_rows<T, NORM, 1024, NORM ? 0 : 8>(a, s);
    launch_rows<T, NORM, 1024, 0>(a, s);
}

// Probabilities of one row: exp2((l - m) log2(e) / temperature) / sum, m the
// largest allowed logit; temperature 0 leaves the lowest place of m alone.
struct ProbArgs {
    const void *logits;
    const float *temperatures;
    const uint8_t *mask;
    float *out;
    void *parts;  // [rows][chunks] of ProbPart
    size_t rows, stride, mask_stride;
    uint32_t vocab, chunk, chunks;
    float temperature;
};

// What a stretch of a row says: its largest logit, the sum of weights against it, the
// lowest place of the largest.  A NaN in an allowed place is a NaN sum.
struct __align__(16) ProbPart {
    float top, sum;
    uint32_t first, unused;
};

// A row, or a stretch of one, by THREADS threads: values stay in registers.
template <class T, int THREADS, int STEPS>
struct ProbRow {
    float v[STEPS][kVec];
    float top = -infinity();
    bool nan = false;

    __device__ __forceinline__ void load(const T *logits, const uint8_t *mask, uint32_t begin, uint32_t end) {
        const uint32_t last = end - kVec;
#pragma unroll
        for (int j = 0; j < STEPS; j++) {
            const uint32_t own = begin + (j * THREADS + threadIdx.x) * kVec;
            allowed_logits(logits, mask, min(own, last), own, v[j]);
        }
#pragma unroll
        for (int j = 0; j < STEPS; j++)
#pragma unroll
            for (int e = 0; e < kVec; e++) {
                nan |= v[j][e] != v[j][e];
                top = fmaxf(top, v[j][e]);
            }
    }
    // the largest of all threads; whether any saw a NaN
    __device__ __forceinline__ void share_top() {
        __shared__ float part[THREADS / 64];
        const float w = wave_max(top);
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = w;
        nan = __syncthreads_or(nan);
        top = part[0];
#pragma unroll
        for (int i = 1; i < THREADS / 64; i++) top = fmaxf(top, part[i]);
    }
    // values become weights against `m`; their sum over all threads
    __device__ __forceinline__ float weights(float m, Heat heat) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < STEPS; j++)
#pragma unroll
            for (int e = 0; e < kVec; e++) {
                v[j][e] = heat.weight(v[j][e], m);
                sum += v[j][e];
            }
        __shared__ float part[THREADS / 64];
        if (THREADS == 1024) {
            // as wave_sum, but the lanes' addresses are formed anew: kept since share_top they push a row's values
            // out of its 64 registers, and back on the way to the sum (320 rows of 32768 20.3 us, kept 21.1; rows of
            // 256 threads have room: 2000 of 5003 15.5 us, anew 15.8)
            uint32_t lane = threadIdx.x;
            asm volatile("" : "+v"(lane));
#pragma unroll
            for (uint32_t d = 32; d; d >>= 1)
                sum += __int_as_float(__builtin_amdgcn_ds_bpermute((int)((lane ^ d) * 4), __float_as_int(sum)));
        } else {
            sum = wave_sum(sum);
        }
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = sum;
        __syncthreads();
        sum = part[0];
#pragma unroll
        for (int i = 1; i < THREADS / 64; i++) sum += part[i];
        return sum;
    }
    // lowest place of `m`
    __device__ __forceinline__ uint32_t first(float m, uint32_t begin, uint32_t end) {
        __shared__ uint32_t at;
        if (threadIdx.x == 0) at = 0xffffffffu;
        __syncthreads();
        const uint32_t last = end - kVec;
        uint32_t low = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < STEPS; j++) {
            const uint32_t i = min(begin + (j * THREADS + (uint32_t)threadIdx.x) * kVec, last);
#pragma unroll
            for (int e = 0; e < kVec; e++)
                if (v[j][e] == m) low = min(low, i + e);
        }
        if (low != 0xffffffffu) atomicMin(&at, low);
        __syncthreads();
        return at;
    }
};

// A row of NaN: its allowed places, 0 elsewhere.
__device__ __forceinline__ void write_nan(const uint8_t *mask, float *out, uint32_t begin, uint32_t end,
                                          uint32_t threads) {
    for (uint32_t i = begin + threadIdx.x; i < end; i += threads) out[i] = !mask || mask[i] ? not_a_number() : 0.f;
}

// Rows in one piece: read once, reduced twice, written once.  Two workgroups of 1024
// threads on a CU (64 registers a lane) let one read while the other writes: 4096 rows of
// 32768 bf16 in 166 us (4.8 TB/s), with one of them 203 us.
template <class T, int THREADS, int STEPS>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 && STEPS <= 4 ? 8 : 1)
k_prob_rows(ProbArgs a) {
    const size_t row = row_of();
    if (row >= a.rows) return;
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    float *out = a.out + row * a.vocab;
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    ProbRow<T, THREADS, STEPS> r;
    r.load(logits, mask, 0, a.vocab);
    r.share_top();
    if (r.nan || !(t >= 0.f) || (t > 0.f && r.top == infinity()))
        return write_nan(mask, out, 0, a.vocab, THREADS);
    const bool greedy = t == 0.f;
    const uint32_t at = greedy && r.top > -infinity() ? r.first(r.top, 0, a.vocab) : 0xffffffffu;
    const float sum = r.weights(r.top == -infinity() ? 0.f : r.top, Heat(t));
    const float scale = sum > 0.f ? 1.f / sum : 0.f;
    const uint32_t last = a.vocab - kVec;
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        const uint32_t own = (j * THREADS + threadIdx.x) * kVec, i = min(own, last);
#pragma unroll
        for (int e = 0; e < kVec; e++) r.v[j][e] = greedy ? (i + e == at ? 1.f : 0.f) : r.v[j][e] * scale;
        // a place before `own` holds weight 0 here and its probability elsewhere
        if (i == own) {
            store_vec<kVec>(out + i, r.v[j]);
        } else if (own < a.vocab) {
#pragma unroll
            for (int e = 0; e < kVec; e++)
                if (i + e >= own) out[i + e] = r.v[j][e];
        }
    }
}

// Long rows, and few rows: stretches of `chunk` places by a workgroup each, in two
// launches.  The first leaves a ProbPart for each stretch, the second joins a row's and
// writes the probabilities; its second reading of the logits comes from the caches.  5
// rows of 131072 float32: 3.6 + 4.2 us, bound by the launches and the reductions.
constexpr int kChunkThreads = 256;

template <class T, int STEPS>
__global__ void __launch_bounds__(kChunkThreads)
k_prob_parts(ProbArgs a) {
    const size_t job = row_of(), row = job / a.chunks;
    if (row >= a.rows) return;
    const uint32_t begin = (uint32_t)(job % a.chunks) * a.chunk, end = min(begin + a.chunk, a.vocab);
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    ProbRow<T, kChunkThreads, STEPS> r;
    r.load(logits, mask, begin, end);
    r.share_top();
    ProbPart p{r.top, 0.f, 0xffffffffu, 0u};
    if (r.nan || !(t >= 0.f) || (t > 0.f && r.top == infinity()))
        p.sum = not_a_number();
    else if (t == 0.f)
        p.first = r.top == -infinity() ? 0xffffffffu : r.first(r.top, begin, end);
    else
        p.sum = r.weights(r.top == -infinity() ? 0.f : r.top, Heat(t));
    if (threadIdx.x == 0) static_cast<ProbPart *>(a.parts)[job] = p;
}

template <class T, int STEPS>
__global__ void __launch_bounds__(kChunkThreads)
k_prob_write(ProbArgs a) {
    __shared__ float part[kChunkThreads / 64], part_sum[kChunkThreads / 64];
    __shared__ uint32_t part_first[kChunkThreads / 64];
    const size_t job = row_of(), row = job / a.chunks;
    if (row >= a.rows) return;
    const uint32_t begin = (uint32_t)(job % a.chunks) * a.chunk, end = min(begin + a.chunk, a.vocab);
    const uint32_t last = end - kVec, wave = threadIdx.x / 64;
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    float *out = a.out + row * a.vocab;
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    const Heat heat(t);
    float v[STEPS][kVec];
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        const uint32_t own = begin + (j * kChunkThreads + threadIdx.x) * kVec;
        allowed_logits(logits, mask, min(own, last), 0, v[j]);
    }
    const ProbPart *parts = static_cast<const ProbPart *>(a.parts) + row * a.chunks;
    float top = -infinity(), sum = 0.f;
    uint32_t first = 0xffffffffu;
    for (uint32_t i = threadIdx.x; i < a.chunks; i += kChunkThreads) top = fmaxf(top, parts[i].top);
    top = wave_max(top);
    if (threadIdx.x % 64 == 0) part[wave] = top;
    __syncthreads();
    top = part[0];
#pragma unroll
    for (int i = 1; i < kChunkThreads / 64; i++) top = fmaxf(top, part[i]);
    const float m = top == -infinity() ? 0.f : top;
    for (uint32_t i = threadIdx.x; i < a.chunks; i += kChunkThreads) {
        const ProbPart p = parts[i];
        if (t == 0.f && p.top == top) first = min(first, p.first);
        sum += t == 0.f ? p.sum : p.sum == 0.f ? 0.f : p.sum * heat.weight(p.top, m);
    }
    sum = wave_sum(sum);
    first = ~wave_max(~first);
    if (threadIdx.x % 64 == 0) {
        part_sum[wave] = sum;
        part_first[wave] = first;
    }
    __syncthreads();
    sum = 0.f;
    first = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kChunkThreads / 64; i++) {
        sum += part_sum[i];
        first = min(first, part_first[i]);
    }
    if (sum != sum) return write_nan(mask, out, begin, end, kChunkThreads);
    const float scale = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
    for (int j = 0; j < STEPS; j++) {
        const uint32_t own = begin + (j * kChunkThreads + threadIdx.x) * kVec, i = min(own, last);
#pragma unroll
        for (int e = 0; e < kVec; e++)
            v[j][e] = t == 0.f ? (i + e == first ? 1.f : 0.f) : heat.weight(v[j][e], m) * scale;
        if (own < end) store_vec<kVec>(out + i, v[j]);
    }
}

// rows of fewer than kVec places, one a thread: too short for a vector, and its launch is the time
template <class T>
__global__ void __launch_bounds__(kRowThreads)
k_prob_short(ProbArgs a) {
    const size_t row = row_of() * kRowThreads + threadIdx.x;
    if (row >= a.rows) return;
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    float *out = a.out + row * a.vocab;
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    float top = -infinity(), sum = 0.f;
    uint32_t first = 0xffffffffu;
    bool nan = !(t >= 0.f);
    for (uint32_t i = 0; i < a.vocab; i++) {
        const float l = !mask || mask[i] ? (float)logits[i] : -infinity();
        nan |= l != l;
        if (l > top) {
            top = l;
            first = i;
        }
    }
    if (nan || (t > 0.f && top == infinity())) {
        for (uint32_t i = 0; i < a.vocab; i++) out[i] = !mask || mask[i] ? not_a_number() : 0.f;
        return;
    }
    const Heat heat(t);
    const float m = top == -infinity() ? 0.f : top;
    for (int write = 0; write < 2; write++) {
        const float scale = sum > 0.f ? 1.f / sum : 0.f;
        for (uint32_t i = 0; i < a.vocab; i++) {
            const float l = !mask || mask[i] ? (float)logits[i] : -infinity();
            const float w = t == 0.f ? (i == first ? 1.f : 0.f) : heat.weight(l, m);
            if (write)
                out[i] = w * scale;
            else
                sum += w;
        }
    }
}

// One piece while a row's values fit the registers of 1024 threads, unless there are too
// few rows for the card (measured, bf16, us, one piece / cut: 16 rows of 32768 8.0 / 6.9, 128
// rows 11.7 / 13.4; 128 rows of 65536 20.2 / 18.9, 512 rows 50 / 57).  Stretches have one vector
// a thread while that gives the card little to do, then two, which share a workgroup's
// start and reductions (16 rows of 131072 10.0 / 9.9, 512 rows 127 / 114; four: 115).
Cut cut_probabilities(size_t rows, uint32_t vocab) {
    if (vocab <= 16384 || (vocab <= 32768 && rows >= 64) || (vocab <= 65536 && rows >= 256)) return {vocab, 1};
    const uint32_t least = kChunkThreads * kVec;
    const uint32_t chunk = rows * ((vocab + least - 1) / least) < 1024 ? least : 2 * least;
    return {chunk, (vocab + chunk - 1) / chunk};
}

template <class T>
void probabilities(const ProbArgs &a, hipStream_t s) {
    const uint32_t vecs = (a.vocab + kVec - 1) / kVec;
#define PFA_LAUNCH(kernel, jobs, threads) hipLaunchKernelGGL((kernel), row_grid(jobs), dim3(threads), 0, s, a)
    if (a.vocab < kVec) {
        PFA_LAUNCH(k_prob_short<T>, (a.rows + kRowThreads - 1) / kRowThreads, kRowThreads);
    } else if (a.chunks == 1) {
        if (vecs <= 64)
            PFA_LAUNCH((k_prob_rows<T, 64, 1>), a.rows, 64);
        else if (vecs <= 256)
            PFA_LAUNCH((k_prob_rows<T, 256, 1>), a.rows, 256);
        else if (vecs <= 512)
            PFA_LAUNCH((k_prob_rows<T, 256, 2>), a.rows, 256);
        else if (vecs <= 1024)
            PFA_LAUNCH((k_prob_rows<T, 256, 4>), a.rows, 256);
        else if (vecs <= 2048)
            PFA_LAUNCH((k_prob_rows<T, 1024, 2>), a.rows, 1024);
        else if (vecs <= 4096)
            PFA_LAUNCH((k_prob_rows<T, 1024, 4>), a.rows, 1024);
        else
            PFA_LAUNCH((k_prob_rows<T, 1024, 8>), a.rows, 1024);
    } else {
        const size_t jobs = a.rows * a.chunks;
        if (a.chunk == kChunkThreads * kVec) {
            PFA_LAUNCH((k_prob_parts<T, 1>), jobs, kChunkThreads);
            PFA_LAUNCH((k_prob_write<T, 1>), jobs, kChunkThreads);
        } else {
            PFA_LAUNCH((k_prob_parts<T, 2>), jobs, kChunkThreads);
            PFA_LAUNCH((k_prob_write<T, 2>), jobs, kChunkThreads);
        }
    }
#undef PFA_LAUNCH
}

struct VerifyArgs {
    const void *drafts;     // [batch][K] tokens of 4 or 8 bytes
    const void *lengths;    // [batch] of 4 or 8 bytes, or null
    const void *target;     // [batch][K + 1][vocab]
    const void *draft;      // [batch][K][vocab] or null: the drafts were certain
    const float *uniforms;  // [batch][K]
    const float *noise;     // [batch][vocab]
    void *tokens;           // [batch][K + 1], like drafts
    int32_t *accepted;      // [batch]
    uint64_t *parts;        // [batch][chunks] race keys, with more than one chunk
    size_t target_batch, target_place, draft_batch, draft_place, noise_batch;  // strides in elements
    size_t batch;
    uint32_t K, vocab, chunk, chunks;
    bool tokens64, lengths64;
};

__device__ __forceinline__ int64_t whole(const void *p, size_t i, bool wide) {
    return wide ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

// w / e as a key that compares like it, with the lower index first among equals; 0: no weight
__device__ __forceinline__ uint64_t race_key(float w, float e, uint32_t i) {
    return w > 0.f ? (uint64_t)__float_as_uint(w / e) << 32 | (0xffffffffu - i) : 0;
}
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ uint32_t length_of(const VerifyArgs &a, size_t b) {
    const int64_t given = a.lengths ? whole(a.lengths, b, a.lengths64) : (int64_t)a.K;
    return (uint32_t)(given < 0 ? 0 : given > (int64_t)a.K ? (int64_t)a.K : given);
}

// How many of the drafts of sequence b are kept: every wave looks at 64 of them at once,
// so the two dependent readings (token, then probability) are paid once and not K times.
template <class T>
__device__ __forceinline__ uint32_t kept(const VerifyArgs &a, size_t b, uint32_t len) {
#pragma clang fp contract(off)
    const T *target = static_cast<const T *>(a.target) + b * a.target_batch;
    const T *draft = static_cast<const T *>(a.draft) + b * a.draft_batch;
    for (uint32_t n = 0; n < len; n += 64) {
        const uint32_t i = n + threadIdx.x % 64;
        bool keep = false;
        if (i < len) {
            const int64_t x = whole(a.drafts, b * a.K + i, a.tokens64);
            if (x >= 0 && x < (int64_t)a.vocab) {
                const float p = (float)target[i * a.target_place + x];
                const float q = a.draft ? (float)draft[i * a.draft_place + x] : 1.f;
                keep = a.uniforms[b * a.K + i] * q < p;
            }
        }
        const uint64_t lost = ~__ballot(keep);
        if (lost) return min(n + (uint32_t)__builtin_ctzll(lost), len);
    }
    return len;
}

constexpr uint32_t kNowhere = 0xffffffffu;

// Largest key over the places [begin, end) of w / noise: w = target, less the draft's
// where `draft` is given, but 0 at place `without`.
template <class T>
__device__ __forceinline__ uint64_t race(const T *target, const T *draft, const float *noise, uint32_t without,
                                         uint32_t begin, uint32_t end, uint32_t threads) {
#pragma clang fp contract(off)
    uint64_t key = 0;
    uint32_t i = begin + threadIdx.x * kVec;
    for (; i + kVec <= end; i += threads * kVec) {
        float e[kVec], w[kVec];
        load_vec<kVec>(noise + i, e);
        load_vec<kVec>(target + i, w);
        if (draft) {
            float q[kVec];
            load_vec<kVec>(draft + i, q);
#pragma unroll
            for (int k = 0; k < kVec; k++) w[k] -= q[k];
        }
#pragma unroll
        for (int k = 0; k < kVec; k++) key = larger(key, race_key(i + k == without ? 0.f : w[k], e[k], i + k));
    }
    for (; i < end; i++) {
        const float w = (float)target[i] - (draft ? (float)draft[i] : 0.f);
        key = larger(key, race_key(i == without ? 0.f : w, noise[i], i));
    }
    return key;
}

template <int THREADS>
__device__ __forceinline__ uint64_t block_largest(uint64_t key) {
    __shared__ uint64_t part[THREADS / 64];
    key = wave_max(key);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = key;
    __syncthreads();
    key = part[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; i++) key = larger(key, part[i]);
    __syncthreads();
    return key;
}

// The tokens of sequence b, given the winner of its race.  A refusal that leaves nothing
// over is rare: the target's own race is run here then.
template <class T>
__device__ __forceinline__ void finish(const VerifyArgs &a, size_t b, uint32_t n, uint32_t len, uint64_t key) {
    if (!key && n < len) {
        const T *target = static_cast<const T *>(a.target) + b * a.target_batch + n * a.target_place;
        key = block_largest<kRowThreads>(
            race<T>(target, nullptr, a.noise + b * a.noise_batch, kNowhere, 0, a.vocab, kRowThreads));
    }
    const int64_t token = key ? (int64_t)(0xffffffffu - (uint32_t)key) : -1;
    for (uint32_t i = threadIdx.x; i <= a.K; i += kRowThreads) {
        const int64_t v = i < n ? whole(a.drafts, b * a.K + i, a.tokens64) : i == n ? token : -1;
        if (a.tokens64)
            static_cast<int64_t *>(a.tokens)[b * (a.K + 1) + i] = v;
        else
            static_cast<int32_t *>(a.tokens)[b * (a.K + 1) + i] = (int32_t)v;
    }
}

// Draft i stays while u_i q_i(x_i) < p_i(x_i); the token after the first that does not is
// drawn from max(p - q, 0), after the last one from p: the largest weight / noise, an
// exponential race, has exactly that distribution, and needs no sum over the row, so the
// stretches of a row are independent.  Each product, difference and quotient is one
// rounding of 32 bits and a largest key has no order, so neither has the choice.  Only the
// row that is drawn from is read, so reading it bounds many sequences (64 of 100003
// places, 77 MB: 13.5 us, 5.7 TB/s) and the two dependent readings few (1 of 131072: 4.2 us).
template <class T>
__global__ void __launch_bounds__(kRowThreads)
k_verify(VerifyArgs a) {
    const size_t job = row_of(), b = job / a.chunks;
    if (b >= a.batch) return;
    const uint32_t begin = (uint32_t)(job % a.chunks) * a.chunk, end = min(begin + a.chunk, a.vocab);
    const uint32_t len = length_of(a, b), n = kept<T>(a, b, len);
    const T *target = static_cast<const T *>(a.target) + b * a.target_batch + n * a.target_place;
    const T *draft = a.draft && n < len
                         ? static_cast<const T *>(a.draft) + b * a.draft_batch + n * a.draft_place
                         : nullptr;
    uint32_t without = kNowhere;
    if (!a.draft && n < len) {
        const int64_t x = whole(a.drafts, b * a.K + n, a.tokens64);
        if (x >= 0 && x < (int64_t)a.vocab) without = (uint32_t)x;
    }
    const uint64_t key = block_largest<kRowThreads>(
        race<T>(target, draft, a.noise + b * a.noise_batch, without, begin, end, kRowThreads));
    if (a.chunks == 1) finish<T>(a, b, n, len, key);
    if (threadIdx.x == 0) {
        if (a.chunks > 1) a.parts[job] = key;
        if (begin == 0) a.accepted[b] = (int32_t)n;
    }
}

// joins the stretches of each sequence (64 of them: 4 us, 1: 2 us)
template <class T>
__global__ void __launch_bounds__(kRowThreads)
k_verify_join(VerifyArgs a) {
    const size_t b = row_of();
    if (b >= a.batch) return;
    uint64_t key = 0;
    for (uint32_t i = threadIdx.x; i < a.chunks; i += kRowThreads) key = larger(key, a.parts[b * a.chunks + i]);
    key = block_largest<kRowThreads>(key);
    finish<T>(a, b, (uint32_t)a.accepted[b], length_of(a, b), key);
}

// Stretches of one vector a thread (64 sequences of 100003: 19.0 us, of eight 19.6; one of
// 131072: 5.8 and 10.2), unless a row is so short that a workgroup takes it as fast
// (8192 places, 1 sequence: 5.8 us either way; 256: 8.3 in one piece, 10.5 cut).
Cut cut_race(uint32_t vocab) {
    const uint32_t chunk = kRowThreads * kVec;
    if (vocab <= 4 * chunk) return {vocab, 1};
    return {chunk, (vocab + chunk - 1) / chunk};
}

}  // namespace

}  // namespace pfa

using namespace pfa;

extern "C" {

int pfa_quantize_int8(const void *x, size_t x_stride, int type, size_t rows, size_t width, int8_t *codes,
                      size_t codes_stride, float *scales, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        check_rows(rows, width, "pfa_quantize_int8");
        if (rows == 0) return;
        require(scales && (width == 0 || (x && codes)), "null argument");
        require(apart(rows, x_stride, width) && apart(rows, codes_stride, width, true), "rows overlap");
        aligned(x, size, "x");
        aligned(scales, 4, "scales");
        RowArgs a{};
        a.x = x;
        a.codes = codes;
        a.scales = scales;
        a.rows = rows;
        a.x_stride = x_stride;
        a.codes_stride = codes_stride;
        a.width = (uint32_t)width;
        with_type(type, [&](auto t) { quantize_rows<decltype(t), false>(a, as_stream(stream)); });
        PFA_HIP(hipGetLastError());
    });
}

int pfa_rms_norm_int8(const void *x, size_t x_stride, const void *residual, size_t residual_stride,
                      const void *weight, int type, size_t rows, size_t width, double eps, void *total,
                      size_t total_stride, int8_t *codes, size_t codes_stride, float *scales, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        check_rows(rows, width, "pfa_rms_norm_int8");
        require(eps >= 0 && eps < INFINITY, "pfa_rms_norm_int8: eps must be finite and 0 or more");
        if (rows == 0) return;
        require(width >= 1, "pfa_rms_norm_int8: the mean of an empty row");
        require(x && weight && codes && scales && (!residual || total), "null argument");
        require(apart(rows, x_stride, width) && apart(rows, codes_stride, width, true) &&
                    (!residual ||
                     (apart(rows, residual_stride, width) && apart(rows, total_stride, width, true))),
                "rows overlap");
        aligned(x, size, "x");
        aligned(residual, size, "residual");
        aligned(weight, size, "weight");
        aligned(total, size, "total");
        aligned(scales, 4, "scales");
        const RowArgs a{x,        residual,        weight,       total,        codes,           scales, rows,
                        x_stride, residual_stride, total_stride, codes_stride, (uint32_t)width, eps};
        with_type(type, [&](auto t) { quantize_rows<decltype(t), true>(a, as_stream(stream)); });
        PFA_HIP(hipGetLastError());
    });
}

int pfa_token_probabilities(const void *logits, size_t stride, int type, size_t rows, size_t vocab,
                            const float *temperatures, double temperature, const uint8_t *mask, size_t mask_stride,
                            float *out, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        check_rows(rows, vocab, "pfa_token_probabilities");
        require(temperatures || temperature >= 0, "pfa_token_probabilities: the temperature must be 0 or more");
        require(!workspace_bytes || workspace, "null workspace");
        if (rows == 0 || vocab == 0) return;
        require(logits && out, "null argument");
        require(apart(rows, stride, vocab) && (!mask || apart(rows, mask_stride, vocab)), "rows overlap");
        aligned(logits, size, "logits");
        aligned(out, 4, "out");
        aligned(temperatures, 4, "temperatures");
        const Cut cut = cut_probabilities(rows, (uint32_t)vocab);
        const size_t need = cut.chunks == 1 ? 0 : rows * cut.chunks * sizeof(ProbPart);
        require(workspace_bytes >= need, "pfa_token_probabilities: the workspace needs " + std::to_string(need) + " bytes");
        aligned(workspace, 16, "workspace");
        const ProbArgs a{logits, temperatures, mask, out, workspace, rows, stride, mask_stride, (uint32_t)vocab,
                         cut.chunk, cut.chunks, (float)temperature};
        with_type(type, [&](auto t) { probabilities<decltype(t)>(a, as_stream(stream)); });
        PFA_HIP(hipGetLastError());
    });
}

int pfa_token_workspace(size_t rows, size_t vocab, size_t *bytes) {
    return guarded([&] {
        check_rows(rows, vocab, "pfa_token_workspace");
        require(bytes != nullptr, "null argument");
        const Cut p = cut_probabilities(rows, (uint32_t)vocab), v = cut_race((uint32_t)vocab);
        *bytes = std::max(p.chunks == 1 ? 0 : rows * p.chunks * sizeof(ProbPart), v.chunks == 1 ? 0 : rows * v.chunks * 8);
    });
}

int pfa_verify_drafts(const void *drafts, int token_bytes, const void *lengths, int length_bytes, size_t batch,
                      size_t K, size_t vocab, const void *target, size_t target_batch, size_t target_place,
                      const void *draft, size_t draft_batch, size_t draft_place, int type, const float *uniforms,
                      const float *noise, size_t noise_batch, void *tokens, int32_t *accepted, void *workspace,
                      size_t workspace_bytes, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        require(token_bytes == 4 || token_bytes == 8, "tokens have 4 or 8 bytes");
        require(!lengths || length_bytes == 4 || length_bytes == 8, "lengths have 4 or 8 bytes");
        check_rows(batch, vocab, "pfa_verify_drafts");
        require(K < 0x7fffffffu, "pfa_verify_drafts: too many drafts");
        require(!workspace_bytes || workspace, "null workspace");
        if (batch == 0) return;
        require(tokens && accepted && (K == 0 || (drafts && uniforms)) && (vocab == 0 || (target && noise)),
                "null argument");
        aligned(drafts, token_bytes, "drafts");
        aligned(tokens, token_bytes, "tokens");
        if (lengths) aligned(lengths, length_bytes, "lengths");
        aligned(target, size, "target");
        aligned(draft, size, "draft");
        aligned(uniforms, 4, "uniforms");
        aligned(noise, 4, "noise");
        aligned(accepted, 4, "accepted");
        const Cut cut = cut_race((uint32_t)vocab);
        const size_t need = cut.chunks == 1 ? 0 : batch * cut.chunks * 8;
        require(workspace_bytes >= need, "pfa_verify_drafts: the workspace needs " + std::to_string(need) + " bytes");
        aligned(workspace, 8, "workspace");
        VerifyArgs a{drafts, lengths, target, draft, uniforms, noise, tokens, accepted, (uint64_t *)workspace,
                     target_batch, target_place, draft_batch, draft_place, noise_batch, batch, (uint32_t)K,
                     (uint32_t)vocab, cut.chunk, cut.chunks, token_bytes == 8, length_bytes == 8};
        const hipStream_t s = as_stream(stream);
        with_type(type, [&](auto t) {
            using T = decltype(t);
            hipLaunchKernelGGL(k_verify<T>, row_grid(batch * cut.chunks), dim3(kRowThreads), 0, s, a);
            if (cut.chunks > 1) hipLaunchKernelGGL(k_verify_join<T>, row_grid(batch), dim3(kRowThreads), 0, s, a);
        });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
