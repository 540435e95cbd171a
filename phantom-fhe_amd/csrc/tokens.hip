// The clear end of an encrypted generation step, row by row: root-mean-square
// norm and quantization to 8-bit codes, probabilities of tokens, and the check
// of drafted tokens.  No counterpart in the reference, whose client side does
// these on the CPU; the products between them are in int8_matmul.hip.
//
// All of them are bound by memory: a few operations for each element that is
// read.  Statistics are held in 32 bits throughout.
#include <algorithm>

#include "element.h"

namespace pfa {

namespace {

constexpr int kRowThreads = 256;

// Rows go over x and y of the grid: a launch has at most 2^32 threads along one of them.
constexpr uint32_t kRowsX = 1u << 20;
__device__ __forceinline__ size_t row_of() { return (size_t)blockIdx.y * kRowsX + blockIdx.x; }
dim3 row_grid(size_t rows) {
    return dim3((uint32_t)std::min<size_t>(rows, kRowsX), (uint32_t)((rows + kRowsX - 1) / kRowsX));
}

// Codes of one row.  With k = 127 / max|v| every code is rint(v k); the norm's
// factor rsqrt(mean + eps) is common to the row and cancels, so the sum of
// squares and the maximum come from the same pass.
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
    float eps;
};

constexpr int kVec = 8;  // elements a thread takes at once: 16 bytes of the 2-byte types, 8 codes

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

// rint(v lift k) by one fused step: 1.5 2^23 leaves the sum's last bit at 1, so its low
// byte is the code, rounded once to nearest even.  keep: ~0, or 0 for codes of 0.
__device__ __forceinline__ uint32_t code_of(float v, float lift, float k) {
    return __float_as_uint(fmaf(v * lift, k, 12582912.f));
}
__device__ __forceinline__ void store_codes(int8_t *codes, const float (&v)[kVec], float lift, float k, uint32_t keep) {
    uint32_t w[kVec / 4];
#pragma unroll
    for (int e = 0; e < kVec; e += 4) {
        const uint32_t lo = __builtin_amdgcn_perm(code_of(v[e + 1], lift, k), code_of(v[e], lift, k), 0x0c0c0400);
        const uint32_t hi = __builtin_amdgcn_perm(code_of(v[e + 3], lift, k), code_of(v[e + 2], lift, k), 0x04000c0c);
        w[e / 4] = (lo | hi) & keep;
    }
    __builtin_memcpy(codes, w, kVec);
}

// A row is read once: its values stay in registers, STEPS x kVec a thread, between the
// reduction and the codes.  The row's last kVec places are one thread's even where the
// width is no multiple of kVec (its vector then starts early, and threads past the end
// read it too), so no load stands behind a branch and all of them are in flight at once.
// THREADS = 64: four rows a workgroup, one a wave, no barrier.  STEPS = 0: rows too
// long for the registers are read twice.
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
    // 127 / top passes float's range below 2^-121: such rows are lifted by 2^64 first
    float lift = 1.f, top = __uint_as_float(s.top);
    if (top < 1e-36f) {
        lift = 0x1p64f;
        top *= lift;
    }
    const float k = s.top == 0 ? 0.f : 127.f / top;
    const uint32_t keep = bad ? 0u : ~0u;
    if (t == 0) {
        float scale = __uint_as_float(s.top) / 127.f;
        if (NORM) scale *= rsqrtf(s.sum / (float)a.width + a.eps);
        a.scales[row] = bad ? __uint_as_float(0x7fc00000u) : scale;
    }
    if (brief) {
        if (t == 0)
#pragma unroll
            for (int e = 0; e < kVec; e++)
                if (e < (int)a.width) codes[e] = (int8_t)(code_of(v[0][e], lift, k) & keep);
    } else if (STEPS) {
#pragma unroll
        for (int j = 0; j < kHold; j++) {
            const uint32_t own = (j * THREADS + t) * kVec;
            if (own < a.width) store_codes(codes + min(own, last), v[j], lift, k, keep);
        }
    } else {
        RowStat again{0.f, 0u};
        for (uint32_t own = t * kVec; own < a.width; own += THREADS * kVec) {
            row_values<T, NORM>(a, x, residual, nullptr, min(own, last), own, again, v[0]);
            store_codes(codes + min(own, last), v[0], lift, k, keep);
        }
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

// Probabilities of one row: exp2((l - m) c) / sum, c = log2(e) / temperature, m the
// largest allowed logit; temperature 0 leaves the lowest place of m alone.
template <class T>
__global__ void __launch_bounds__(kRowThreads)
k_probabilities(size_t rows, const T *logits, size_t stride, const float *temperatures, float temperature, const uint8_t *mask,
                size_t mask_stride, uint32_t vocab, float *out) {
    __shared__ float part[kRowThreads / 64];
    __shared__ uint32_t first;
    const size_t row = row_of();
    if (row >= rows) return;
    logits += row * stride;
    out += row * vocab;
    if (mask) mask += row * mask_stride;
    const float inf = __uint_as_float(kInfBits);
    const float t = temperatures ? temperatures[row] : temperature;
    const float c = fminf(1.44269504088896341f / t, 3e38f);
    float m = -inf;
    bool nan = !(t >= 0.f);
    for (uint32_t i = threadIdx.x; i < vocab; i += kRowThreads) {
        if (mask && !mask[i]) continue;
        const float l = (float)logits[i];
        nan |= l != l;
        m = fmaxf(m, l);
    }
    m = wave_max(nan ? inf : m);
    if (threadIdx.x == 0) first = 0xffffffffu;
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = m;
    nan = __syncthreads_or(nan);
    m = part[0];
    for (int w = 1; w < kRowThreads / 64; w++) m = fmaxf(m, part[w]);
    __syncthreads();
    if (t == 0.f) {
        for (uint32_t i = threadIdx.x; i < vocab; i += kRowThreads)
            if ((!mask || mask[i]) && (float)logits[i] == m && m > -inf) {
                atomicMin(&first, i);
                break;
            }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < vocab; i += kRowThreads)
            out[i] = nan ? (!mask || mask[i] ? __uint_as_float(0x7fc00000u) : 0.f) : i == first ? 1.f : 0.f;
        return;
    }
    float sum = 0.f;
    for (uint32_t i = threadIdx.x; i < vocab; i += kRowThreads) {
        if (mask && !mask[i]) continue;
        const float l = (float)logits[i];
        if (l != -inf) sum += exp2f((l - m) * c);
    }
    sum = wave_sum(sum);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = sum;
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < kRowThreads / 64; w++) sum += part[w];
    const float scale = nan ? __uint_as_float(0x7fc00000u) : m == -inf ? 0.f : 1.f / sum;
    for (uint32_t i = threadIdx.x; i < vocab; i += kRowThreads) {
        const float l = (float)logits[i];
        const bool in = !mask || mask[i];
        out[i] = !in ? 0.f : l == -inf ? 0.f * scale : exp2f((l - m) * c) * scale;
    }
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
    size_t target_batch, target_place, draft_batch, draft_place, noise_batch;  // strides in elements
    size_t batch;
    uint32_t K, vocab;
    bool tokens64, lengths64;
};

__device__ __forceinline__ int64_t whole(const void *p, size_t i, bool wide) {
    return wide ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

// w / e as a key that compares like it, with the lower index first among equals; 0: no weight
__device__ __forceinline__ uint64_t race_key(float w, float e, uint32_t i) {
    return w > 0.f ? (uint64_t)__float_as_uint(w / e) << 32 | (0xffffffffu - i) : 0;
}

// One sequence a workgroup.  Draft i stays while u_i q_i(x_i) < p_i(x_i); the token
// after the first that does not is drawn from max(p - q, 0), after the last one from
// p: the largest weight / noise, an exponential race, has exactly that distribution.
// Each product, difference and quotient is one rounding of 32 bits, so the choice
// does not depend on the order of anything.
template <class T>
__global__ void __launch_bounds__(kRowThreads)
k_verify(VerifyArgs a) {
#pragma clang fp contract(off)
    __shared__ uint64_t best_rest[kRowThreads / 64], best_all[kRowThreads / 64];
    const size_t b = row_of();
    if (b >= a.batch) return;
    const T *target = static_cast<const T *>(a.target) + b * a.target_batch;
    const T *draft = static_cast<const T *>(a.draft) + b * a.draft_batch;
    const int64_t given = a.lengths ? whole(a.lengths, b, a.lengths64) : (int64_t)a.K;
    const uint32_t len = (uint32_t)(given < 0 ? 0 : given > (int64_t)a.K ? (int64_t)a.K : given);
    uint32_t n = 0;
    for (; n < len; n++) {
        const int64_t x = whole(a.drafts, b * a.K + n, a.tokens64);
        if (x < 0 || x >= (int64_t)a.vocab) break;
        const float p = (float)target[n * a.target_place + x];
        const float q = a.draft ? (float)draft[n * a.draft_place + x] : 1.f;
        if (!(a.uniforms[b * a.K + n] * q < p)) break;
    }
    target += n * a.target_place;
    const bool rest = n < len;
    const int64_t refused = rest ? whole(a.drafts, b * a.K + n, a.tokens64) : -1;
    const float *noise = a.noise + b * a.noise_batch;
    uint64_t key_rest = 0, key_all = 0;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kRowThreads) {
        const float p = (float)target[i], e = noise[i];
        const uint64_t k = race_key(p, e, i);
        key_all = k > key_all ? k : key_all;
        if (rest) {
            const float w = a.draft ? p - (float)draft[n * a.draft_place + i] : (int64_t)i == refused ? 0.f : p;
            const uint64_t r = race_key(w, e, i);
            key_rest = r > key_rest ? r : key_rest;
        }
    }
    key_all = wave_max(key_all);
    key_rest = wave_max(key_rest);
    if (threadIdx.x % 64 == 0) {
        best_all[threadIdx.x / 64] = key_all;
        best_rest[threadIdx.x / 64] = key_rest;
    }
    __syncthreads();
    for (int w = 0; w < kRowThreads / 64; w++) {
        key_all = best_all[w] > key_all ? best_all[w] : key_all;
        key_rest = best_rest[w] > key_rest ? best_rest[w] : key_rest;
    }
    const uint64_t key = key_rest ? key_rest : key_all;
    const int64_t token = key ? (int64_t)(0xffffffffu - (uint32_t)key) : -1;
    for (uint32_t i = threadIdx.x; i <= a.K; i += kRowThreads) {
        const int64_t v = i < n ? whole(a.drafts, b * a.K + i, a.tokens64) : i == n ? token : -1;
        if (a.tokens64)
            static_cast<int64_t *>(a.tokens)[b * (a.K + 1) + i] = v;
        else
            static_cast<int32_t *>(a.tokens)[b * (a.K + 1) + i] = (int32_t)v;
    }
    if (threadIdx.x == 0) a.accepted[b] = (int32_t)n;
}

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
        require(eps >= 0 && eps <= 1e30, "pfa_rms_norm_int8: eps must be 0 or more");
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
                        x_stride, residual_stride, total_stride, codes_stride, (uint32_t)width, (float)eps};
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
        require(temperatures || (temperature >= 0 && temperature <= 1e30),
                "pfa_token_probabilities: the temperature must be 0 or more");
        require(!workspace_bytes || workspace, "null workspace");
        if (rows == 0 || vocab == 0) return;
        require(logits && out, "null argument");
        require(apart(rows, stride, vocab), "rows overlap");
        aligned(logits, size, "logits");
        aligned(out, 4, "out");
        aligned(temperatures, 4, "temperatures");
        with_type(type, [&](auto t) {
            using T = decltype(t);
            hipLaunchKernelGGL(k_probabilities<T>, row_grid(rows), dim3(kRowThreads), 0, as_stream(stream),
                               rows, (const T *)logits, stride, temperatures, (float)temperature, mask, mask_stride,
                               (uint32_t)vocab, out);
        });
        PFA_HIP(hipGetLastError());
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
        VerifyArgs a{drafts, lengths, target, draft, uniforms, noise, tokens, accepted, target_batch, target_place,
                     draft_batch, draft_place, noise_batch, batch, (uint32_t)K, (uint32_t)vocab, token_bytes == 8,
                     length_bytes == 8};
        with_type(type, [&](auto t) {
            using T = decltype(t);
            hipLaunchKernelGGL(k_verify<T>, row_grid(batch), dim3(kRowThreads), 0, as_stream(stream), a);
        });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
