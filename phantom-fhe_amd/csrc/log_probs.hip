// Log probabilities of given tokens, the entropy of the distribution, and its largest alternatives, from
// logits: with d = (l - m) / t, m the largest allowed logit of a row, and S = sum e^d,
//   log p = d - log S,   H = log S - (sum e^d d) / S.
// The logits are read once, with a running maximum a thread, and no probability is written.
//
// The alternatives need no order of the row.  The largest logits of 64 classes of its places (the lanes' classes) are
// 64 places' logits: their k-th largest has k places at or above it, so the k largest of the row are among the
// places that reach it.  Those are collected (about k of them where the classes share them out evenly) and
// ranked by comparing each with all.  Where they are too many to collect (long ties, logits in step with the
// classes), the k-th largest of what was collected is the next threshold, until they fit.
#include <algorithm>
#include <cmath>

#include "rows.h"

namespace pfa {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr uint32_t kMostTop = 64;      // alternatives: one class of places each
constexpr uint32_t kKept = 1024;       // places that one collection holds
constexpr uint32_t kMostGroups = 1024; // groups of a row's places whose largest are kept, in a cut row
constexpr float kLn2 = 0.69314718055994531f;

struct LogArgs {
    const void *logits;
    const void *tokens;  // [rows][given] of 4 or 8 bytes
    const float *temperatures;
    const uint8_t *mask;
    float *log_probs, *entropy, *top_log_probs;  // [rows][given], [rows], [rows][top]
    void *top_tokens;                            // [rows][top], like tokens
    void *parts;                                 // [rows][chunks] of LogPart, then [rows][chunks kWaves] floats
    size_t rows, stride, mask_stride;
    uint32_t vocab, given, top, chunk, chunks;
    float temperature;
    bool tokens64;
};

// What a stretch of a row says: its largest logit, and against it the sum of weights 2^g and of
// weights times g, g = d log2(e).  A NaN in an allowed place, or +infinity, is a NaN sum.
struct __align__(16) LogPart {
    float top, sum, turn, unused;
};

// largest below nothing: a stretch that allows nothing has top -infinity and sum 0
struct Running {
    float top = -infinity(), sum = 0.f, turn = 0.f;

    __device__ __forceinline__ static float exponent(float l, float m, const Heat &heat) {
        return fmaxf(fmaf(l, heat.half, -heat.half * m) * heat.rate, -200.f);
    }
    // sums against `m`, which is no smaller than top
    __device__ __forceinline__ void lift(float m, const Heat &heat) {
        if (top == m) return;
        const float g = top == -infinity() ? -200.f : exponent(top, m, heat), w = __builtin_amdgcn_exp2f(g);
        turn = (turn + g * sum) * w;
        sum *= w;
        top = m;
    }
    __device__ __forceinline__ void add(const float (&v)[kVec], const Heat &heat) {
        float m = v[0];
#pragma unroll
        for (int e = 1; e < kVec; e++) m = fmaxf(m, v[e]);
        if (m > top) lift(m, heat);
        const float base = top == -infinity() ? 0.f : top;
#pragma unroll
        for (int e = 0; e < kVec; e++) {
            const float g = exponent(v[e], base, heat), w = __builtin_amdgcn_exp2f(g);
            sum += w;
            turn = fmaf(w, g, turn);
        }
    }
    __device__ __forceinline__ void join(float other_top, float other_sum, float other_turn, const Heat &heat) {
        Running o;
        o.top = other_top;
        o.sum = other_sum;
        o.turn = other_turn;
        const float m = fmaxf(top, o.top);
        lift(m, heat);
        o.lift(m, heat);
        sum += o.sum;
        turn += o.turn;
    }
};

// kVec allowed logits from i on of [begin, end), -infinity elsewhere; rows shorter than a vector one by one
template <class T>
__device__ __forceinline__ void fetch(const T *logits, const uint8_t *mask, uint32_t own, uint32_t end, uint32_t vocab,
                                      float (&v)[kVec]) {
    if (vocab >= kVec) {
        allowed_logits(logits, mask, min(own, vocab - kVec), own, v);
    } else {
#pragma unroll
        for (int e = 0; e < kVec; e++)
            v[e] = own + e < vocab && (!mask || mask[own + e]) ? (float)logits[own + e] : -infinity();
    }
}

// order of a logit among a row's: larger logits first, then lower places; 0 is no place
__device__ __forceinline__ uint32_t ordered(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);  // -0 is 0
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float l, uint32_t i) {
    return l > -infinity() ? (uint64_t)ordered(l) << 32 | (0xffffffffu - i) : 0;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o);
}

// The workgroup's shared memory
struct Shared {
    uint64_t kept[kKept];
    float tops[kWaves][64];
    float top[kWaves], sum[kWaves], turn[kWaves];
    uint32_t count, groups, list[kMostGroups];
    uint64_t limit;
};

// The k-th largest of 64 lanes' numbers, in every lane
__device__ __forceinline__ uint32_t kth_of_lanes(uint32_t v, uint32_t k) {
    uint32_t above = 0, least = 0xffffffffu;  // how many are larger
#pragma unroll
    for (int j = 0; j < 64; j++) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)v, j);
        above += o > v;
    }
    // the smallest of those with fewer than k above them
    if (above < k) least = v;
    return ~wave_max(~least);
}

// The `count` collected keys by rank; the first k of them to `put(rank, key)`, the k-th to shared.limit
template <class F>
__device__ __forceinline__ void rank_kept(Shared &s, uint32_t count, uint32_t k, F put) {
    for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
        const uint64_t mine = s.kept[i];
        uint32_t above = 0;
        for (uint32_t j = 0; j < count; j++) above += s.kept[j] > mine;
        if (above + 1 == k) s.limit = mine;
        if (above < k) put(above, mine);
    }
}

// The k largest places of a row: put(rank, key) once for each of them.  `scan(f)` calls f(v, at) for vectors of places
// among which are all whose logit is `floor` or more (as ordered()).
template <class S, class F>
__device__ __forceinline__ void largest(Shared &s, uint32_t k, uint32_t floor, S scan, F put) {
    uint64_t limit = max((uint64_t)floor << 32, (uint64_t)1);
    for (;;) {
        __syncthreads();
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        scan([&](const float (&v)[kVec], uint32_t at) {
#pragma unroll
            for (int e = 0; e < kVec; e++) {
                const uint64_t key = key_of(v[e], at + e);
                if (key >= limit) {
                    const uint32_t n = atomicAdd(&s.count, 1u);
                    if (n < kKept) s.kept[n] = key;
                }
            }
        });
        __syncthreads();
        const uint32_t count = s.count;
        if (count <= kKept) return rank_kept(s, count, k, put);
        rank_kept(s, kKept, k, [](uint32_t, uint64_t) {});
        __syncthreads();
        limit = s.limit;
    }
}

__device__ __forceinline__ void set_token(const LogArgs &a, size_t i, int64_t v) {
    if (a.tokens64)
        static_cast<int64_t *>(a.top_tokens)[i] = v;
    else
        static_cast<int32_t *>(a.top_tokens)[i] = (int32_t)v;
}

// What a row gives, its sums known: by all threads of a workgroup.  `floor` as in largest().
template <class T, class S>
__device__ __forceinline__ void finish(const LogArgs &a, size_t row, float t, const Running &r, uint32_t floor, Shared &s,
                                       S scan) {
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const bool nan = r.sum != r.sum || !(t >= 0.f) || (t > 0.f && r.top == infinity()), none = r.top == -infinity();
    const bool greedy = t == 0.f;
    const float log_sum = logf(r.sum);
    // differences are formed halved: see Heat
    const float half = t >= 1.f ? 0.5f : 1.f;
    auto log_prob = [&](float l) {
        if (nan) return not_a_number();
        if (none || l == -infinity()) return -infinity();
        return (l * half - r.top * half) / (t * half) - log_sum;
    };
    const uint32_t k = nan || none ? 0 : greedy ? max(a.top, 1u) : a.top;
    float *tops = a.top_log_probs + row * a.top;
    __shared__ uint32_t first;
    if (k) {
        largest(s, k, floor, scan, [&](uint32_t rank, uint64_t key) {
            const uint32_t i = 0xffffffffu - (uint32_t)key;
            if (rank == 0) first = i;
            if (rank < a.top) {
                set_token(a, row * a.top + rank, i);
                tops[rank] = greedy ? (rank ? -infinity() : 0.f) : log_prob(logit_of(key));
            }
        });
        __syncthreads();
    }
    const uint32_t found = k ? min(s.count, k) : 0;
    for (uint32_t i = found + threadIdx.x; i < a.top; i += kThreads) {
        set_token(a, row * a.top + i, -1);
        tops[i] = nan ? not_a_number() : -infinity();
    }
    for (uint32_t i = threadIdx.x; i < a.given; i += kThreads) {
        const int64_t x = a.tokens64 ? static_cast<const int64_t *>(a.tokens)[row * a.given + i]
                                     : static_cast<const int32_t *>(a.tokens)[row * a.given + i];
        float p = -infinity();
        if (x >= 0 && x < (int64_t)a.vocab && (!mask || mask[x]))
            p = greedy && !nan ? (k && (uint32_t)x == first ? 0.f : -infinity()) : log_prob((float)logits[x]);
        a.log_probs[row * a.given + i] = p;
    }
    if (threadIdx.x == 0)
        a.entropy[row] = nan ? not_a_number() : none || greedy ? 0.f : log_sum - kLn2 * (r.turn / r.sum);
}

// sums of the workgroup's threads; tops[w] holds its waves' lanes' largest afterwards
__device__ __forceinline__ void share(Shared &s, Running &r, const Heat &heat) {
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    s.tops[wave][lane] = r.top;
    const float w = wave_max(r.top);
    r.lift(w, heat);
    r.sum = wave_sum(r.sum);
    r.turn = wave_sum(r.turn);
    if (lane == 0) {
        s.top[wave] = r.top;
        s.sum[wave] = r.sum;
        s.turn[wave] = r.turn;
    }
    __syncthreads();
    r = Running{};
#pragma unroll
    for (int i = 0; i < kWaves; i++) r.join(s.top[i], s.sum[i], s.turn[i], heat);
}

// The 64 classes are those of a thread's lane.
__device__ __forceinline__ uint32_t floor_of(const Shared &s, uint32_t k) {
    float m = -infinity();
#pragma unroll
    for (int i = 0; i < kWaves; i++) m = fmaxf(m, s.tops[i][threadIdx.x % 64]);
    return kth_of_lanes(m == -infinity() ? 0u : ordered(m), k);
}

// A workgroup a row.
template <class T>
__global__ void __launch_bounds__(kThreads)
k_log_rows(LogArgs a) {
    __shared__ Shared s;
    const size_t row = row_of();
    if (row >= a.rows) return;
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    const Heat heat(t);
    Running r;
    bool nan = false;
    for (uint32_t i = threadIdx.x * kVec; i < a.vocab; i += kThreads * kVec) {
        float v[kVec];
        fetch(logits, mask, i, a.vocab, a.vocab, v);
#pragma unroll
        for (int e = 0; e < kVec; e++) nan |= v[e] != v[e];
        r.add(v, heat);
    }
    const float mine = r.top;
    nan = __syncthreads_or(nan);
    share(s, r, heat);
    if (nan) r.sum = not_a_number();
    const uint32_t k = max(a.top, 1u), floor = a.top || t == 0.f ? floor_of(s, k) : 0u;
    finish<T>(a, row, t, r, floor, s, [&](auto f) {
        if (mine == -infinity() || ordered(mine) < floor) return;
        for (uint32_t i = threadIdx.x * kVec; i < a.vocab; i += kThreads * kVec) {
            float v[kVec];
            fetch(logits, mask, i, a.vocab, a.vocab, v);
            f(v, a.vocab >= kVec ? min(i, a.vocab - kVec) : i);
        }
    });
}

// Few rows: stretches of `chunk` places by a workgroup each, joined by a second launch.  A
// stretch leaves its LogPart and the largest of each wave's places; the second launch looks at
// those waves' places again whose largest reach the threshold.
template <class T>
__global__ void __launch_bounds__(kThreads)
k_log_parts(LogArgs a) {
    __shared__ Shared s;
    const size_t job = row_of(), row = job / a.chunks;
    if (row >= a.rows) return;
    const uint32_t begin = (uint32_t)(job % a.chunks) * a.chunk, end = min(begin + a.chunk, a.vocab);
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    const Heat heat(t);
    Running r;
    bool nan = false;
    for (uint32_t i = begin + threadIdx.x * kVec; i < end; i += kThreads * kVec) {
        float v[kVec];
        fetch(logits, mask, i, end, a.vocab, v);
#pragma unroll
        for (int e = 0; e < kVec; e++) nan |= v[e] != v[e];
        r.add(v, heat);
    }
    nan = __syncthreads_or(nan);
    share(s, r, heat);
    if (nan || (t > 0.f && r.top == infinity())) r.sum = not_a_number();
    LogPart *parts = static_cast<LogPart *>(a.parts);
    float *tops = reinterpret_cast<float *>(parts + a.rows * a.chunks);
    if (threadIdx.x == 0) parts[job] = {r.top, r.sum, r.turn, 0.f};
    if (threadIdx.x < kWaves) tops[job * kWaves + threadIdx.x] = s.top[threadIdx.x];
}

template <class T>
__global__ void __launch_bounds__(kThreads)
k_log_join(LogArgs a) {
    __shared__ Shared s;
    const size_t row = row_of();
    if (row >= a.rows) return;
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    const Heat heat(t);
    const LogPart *parts = static_cast<const LogPart *>(a.parts);
    const uint32_t groups = a.chunks * kWaves;
    const float *tops = reinterpret_cast<const float *>(parts + a.rows * a.chunks) + row * groups;
    Running r;
    bool nan = false;
    for (uint32_t i = threadIdx.x; i < a.chunks; i += kThreads) {
        const LogPart p = parts[row * a.chunks + i];
        nan |= p.sum != p.sum;
        r.join(p.top, p.sum, p.turn, heat);
    }
    nan = __syncthreads_or(nan);
    share(s, r, heat);
    if (nan) r.sum = not_a_number();
    const uint32_t k = max(a.top, 1u);
    uint32_t floor = 0;
    if ((a.top || t == 0.f) && r.sum == r.sum) {
        // classes here: a group's place modulo 64
        __syncthreads();
        float m = -infinity();
        for (uint32_t i = threadIdx.x; i < groups; i += kThreads) m = fmaxf(m, tops[i]);
        s.tops[threadIdx.x / 64][threadIdx.x % 64] = m;
        if (threadIdx.x == 0) s.groups = 0;
        __syncthreads();
        floor = floor_of(s, k);
        for (uint32_t i = threadIdx.x; i < groups; i += kThreads)
            if (tops[i] > -infinity() && ordered(tops[i]) >= floor) s.list[atomicAdd(&s.groups, 1u)] = i;
        __syncthreads();
    }
    finish<T>(a, row, t, r, floor, s, [&](auto f) {
        for (uint32_t n = threadIdx.x / 64; n < s.groups; n += kWaves) {
            const uint32_t group = s.list[n], begin = group / kWaves * a.chunk, end = min(begin + a.chunk, a.vocab);
            for (uint32_t i = begin + (group % kWaves * 64 + threadIdx.x % 64) * kVec; i < end; i += kThreads * kVec) {
                float v[kVec];
                fetch(logits, mask, i, end, a.vocab, v);
                f(v, min(i, a.vocab - kVec));
            }
        }
    });
}

// One workgroup a row where rows are many, stretches where they are few.
Cut cut_log_probs(size_t rows, uint32_t vocab) {
    const uint32_t least = kThreads * kVec;
    if (vocab <= 2 * least || rows >= 1024) return {vocab, 1};
    const uint64_t want = std::max<uint64_t>(1, (uint64_t)rows * vocab / (2048 * least));  // vectors a thread
    uint64_t chunk = std::min<uint64_t>(want, 8) * least;
    const uint64_t most = kMostGroups / kWaves;
    chunk = std::max<uint64_t>(chunk, ((vocab + most - 1) / most + least - 1) / least * least);
    return {(uint32_t)chunk, (uint32_t)((vocab + chunk - 1) / chunk)};
}

size_t log_probs_bytes(size_t rows, const Cut &c) {
    return c.chunks == 1 ? 0 : rows * c.chunks * (sizeof(LogPart) + kWaves * sizeof(float));
}

}  // namespace

}  // namespace pfa

using namespace pfa;

extern "C" {

int pfa_log_probs_workspace(size_t rows, size_t vocab, size_t *bytes) {
    return guarded([&] {
        check_rows(rows, vocab, "pfa_log_probs_workspace");
        require(bytes != nullptr, "null argument");
        *bytes = log_probs_bytes(rows, cut_log_probs(rows, (uint32_t)vocab));
    });
}

int pfa_token_log_probs(const void *logits, size_t stride, int type, size_t rows, size_t vocab, const void *tokens,
                        int token_bytes, size_t given, size_t top, const float *temperatures, double temperature,
                        const uint8_t *mask, size_t mask_stride, float *log_probs, float *entropy, float *top_log_probs,
                        void *top_tokens, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        const size_t size = type_bytes(type);
        require(token_bytes == 4 || token_bytes == 8, "tokens have 4 or 8 bytes");
        check_rows(rows, vocab, "pfa_token_log_probs");
        require(given <= kMostWidth, "pfa_token_log_probs: more than 2^30 tokens a row");
        require(top <= kMostTop, "pfa_token_log_probs: at most 64 alternatives");
        require(temperatures || temperature >= 0, "pfa_token_log_probs: the temperature must be 0 or more");
        require(!workspace_bytes || workspace, "null workspace");
        if (rows == 0) return;
        require(entropy && (vocab == 0 || logits) && (given == 0 || (tokens && log_probs)) &&
                    (top == 0 || (top_log_probs && top_tokens)),
                "null argument");
        require(apart(rows, stride, vocab) && (!mask || apart(rows, mask_stride, vocab)), "rows overlap");
        aligned(logits, size, "logits");
        aligned(tokens, token_bytes, "tokens");
        aligned(top_tokens, token_bytes, "top_tokens");
        aligned(temperatures, 4, "temperatures");
        aligned(log_probs, 4, "log_probs");
        aligned(entropy, 4, "entropy");
        aligned(top_log_probs, 4, "top_log_probs");
        const Cut cut = cut_log_probs(rows, (uint32_t)vocab);
        const size_t need = log_probs_bytes(rows, cut);
        require(workspace_bytes >= need, "pfa_token_log_probs: the workspace needs " + std::to_string(need) + " bytes");
        aligned(workspace, 16, "workspace");
        const LogArgs a{logits,        tokens,    temperatures,    mask,           log_probs,       entropy,   top_log_probs,
                        top_tokens,    workspace, rows,            stride,         mask_stride,     (uint32_t)vocab,
                        (uint32_t)given, (uint32_t)top, cut.chunk, cut.chunks, (float)temperature, token_bytes == 8};
        const hipStream_t s = as_stream(stream);
        with_type(type, [&](auto t) {
            using T = decltype(t);
            if (cut.chunks == 1) {
                hipLaunchKernelGGL(k_log_rows<T>, row_grid(rows), dim3(kThreads), 0, s, a);
            } else {
                hipLaunchKernelGGL(k_log_parts<T>, row_grid(rows * cut.chunks), dim3(kThreads), 0, s, a);
                hipLaunchKernelGGL(k_log_join<T>, row_grid(rows), dim3(kThreads), 0, s, a);
            }
        });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
