// Log probabilities of given tokens, the entropy of the distribution, and its largest alternatives, from
// logits: with d = (l - m) / t, m the largest allowed logit of a row, and S = sum e^d,
//   log p = d - log S,   H = log S - (sum e^d d) / S.
// The logits are read once, with a running maximum a thread, and no probability is written.
//
// The alternatives need no order of the row.  The largest logits of 64 or 128 classes of its places (the lanes' classes)
// are as many places' logits: their k-th largest has k places at or above it, so the k largest of the row are among
// the places that reach it.  Those are collected (about k of them where the classes share them out evenly) and
// ranked by comparing each with all.  Where they are too many to collect (long ties, logits in step with the
// classes), they are thrown into other classes, whose k-th largest is the next threshold.
#include <algorithm>
#include <cmath>

#include "rows.h"

namespace pfa {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;  // of a row, and of a stretch of one
constexpr int kRowThreads = 512;                       // of a long row where rows are few
constexpr int kJoinThreads = 512;                      // that join a row's stretches
constexpr int kUnroll = 4;                             // vectors of a thread on their way at once
constexpr uint32_t kMostTop = 64;        // alternatives: at most half of the classes of places
constexpr uint32_t kKept = 512;          // places that one collection holds (9 bits number them)
constexpr uint32_t kListed = 1024;       // groups of places that a collection looks at, all of them where more reach it
constexpr uint32_t kRowGroups = 2048;    // groups of places a whole row
constexpr uint32_t kChunkGroups = 16;    // groups of places a stretch
constexpr uint32_t kMostGroups = 1024;   // groups of places a cut row
constexpr float kLn2 = 0.69314718055994531f;

struct LogArgs {
    const void *logits;
    const void *tokens;  // [rows][given] of 4 or 8 bytes
    const float *temperatures;
    const uint8_t *mask;
    float *log_probs, *entropy, *top_log_probs;  // [rows][given], [rows], [rows][top]
    void *top_tokens;                            // [rows][top], like tokens
    void *parts;  // [rows][chunks] of LogPart, then the largest of [rows][chunks kChunkGroups] groups of places
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
    // V more logits; their largest
    template <int V>
    __device__ __forceinline__ float add(const float (&v)[V], const Heat &heat) {
        float m = v[0];
#pragma unroll
        for (int e = 1; e < V; e++) m = fmaxf(m, v[e]);
        if (m > top) lift(m, heat);
        const float base = top == -infinity() ? 0.f : top;
#pragma unroll
        for (int e = 0; e < V; e++) {
            const float g = exponent(v[e], base, heat), w = __builtin_amdgcn_exp2f(g);
            sum += w;
            turn = fmaf(w, g, turn);
        }
        return m;
    }
};

// A row's logits, and which of its places are allowed.  MASKED: a call without a mask has no code for one in its loop.
template <class T, bool MASKED>
struct Row {
    const T *logits;
    const uint8_t *mask;
    uint32_t vocab;
    __device__ __forceinline__ Row(const LogArgs &a, size_t row)
        : logits(static_cast<const T *>(a.logits) + row * a.stride),
          mask(MASKED ? a.mask + row * a.mask_stride : nullptr),
          vocab(a.vocab) {}

    // place of the first of the vector at `own`: the row's last vector starts early
    __device__ __forceinline__ uint32_t at(uint32_t own) const { return vocab >= kVec ? min(own, vocab - kVec) : own; }
    // kVec logits from own on, -infinity where none is allowed, before own and behind the row
    __device__ __forceinline__ void fetch(uint32_t own, float *v) const {
        float w[kVec];
        if (vocab >= kVec) {
            allowed_logits(logits, MASKED ? mask : nullptr, at(own), own, w);
        } else {
#pragma unroll
            for (int e = 0; e < kVec; e++)
                w[e] = own + e < vocab && (!MASKED || mask[own + e]) ? (float)logits[own + e] : -infinity();
        }
#pragma unroll
        for (int e = 0; e < kVec; e++) v[e] = w[e];
    }
    // kUnroll vectors a thread from `begin` on, the workgroup's side by side; those behind `end` are -infinity
    template <int THREADS>
    __device__ __forceinline__ void fetch_all(uint32_t begin, uint32_t end, float (&v)[kUnroll * kVec]) const {
        if (begin + kUnroll * THREADS * kVec <= end) {  // all there: no load behind a branch, nothing to clear
            const uint32_t i = begin + threadIdx.x * kVec;
            auto load = [&](int j) {
                float w[kVec];
                load_vec<kVec>(logits + i + j * THREADS * kVec, w);
#pragma unroll
                for (int e = 0; e < kVec; e++) v[j * kVec + e] = w[e];
            };
            if (!MASKED) {
#pragma unroll
                for (int j = 0; j < kUnroll; j++) load(j);
                return;
            }
            uint32_t w[kUnroll][2];
#pragma unroll
            for (int j = 0; j < kUnroll; j++) {
                __builtin_memcpy(w[j], mask + i + j * THREADS * kVec, 8);
                load(j);
            }
#pragma unroll
            for (int j = 0; j < kUnroll; j++)
#pragma unroll
                for (int e = 0; e < kVec; e++)
                    v[j * kVec + e] = w[j][e / 4] >> (e % 4 * 8) & 0xff ? v[j * kVec + e] : -infinity();
        } else {
#pragma unroll
            for (int j = 0; j < kUnroll; j++) {
                const uint32_t i = begin + (j * THREADS + threadIdx.x) * kVec;
                if (i < end) {
                    fetch(i, v + j * kVec);
                } else {
#pragma unroll
                    for (int e = 0; e < kVec; e++) v[j * kVec + e] = -infinity();
                }
            }
        }
    }
};

template <int V>
__device__ __forceinline__ bool any_nan(const float (&v)[V]) {
    bool nan = false;
#pragma unroll
    for (int e = 0; e < V; e += 2) nan |= __builtin_isunordered(v[e], v[e + 1]);
    return nan;
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
template <int THREADS>
struct Shared {
    uint64_t kept[kKept], limit;
    float tops[THREADS / 64][64];
    float top[THREADS / 64], sum[THREADS / 64], turn[THREADS / 64];
    uint32_t count, listed, first;
    uint16_t list[kListed];
};

// The k-th largest of N numbers in each of 64 lanes, in every lane
template <int N>
__device__ __forceinline__ uint32_t kth_of_lanes(const uint32_t (&v)[N], uint32_t k) {
    uint32_t above[N] = {}, least = 0xffffffffu;  // how many are larger
#pragma unroll
    for (int j = 0; j < 64 * N; j++) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)v[j / 64], j % 64);
#pragma unroll
        for (int i = 0; i < N; i++) above[i] += o > v[i];
    }
    // the smallest of those with fewer than k above them
#pragma unroll
    for (int i = 0; i < N; i++)
        if (above[i] < k) least = min(least, v[i]);
    return ~wave_max(~least);
}

// The `count` collected keys by rank; the first k of them to `put(rank, key)`, the k-th to shared.limit
template <int THREADS, class F>
__device__ __forceinline__ void rank_kept(Shared<THREADS> &s, uint32_t count, uint32_t k, F put) {
    for (uint32_t i = threadIdx.x; i < count; i += THREADS) {
        const uint64_t mine = s.kept[i];
        uint32_t above = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < count; j++) above += s.kept[j] > mine;
        if (above + 1 == k) s.limit = mine;
        if (above < k) put(above, mine);
    }
}

// The k largest places of a row: put(rank, key) once for each of them.  k places or more have logits of `floor` or
// more, as ordered().  The row's places are in `groups` groups, tops[group] the largest logit of one, of `vectors` vectors each,
// vector(group, i) the place of the i-th or vocab and more.
template <int THREADS, class R, class V, class F>
__device__ __forceinline__ void largest(Shared<THREADS> &s, const R &row, uint32_t k, uint32_t floor, const float *tops,
                                        uint32_t groups, uint32_t vectors, V vector, F put) {
    uint64_t limit = max((uint64_t)floor << 32, (uint64_t)1);
    // f(key) for every place that reaches the limit
    auto scan = [&](auto f) {
        __syncthreads();
        if (threadIdx.x == 0) s.count = s.listed = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < groups; i += THREADS)
            if (key_of(tops[i], 0) >= limit) {  // no place of it can reach the limit otherwise
                const uint32_t n = atomicAdd(&s.listed, 1u);
                if (n < kListed) s.list[n] = (uint16_t)i;
            }
        __syncthreads();
        const bool all = s.listed > kListed;
        const uint32_t jobs = (all ? groups : s.listed) * vectors;
        for (uint32_t n = threadIdx.x; n < jobs; n += THREADS) {
            const uint32_t own = vector(all ? n / vectors : (uint32_t)s.list[n / vectors], n % vectors);
            if (own >= row.vocab) continue;
            float v[kVec];
            row.fetch(own, v);
            const uint32_t at = row.at(own);
#pragma unroll
            for (int e = 0; e < kVec; e++) {
                const uint64_t key = key_of(v[e], at + e);
                if (key >= limit) f(key);
            }
        }
        __syncthreads();
    };
    for (uint32_t turn = 1;; turn += 2) {
        scan([&](uint64_t key) {
            const uint32_t n = atomicAdd(&s.count, 1u);
            if (n < kKept) s.kept[n] = key;
        });
        const uint32_t count = s.count;
        if (count <= kKept) return rank_kept(s, count, k, put);
        // Too many: the largest of kKept classes that places are thrown into, others each time.  Their k-th largest
        // leaves about k places, whatever the row looks like.
        for (uint32_t i = threadIdx.x; i < kKept; i += THREADS) s.kept[i] = 0;
        if (threadIdx.x == 0) s.limit = limit;
        scan([&](uint64_t key) {
            const uint32_t into = (uint32_t)key * (0x9e3779b1u * turn) >> 23;
            atomicMax((unsigned long long *)&s.kept[into], (unsigned long long)key);
        });
        rank_kept(s, kKept, k, [](uint32_t, uint64_t) {});
        __syncthreads();
        limit = max(limit, s.limit);  // 0 where fewer than k classes have a place
    }
}

__device__ __forceinline__ void set_token(const LogArgs &a, size_t i, int64_t v) {
    if (a.tokens64)
        static_cast<int64_t *>(a.top_tokens)[i] = v;
    else
        static_cast<int32_t *>(a.top_tokens)[i] = (int32_t)v;
}

// A thread's first given token and its logit, asked for before the row is read
struct Given {
    int64_t token;
    float logit;
    template <class R>
    __device__ __forceinline__ Given(const LogArgs &a, size_t r, const R &row, uint32_t i) : token(-1), logit(0.f) {
        if (i >= a.given) return;
        token = a.tokens64 ? static_cast<const int64_t *>(a.tokens)[r * a.given + i]
                           : static_cast<const int32_t *>(a.tokens)[r * a.given + i];
        const bool there = token >= 0 && token < (int64_t)a.vocab && (!row.mask || row.mask[token]);
        token = there ? token : -1;
        if (there) logit = (float)row.logits[token];
    }
};

// What row r gives, its sums known: by all threads of a workgroup.  The rest as in largest().
template <int THREADS, class R, class V>
__device__ __forceinline__ void finish(const LogArgs &a, size_t r, const R &row, float t, const Running &run,
                                       const Given &early, uint32_t floor, Shared<THREADS> &s, const float *group_tops,
                                       uint32_t groups, uint32_t vectors, V vector) {
    const bool nan = run.sum != run.sum || !(t >= 0.f) || (t > 0.f && run.top == infinity()), none = run.top == -infinity();
    const bool greedy = t == 0.f;
    const float log_sum = logf(run.sum);
    // differences are formed halved: see Heat
    const float half = t >= 1.f ? 0.5f : 1.f;
    auto log_prob = [&](float l) {
        if (nan) return not_a_number();
        if (none || l == -infinity()) return -infinity();
        return (l * half - run.top * half) / (t * half) - log_sum;
    };
    const uint32_t k = nan || none ? 0 : greedy ? max(a.top, 1u) : a.top;
    float *tops = a.top_log_probs + r * a.top;
    if (k) {
        largest(s, row, k, floor, group_tops, groups, vectors, vector, [&](uint32_t rank, uint64_t key) {
            const uint32_t i = 0xffffffffu - (uint32_t)key;
            if (rank == 0) s.first = i;
            if (rank < a.top) {
                set_token(a, r * a.top + rank, i);
                tops[rank] = greedy ? (rank ? -infinity() : 0.f) : log_prob(logit_of(key));
            }
        });
        if (greedy) __syncthreads();
    }
    const uint32_t found = k ? min(s.count, k) : 0;
    for (uint32_t i = found + threadIdx.x; i < a.top; i += THREADS) {
        set_token(a, r * a.top + i, -1);
        tops[i] = nan ? not_a_number() : -infinity();
    }
    for (uint32_t i = threadIdx.x; i < a.given; i += THREADS) {
        const Given g = i == threadIdx.x ? early : Given(a, r, row, i);
        a.log_probs[r * a.given + i] = g.token < 0      ? -infinity()
                                       : greedy && !nan ? (k && (uint32_t)g.token == s.first ? 0.f : -infinity())
                                                        : log_prob(g.logit);
    }
    if (threadIdx.x == 0)
        a.entropy[r] = nan ? not_a_number() : none || greedy ? 0.f : log_sum - kLn2 * (run.turn / run.sum);
}

// sums of the workgroup's threads; tops[w] holds its waves' lanes' largest afterwards
template <int THREADS>
__device__ __forceinline__ void share(Shared<THREADS> &s, Running &r, const Heat &heat) {
    const uint32_t wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    s.tops[wave][lane] = r.top;
    r.lift(wave_max(r.top), heat);
    r.sum = wave_sum(r.sum);
    r.turn = wave_sum(r.turn);
    if (lane == 0) {
        s.top[wave] = r.top;
        s.sum[wave] = r.sum;
        s.turn[wave] = r.turn;
    }
    __syncthreads();
    // every wave joins the waves' sums, one a lane
    r = Running{};
    if (lane < THREADS / 64) {
        r.top = s.top[lane];
        r.sum = s.sum[lane];
        r.turn = s.turn[lane];
    }
    r.lift(wave_max(r.top), heat);
    r.sum = wave_sum(r.sum);
    r.turn = wave_sum(r.turn);
}

// The classes are a thread's lane; for more than half as many alternatives, its lane and whether its wave is odd
// (64 of 64 classes: some 300 places reach the threshold and 1 of 131072 takes 21 us; of 128: 90).
template <int THREADS>
__device__ __forceinline__ uint32_t floor_of(const Shared<THREADS> &s, uint32_t k) {
    float m[2] = {-infinity(), -infinity()};
#pragma unroll
    for (int i = 0; i < THREADS / 64; i++) m[i % 2] = fmaxf(m[i % 2], s.tops[i][threadIdx.x % 64]);
    uint32_t v[2];
#pragma unroll
    for (int i = 0; i < 2; i++) v[i] = m[i] == -infinity() ? 0u : ordered(m[i]);
    if (k > 32) return kth_of_lanes(v, k);
    const uint32_t one[1] = {max(v[0], v[1])};
    return kth_of_lanes(one, k);
}

// A workgroup a row.  Bound by memory: 2048 x 131072 bf16 104-109 us (4.9-5.2 TB/s), 1024 x 131072 float32 96 us (5.6
// TB/s).  Shorter rows pay for the search of the alternatives behind the reading, 4096 x 32768 bf16 66 us (4.1 TB/s), with a
// mask for each row 89 us (4.5 TB/s).
template <class T, bool MASKED, int THREADS>
__global__ void __launch_bounds__(THREADS, !MASKED ? 8 : THREADS == kThreads ? 6 : 4)
k_log_rows(LogArgs a) {
    __shared__ Shared<THREADS> s;
    __shared__ float group_tops[kRowGroups];
    const size_t r = row_of();
    if (r >= a.rows) return;
    const Row<T, MASKED> row(a, r);
    const float t = a.temperatures ? a.temperatures[r] : a.temperature;
    const Given early(a, r, row, threadIdx.x);
    const Heat heat(t);
    Running run;
    bool nan = false;
    constexpr uint32_t kRound = kUnroll * THREADS * kVec;
    // a group is `span` rounds of a thread
    const uint32_t rounds = (a.vocab + kRound - 1) / kRound, span = (rounds + kRowGroups / THREADS - 1) / (kRowGroups / THREADS);
    float group_top = -infinity();
    for (uint32_t i = 0, left = span, group = threadIdx.x; i < rounds; i++) {
        float v[kUnroll * kVec];
        row.template fetch_all<THREADS>(i * kRound, a.vocab, v);
        nan |= any_nan(v);
        group_top = fmaxf(group_top, run.add(v, heat));
        if (--left == 0 || i + 1 == rounds) {
            group_tops[group] = group_top;
            group += THREADS;
            group_top = -infinity();
            left = span;
        }
    }
    nan = __syncthreads_or(nan);
    share(s, run, heat);
    if (nan) run.sum = not_a_number();
    const uint32_t k = max(a.top, 1u), floor = a.top || t == 0.f ? floor_of(s, k) : 0u;
    finish(a, r, row, t, run, early, floor, s, group_tops, (rounds + span - 1) / max(span, 1u) * THREADS, span * kUnroll,
           [&](uint32_t group, uint32_t i) {
               const uint64_t at = ((uint64_t)(group / THREADS) * span * kUnroll + i) * THREADS + group % THREADS;
               return (uint32_t)min(at * kVec, (uint64_t)0xffffffffu);
           });
}

// Few rows: stretches of `chunk` places by a workgroup each, joined by a second launch.  A stretch leaves its LogPart
// and the largest of each 16 lanes' places.  1 x 131072 float32 with 20 alternatives: 4.2 us and 7.1-7.8 of the join,
// which is a chain of small steps: parts, threshold, groups, their places, ranks.
template <class T, bool MASKED>
__global__ void __launch_bounds__(kThreads, MASKED ? 6 : 8)
k_log_parts(LogArgs a) {
    __shared__ Shared<kThreads> s;
    const size_t job = row_of(), r = job / a.chunks;
    if (r >= a.rows) return;
    const uint32_t begin = (uint32_t)(job % a.chunks) * a.chunk, end = min(begin + a.chunk, a.vocab);
    const Row<T, MASKED> row(a, r);
    const float t = a.temperatures ? a.temperatures[r] : a.temperature;
    const Heat heat(t);
    Running run;
    bool nan = false;
    if (a.chunk == kThreads * kVec) {  // the shortest: a vector each
        float v[kVec];
        row.fetch(begin + threadIdx.x * kVec, v);
        nan = any_nan(v);
        run.add(v, heat);
    } else {
        for (uint32_t i = begin; i < end; i += kUnroll * kThreads * kVec) {
            float v[kUnroll * kVec];
            row.template fetch_all<kThreads>(i, end, v);
            nan |= any_nan(v);
            run.add(v, heat);
        }
    }
    nan = __syncthreads_or(nan);
    float most = run.top;
#pragma unroll
    for (int d = 1; d < 64 / (kChunkGroups / kWaves); d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    share(s, run, heat);
    if (nan || (t > 0.f && run.top == infinity())) run.sum = not_a_number();
    LogPart *parts = static_cast<LogPart *>(a.parts);
    float *tops = reinterpret_cast<float *>(parts + a.rows * a.chunks);
    if (threadIdx.x == 0) parts[job] = {run.top, run.sum, run.turn, 0.f};
    constexpr uint32_t kLanes = kThreads / kChunkGroups;
    if (threadIdx.x % kLanes == 0) tops[job * kChunkGroups + threadIdx.x / kLanes] = most;
}

template <class T, bool MASKED>
__global__ void __launch_bounds__(kJoinThreads)
k_log_join(LogArgs a) {
    __shared__ Shared<kJoinThreads> s;
    __shared__ float group_tops[kMostGroups];
    const size_t r = row_of();
    if (r >= a.rows) return;
    const Row<T, MASKED> row(a, r);
    const float t = a.temperatures ? a.temperatures[r] : a.temperature;
    const Given early(a, r, row, threadIdx.x);
    const Heat heat(t);
    const LogPart *parts = static_cast<const LogPart *>(a.parts);
    const uint32_t groups = a.chunks * kChunkGroups;
    const float *tops = reinterpret_cast<const float *>(parts + a.rows * a.chunks) + r * groups;
    Running run;
    if (threadIdx.x < a.chunks) {
        const LogPart p = parts[r * a.chunks + threadIdx.x];
        run.top = p.top;
        run.sum = p.sum;
        run.turn = p.turn;
    }
    float most = -infinity();  // classes here: a group's place modulo 64
#pragma unroll
    for (uint32_t i = threadIdx.x; i < kMostGroups; i += kJoinThreads) {
        const float top = i < groups ? tops[i] : -infinity();
        group_tops[i] = top;
        most = fmaxf(most, top);
    }
    const bool nan = __syncthreads_or(run.sum != run.sum);
    share(s, run, heat);
    if (nan) run.sum = not_a_number();
    const uint32_t k = max(a.top, 1u);
    uint32_t floor = 0;
    if ((a.top || t == 0.f) && !nan) {
        __syncthreads();
        s.tops[threadIdx.x / 64][threadIdx.x % 64] = most;
        __syncthreads();
        floor = floor_of(s, k);
    }
    constexpr uint32_t kLanes = kThreads / kChunkGroups;
    finish(a, r, row, t, run, early, floor, s, group_tops, groups, a.chunk / kChunkGroups / kVec,
           [&](uint32_t group, uint32_t i) {
               const uint64_t own = (uint64_t)(group / kChunkGroups) * a.chunk +
                                    ((i / kLanes * kChunkGroups + group % kChunkGroups) * kLanes + i % kLanes) * kVec;
               return (uint32_t)min(own, (uint64_t)0xffffffffu);
           });
}

// How a call is cut: chunks == 1 is one workgroup of `threads` a row.
struct LogCut {
    uint32_t chunk, chunks;
    int threads;
};

// Measured, bf16, us, rows of 256 threads / of 512 / cut (two launches): 16 rows of 8192 7.5 / 8.5, of 16384 8.5 / 8.3, of 32768
// 10.3 / 9.7, of 65536 14.0 / 12.3 / 13, of 131072 21 / 18 / 13; 128 of 65536 16.5 / 13.6 / 18.5, of 131072 24.5 / 19.1 / 21;
// 256 of 32768 12.5 / 11.3, of 131072 25 / 20; 320 of 32768 13.8 / 14.2, of 131072 float32 39 / 45.  1024 threads are 512's
// equal at best (16 of 131072) and up to 2.5 us slower to begin and end.  Stretches have one vector a thread, and four
// where those would be more than eight workgroups a CU.
LogCut cut_log_probs(size_t rows, uint32_t vocab) {
    if (vocab <= 65536 || rows > vocab / 4096)
        return {vocab, 1, vocab >= 16384 && rows <= 256 ? kRowThreads : kThreads};
    const uint64_t least = kThreads * kVec, most = kMostGroups / kChunkGroups;  // places, stretches
    uint64_t chunk = rows * vocab <= 2048 * least && vocab <= least * most ? least : kUnroll * least;
    chunk *= (vocab + chunk * most - 1) / (chunk * most);
    return {(uint32_t)chunk, (uint32_t)((vocab + chunk - 1) / chunk), kThreads};
}

template <class T, bool MASKED>
void launch_log_probs(const LogArgs &a, const LogCut &cut, hipStream_t s) {
    if (cut.chunks == 1 && cut.threads == kThreads) {
        hipLaunchKernelGGL((k_log_rows<T, MASKED, kThreads>), row_grid(a.rows), dim3(kThreads), 0, s, a);
    } else if (cut.chunks == 1) {
        hipLaunchKernelGGL((k_log_rows<T, MASKED, kRowThreads>), row_grid(a.rows), dim3(kRowThreads), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_log_parts<T, MASKED>), row_grid(a.rows * cut.chunks), dim3(kThreads), 0, s, a);
        hipLaunchKernelGGL((k_log_join<T, MASKED>), row_grid(a.rows), dim3(kJoinThreads), 0, s, a);
    }
}

size_t log_probs_bytes(size_t rows, const LogCut &c) {
    return c.chunks == 1 ? 0 : rows * c.chunks * (sizeof(LogPart) + kChunkGroups * sizeof(float));
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
        const LogCut cut = cut_log_probs(rows, (uint32_t)vocab);
        const size_t need = log_probs_bytes(rows, cut);
        require(workspace_bytes >= need, "pfa_token_log_probs: the workspace needs " + std::to_string(need) + " bytes");
        aligned(workspace, 16, "workspace");
        const LogArgs a{logits,        tokens,    temperatures,    mask,           log_probs,       entropy,   top_log_probs,
                        top_tokens,    workspace, rows,            stride,         mask_stride,     (uint32_t)vocab,
                        (uint32_t)given, (uint32_t)top, cut.chunk, cut.chunks, (float)temperature, token_bytes == 8};
        const hipStream_t s = as_stream(stream);
        with_type(type, [&](auto t) {
            using T = decltype(t);
            if (mask)
                launch_log_probs<T, true>(a, cut, s);
            else
                launch_log_probs<T, false>(a, cut, s);
        });
        PFA_HIP(hipGetLastError());
    });
}

}  // extern "C"
