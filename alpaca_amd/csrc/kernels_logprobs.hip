// Of rows of logits x: the log probability of a given token, x_t - log sum exp x, the
// entropy log sum exp x - sum p x, and the likeliest tokens with theirs.
//
// One pass over a row takes its maximum m, s = sum e^(x - m) and t = sum e^(x - m)
// (x - m), a running triple a thread whose reference follows the thread's maximum;
// log p = (x - m) - log s, and the entropy is log s - t / s.  Bound by memory.
//
// The top n (at most 32): the row falls to 64 groups of 4 threads, and the n-th largest of
// the groups' maxima is a bound that n values reach, so that of a row in any but a contrived
// order little more than n do.  The threads whose maximum reaches it read their part of the row
// again (it is a cache's by then) and put what reaches it into LDS, where its rank is the
// number of better ones: larger, or as large and of a lower index.
//
// Few rows are split over workgroups, whose triples and best tokens the last one to arrive
// joins in the same launch.
#include "logprobs.h"

#include <algorithm>

#include "attn_parts.h"

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMostTop = kLogprobsMostTop, kGroups = 64;
constexpr int kAbove = 768, kEqual = 256, kListed = kAbove + kEqual;  // candidates in LDS
constexpr int kMostSplits = 32;
static_assert(kMostSplits * kMostTop <= kListed, "the parts' tokens in LDS");
constexpr int kPart = 4 + 2 * kMostTop;  // floats of a part in the workspace
constexpr float kLog2e = 1.4426950408889634f;

struct Sums {
    float m = -INFINITY, s = 0.f, t = 0.f;
    // Taken from the reference m to `to`, at least as large.
    __device__ __forceinline__ void move(float to) {
        if (m == to) return;
        const float f = __builtin_amdgcn_exp2f((m - to) * kLog2e);
        t = m == -INFINITY ? s * f : (t + s * (m - to)) * f;  // (nothing yet, but perhaps a NaN in s)
        s *= f;
        m = to;
    }
};
__device__ __forceinline__ Sums wave_total(Sums x) {
    x.move(wave_max(x.m));
    x.s = wave_sum(x.s);
    x.t = wave_sum(x.t);
    return x;
}

// Part [begin, end) of a row, and which of its elements are thread i's: `head` ones up to the first
// 16-byte line, then every kThreads-th line, then what is left.
template <typename T>
struct Slice {
    static constexpr int V = 16 / sizeof(T);
    const T* x;
    int begin, n, head, lines;
    __device__ __forceinline__ Slice(const T* row, int from, int to) : x(row + from), begin(from), n(to - from) {
        const int off = (int)((uintptr_t)x & 15) / (int)sizeof(T);
        head = min(off ? V - off : 0, n);
        lines = (n - head) / V;
    }
    // U lines of thread i from its k-th on, -inf past the last; returns the first one's element.
    template <int U>
    __device__ __forceinline__ void load(int k, float (&y)[U * V]) const {
        typedef T TV __attribute__((ext_vector_type(V)));
        const AS_GLOBAL TV* p = (const AS_GLOBAL TV*)(x + head);
        TV u[U];
#pragma unroll
        for (int i = 0; i < U; i++) u[i] = p[min(k + i * kThreads, lines - 1)];
#pragma unroll
        for (int i = 0; i < U; i++)
#pragma unroll
            for (int e = 0; e < V; e++) y[i * V + e] = k + i * kThreads < lines ? (float)u[i][e] : -INFINITY;
    }
    // The element of thread i that lies outside the lines (at most one before and one behind), or -1.
    __device__ __forceinline__ int before(int i) const { return i < head ? i : -1; }
    __device__ __forceinline__ int behind(int i) const {
        const int e = head + lines * V + i;
        return e < n ? e : -1;
    }
    // f(value, element) for all of thread i's.
    template <typename F>
    __device__ __forceinline__ void each(int i, F f) const {
        constexpr int U = 32 / V;
        for (int k = i; k < lines; k += U * kThreads) {
            float y[U * V];
            load<U>(k, y);
#pragma unroll
            for (int j = 0; j < U; j++)
                if (k + j * kThreads < lines) {
#pragma unroll
                    for (int e = 0; e < V; e++) f(y[j * V + e], head + (k + j * kThreads) * V + e);
                }
        }
        if (before(i) >= 0) f((float)gptr(x)[before(i)], before(i));
        if (behind(i) >= 0) f((float)gptr(x)[behind(i)], behind(i));
    }
};

// Whether (a, i) ranks before (b, j): numbers before NaN, larger ones first, then the lower index.
__device__ __forceinline__ bool before(float a, int i, float b, int j) {
    if (a > b) return true;
    if (a < b) return false;
    const bool an = a != a, bn = b != b;
    return an == bn ? i < j : bn;
}

struct Shared {
    float m[kWaves], s[kWaves], t[kWaves];
    float group[kGroups];
    float value[kListed];
    int index[kListed];
    float best[kMostTop];
    int token[kMostTop];
    float bound;
    int above, equal, last;
    float wave_value[kWaves];
    int wave_index[kWaves];
};

// The n-th largest of the groups' maxima; by one wave.
__device__ __forceinline__ float nth_largest(const Shared& sh, int n) {
    const int lane = __lane_id();
    const float mine = sh.group[lane];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < kGroups; i++) {
        const float other = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), i));
        rank += other > mine || (other == mine && i < lane);
    }
    const uint64_t at = __builtin_amdgcn_ballot_w64(rank == n - 1);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), __builtin_ctzll(at | 1ull << 63)));
}

// The first `need` elements of the slice, in order, for which f holds, into best / token from `at` on; returns how
// many there were.  By one wave.
template <typename T, typename F>
__device__ __forceinline__ int fill(const Slice<T>& sl, Shared& sh, int at, int need, F f) {
    const int lane = __lane_id();
    int got = 0;
    for (int e0 = 0; e0 < sl.n && got < need; e0 += 64) {
        const int e = e0 + lane;
        const float x = e < sl.n ? (float)gptr(sl.x)[e] : 0.f;
        const bool take = e < sl.n && f(x);
        const uint64_t all = __builtin_amdgcn_ballot_w64(take);
        const int place = got + __builtin_popcountll(all & ((1ull << lane) - 1));
        if (take && place < need) {
            sh.best[at + place] = x;
            sh.token[at + place] = sl.begin + e;
        }
        got += __builtin_popcountll(all);
    }
    return min(got, need);
}

// The n best of `count` candidates in LDS; the threads have met behind their writing.
__device__ __forceinline__ void rank_listed(Shared& sh, int first, int count, int at, int n) {
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const float x = sh.value[first + i];
        const int e = sh.index[first + i];
        int rank = 0;
        for (int j = 0; j < count; j++) rank += before(sh.value[first + j], sh.index[first + j], x, e);
        if (rank < n) {
            sh.best[at + rank] = x;
            sh.token[at + rank] = e;
        }
    }
}

// The n best of a slice into best / token, whoever reads them having met the others afterwards; sh.group holds the groups'
// maxima, `mine` is the thread's own.  Places that the slice is too short for hold (NaN, INT32_MAX).
template <typename T>
__device__ void top_of_slice(const Slice<T>& sl, Shared& sh, int n, float mine) {
    const int tid = threadIdx.x;
    if (tid < 64) {
        const float b = nth_largest(sh, n);
        if (tid == 0) {
            sh.bound = b;
            sh.above = sh.equal = 0;
        }
        if (tid < n) {
            sh.best[tid] = NAN;
            sh.token[tid] = INT32_MAX;
        }
    }
    __syncthreads();
    const float bound = sh.bound;
    if (mine >= bound)
        sl.each(tid, [&](float x, int e) {
            if (x > bound) {
                const int i = atomicAdd(&sh.above, 1);
                if (i < kAbove) {
                    sh.value[i] = x;
                    sh.index[i] = sl.begin + e;
                }
            } else if (x == bound) {
                const int i = atomicAdd(&sh.equal, 1);
                if (i < kEqual) {
                    sh.value[kAbove + i] = x;
                    sh.index[kAbove + i] = sl.begin + e;
                }
            }
        });
    __syncthreads();
    const int above = sh.above, equal = sh.equal;
    if (above <= kAbove) {
        rank_listed(sh, 0, above, 0, n);
        if (above < n) {
            if (equal <= kEqual) rank_listed(sh, kAbove, equal, above, n - above);
            // more equal ones than the list holds (a row of masked tokens), and NaN where the numbers end
            if (tid < 64) {
                if (equal > kEqual) fill(sl, sh, above, n - above, [&](float x) { return x == bound; });
                const int got = min(n, above + equal);
                if (got < n) fill(sl, sh, got, n - got, [](float x) { return x != x; });
            }
        }
        return;
    }
    // a row in an order that hides the bound: the best, then the best behind it, n times
    float last = INFINITY;
    int last_e = -1;
    for (int r = 0; r < n; r++) {
        float b = -INFINITY;
        int be = INT32_MAX;
        sl.each(tid, [&](float x, int e) {
            if (x == x && before(last, last_e, x, e) && before(x, e, b, be)) {
                b = x;
                be = e;
            }
        });
        wave_argmax(b, be);
        if ((tid & 63) == 0) {
            sh.wave_value[tid >> 6] = b;
            sh.wave_index[tid >> 6] = be;
        }
        __syncthreads();
        for (int w = 0; w < kWaves; w++)
            if (w == 0 || before(sh.wave_value[w], sh.wave_index[w], last, last_e)) {
                last = sh.wave_value[w];
                last_e = sh.wave_index[w];
            }
        __syncthreads();
        if (tid == 0) {
            sh.best[r] = last;
            sh.token[r] = sl.begin + last_e;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads, 6) void logprobs_kernel(LogprobsArgs p) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, row = blockIdx.x / p.splits, part = blockIdx.x - row * p.splits, n = p.top;
    const T* x = (const T*)p.logits + (int64_t)row * p.stride;
    const Slice<T> sl(x, min((int64_t)p.vocab, (int64_t)part * p.each), min((int64_t)p.vocab, (part + 1ll) * p.each));
    constexpr int U = 4, N = U * Slice<T>::V;

    Sums sum;
    auto add = [&](auto& y) {
        constexpr int K = sizeof(y) / sizeof(float);
        float top = y[0];
#pragma unroll
        for (int i = 1; i < K; i++) top = fmaxf(top, y[i]);
        if (top > sum.m) sum.move(top);
        const float ref = sum.m == -INFINITY ? 0.f : sum.m;
#pragma unroll
        for (int i = 0; i < K; i++) {
            const float d = y[i] - ref, e = __builtin_amdgcn_exp2f(d * kLog2e);
            sum.s += e;
            sum.t = fmaf(e, fmaxf(d, -1000.f), sum.t);  // (a token masked by -inf adds 0)
        }
    };
    for (int k = tid; k < sl.lines; k += U * kThreads) {
        float y[N];
        sl.template load<U>(k, y);
        add(y);
    }
    if (sl.before(tid) >= 0 || sl.behind(tid) >= 0) {
        float y[2];
        y[0] = sl.before(tid) >= 0 ? (float)gptr(sl.x)[sl.before(tid)] : -INFINITY;
        y[1] = sl.behind(tid) >= 0 ? (float)gptr(sl.x)[sl.behind(tid)] : -INFINITY;
        add(y);
    }
    const float mine = sum.m;
    float group = fmaxf(mine, dpp_mov<0xB1>(mine));
    group = fmaxf(group, dpp_mov<0x4E>(group));
    if ((tid & 3) == 0) sh.group[tid >> 2] = group;
    sum = wave_total(sum);
    if ((tid & 63) == 0) {
        sh.m[tid >> 6] = sum.m;
        sh.s[tid >> 6] = sum.s;
        sh.t[tid >> 6] = sum.t;
    }
    __syncthreads();
    auto joined = [&](int count, auto get) {
        Sums r;
        for (int i = 0; i < count; i++) r.m = fmaxf(r.m, get(i).m);
        for (int i = 0; i < count; i++) {
            Sums y = get(i);
            y.move(r.m);
            r.s += y.s;
            r.t += y.t;
        }
        return r;
    };
    sum = joined(kWaves, [&](int w) {
        Sums y;
        y.m = sh.m[w];
        y.s = sh.s[w];
        y.t = sh.t[w];
        return y;
    });
    if (n) {
        top_of_slice(sl, sh, n, mine);
        __syncthreads();
    }
    if (p.splits > 1) {
        float* const at = p.parts + (int64_t)row * p.splits * kPart;
        float* const to = at + part * kPart;
        if (tid < n) put2(to + 4 + 2 * tid, sh.best[tid], __int_as_float(sh.token[tid]));
        if (tid == 64) {
            put2(to, sum.m, sum.s);
            put2(to + 2, sum.t, 0.f);
        }
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tid == 0) {
            int* counter = p.counters + row;
            sh.last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.splits - 1;
            if (sh.last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!sh.last) return;
        // wave 0: the triples, a lane a part; the tokens of all parts into LDS
        if (tid < 64) {
            Sums y;
            if (tid < p.splits) {
                const float2 a = get2(at + tid * kPart), b = get2(at + tid * kPart + 2);
                y.m = a.x;
                y.s = a.y;
                y.t = b.x;
            }
            y = wave_total(y);
            if (tid == 0) {
                sh.m[0] = y.m;
                sh.s[0] = y.s;
                sh.t[0] = y.t;
            }
        }
        const int listed = p.splits * n;
        for (int i = tid; i < listed; i += kThreads) {
            const float2 y = get2(at + i / n * kPart + 4 + 2 * (i % n));
            sh.value[i] = y.x;
            sh.index[i] = __float_as_int(y.y);
        }
        __syncthreads();
        sum.m = sh.m[0];
        sum.s = sh.s[0];
        sum.t = sh.t[0];
        if (n) {
            // the parts' tokens are in order: a bound from the first ones of each
            if (tid < kGroups) {
                const int s = tid % p.splits, r = tid / p.splits;
                sh.group[tid] = r < n ? fmaxf(-INFINITY, sh.value[s * n + r]) : -INFINITY;
            }
            __syncthreads();
            if (tid < 64) {
                const float b = nth_largest(sh, n);
                if (tid == 0) {
                    sh.bound = b;
                    sh.above = 0;
                }
            }
            __syncthreads();
            constexpr int PER = kListed / kThreads;
            float y[PER];
            int e[PER];
#pragma unroll
            for (int k = 0; k < PER; k++) {
                const int i = tid + k * kThreads;
                y[k] = i < listed ? sh.value[i] : NAN;
                e[k] = i < listed ? sh.index[i] : INT32_MAX;
            }
            const float bound = sh.bound;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PER; k++)
                if (tid + k * kThreads < listed && (y[k] >= bound || bound == -INFINITY)) {
                    const int i = atomicAdd(&sh.above, 1);
                    sh.value[i] = y[k];
                    sh.index[i] = e[k];
                }
            __syncthreads();
            rank_listed(sh, 0, sh.above, 0, n);
            __syncthreads();
        }
    }
    const float log_s = logf(sum.s);
    if (tid < n) {
        gptr(p.top_tokens)[(int64_t)row * n + tid] = sh.token[tid];
        gptr(p.top_logprobs)[(int64_t)row * n + tid] = (sh.best[tid] - sum.m) - log_s;
    }
    if (tid == 64 && p.entropy) gptr(p.entropy)[row] = log_s - sum.t / sum.s;
    if (tid == 128 && p.logprobs) {
        const int token = gptr(p.tokens)[row];
        const bool known = token >= 0 && token < p.vocab;
        gptr(p.logprobs)[row] = known ? ((float)gptr(x)[token] - sum.m) - log_s : NAN;
    }
}

}  // namespace

int64_t logprobs_workspace() { return kLogprobsMostSplitRows * 4 + (int64_t)kLogprobsParts * kPart * 4; }

// Workgroups of a row: one where the rows alone give every CU two; else until they do, each with 2,048 logits at least.
hipError_t launch_logprobs(bool f16_logits, LogprobsArgs p, void* workspace, hipStream_t st) {
    const int64_t want = (2ll * device_cus() + p.rows - 1) / p.rows;
    p.splits = 1;
    if (workspace && p.rows <= kLogprobsMostSplitRows)
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, kMostSplits, p.vocab / 2048, kLogprobsParts / p.rows}));
    p.each = (int)((((int64_t)p.vocab + p.splits - 1) / p.splits + 7) / 8 * 8);
    p.counters = (int*)workspace;
    p.parts = workspace ? (float*)((uint8_t*)workspace + kLogprobsMostSplitRows * 4) : nullptr;
    const unsigned grid = (unsigned)p.rows * p.splits;
    if (f16_logits) logprobs_kernel<f16><<<grid, kThreads, 0, st>>>(p);
    else logprobs_kernel<float><<<grid, kThreads, 0, st>>>(p);
    return hipGetLastError();
}
