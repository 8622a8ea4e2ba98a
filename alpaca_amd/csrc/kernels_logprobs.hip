// Of rows of logits x: the log probability of a given token, x_t - log sum exp x, the
// entropy log sum exp x - sum p x, and the likeliest tokens with theirs.
//
// One pass over a row takes its maximum m, s = sum e^(x - m) and t = sum e^(x - m)
// (x - m), a running triple a thread whose reference follows the thread's maximum;
// log p = (x - m) - log s, and the entropy is log s - t / s.  Bound by memory.
//
// The top n (at most 32): the row falls to 64 groups of 4 threads, and the n-th largest of
// the groups' maxima is a bound that n values reach, so that of a row in any but a contrived
// order little more than n do.  A thread keeps where its two largest groups of lines were:
// where those reach the bound they are read again (a thread that has more such groups: all of its
// part, by its whole wave; a short slice is still in registers), and what reaches it goes into LDS, where its
// rank is the number of better ones: larger, or as large and of a lower index.
//
// Few rows are split over workgroups, whose triples and best tokens the last one to arrive
// joins in the same launch.
//
// 2,048 float32 rows of 49,152, 403 MB: 70 us without top tokens (5.8 TB/s, what a plain sum
// reaches), 81 with 20, for which 5% more is read and a workgroup's memory idles while it ranks
// them.  One row: 8.4 us with 5 of them, 5.0 without, the launch, one trip to memory and the
// chain of joins.
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
constexpr float kFarthest = -1000.f;  // e to this power is 0 in float32: distances below it weigh nothing either

struct Sums {
    float m = -INFINITY, s = 0.f, t = 0.f;
    // Taken from the reference m to `to`, at least as large.
    __device__ __forceinline__ void move(float to) {
        if (m == to) return;
        const float f = __builtin_amdgcn_exp2f((m - to) * kLog2e);
        // (nothing yet, but perhaps a NaN in s; a reference of tokens masked by a large negative number is so far below that
        // f is 0: bounded as in the sums, s times the distance stays a number)
        t = m == -INFINITY ? s * f : (t + s * fmaxf(m - to, kFarthest)) * f;
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
    // Line k, which is thread k % kThreads's.
    __device__ __forceinline__ void load_line(int k, float (&y)[V]) const {
        typedef T TV __attribute__((ext_vector_type(V)));
        const TV u = ((const AS_GLOBAL TV*)(x + head))[min(k, lines - 1)];
#pragma unroll
        for (int e = 0; e < V; e++) y[e] = (float)u[e];
    }
    // f(value, element) for all of thread i's.
    template <typename F>
    __device__ __forceinline__ void each(int i, F f) const {
        for (int k = i; k < lines; k += kThreads) {
            float y[V];
            load_line(k, y);
#pragma unroll
            for (int e = 0; e < V; e++) f(y[e], head + k * V + e);
        }
        ends(i, f);
    }
    // Of the elements outside the lines.
    template <typename F>
    __device__ __forceinline__ void ends(int i, F f) const {
        if (before(i) >= 0) f((float)gptr(x)[before(i)], before(i));
        if (behind(i) >= 0) f((float)gptr(x)[behind(i)], behind(i));
    }
    // f(value, element) for all of the threads of this wave that `take`, the lanes sharing each one's lines, AT threads a
    // round trip to memory.
    template <typename F>
    __device__ __forceinline__ void each_of(bool take, F f) const {
        constexpr int AT = 4;
        const int lane = __lane_id(), first = threadIdx.x - lane;
        if (take) ends(threadIdx.x, f);
        uint64_t left = __builtin_amdgcn_ballot_w64(take);
        while (left) {
            int of[AT];
#pragma unroll
            for (int a = 0; a < AT; a++) {
                of[a] = left ? first + __builtin_ctzll(left) : -1;
                left &= left - 1;
            }
            for (int j = lane; j * kThreads < lines; j += 64) {
                float y[AT][V];
#pragma unroll
                for (int a = 0; a < AT; a++) load_line(max(of[a], 0) + j * kThreads, y[a]);
#pragma unroll
                for (int a = 0; a < AT; a++) {
                    const int k = of[a] + j * kThreads;
                    if (of[a] < 0 || k >= lines) continue;
#pragma unroll
                    for (int e = 0; e < V; e++) f(y[a][e], head + k * V + e);
                }
            }
        }
    }
};

// A token as a number that is larger the better it ranks: numbers before NaN, larger ones first (-0 as 0), then the lower
// index.
typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float x, int token) {
    const uint32_t u = __float_as_uint(x + 0.f), up = u >> 31 ? ~u : u | 0x80000000u;
    return (Key)(x != x ? 0u : up) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float value_of(Key k) {
    const uint32_t up = (uint32_t)(k >> 32);
    return up == 0 ? NAN : __uint_as_float(up >> 31 ? up & 0x7FFFFFFFu : ~up);
}
__device__ __forceinline__ int token_of(Key k) { return (int)~(uint32_t)k; }

struct Shared {
    float m[kWaves], s[kWaves], t[kWaves];
    float group[kGroups];
    Key key[kListed];
    Key best[kMostTop];
    Key next;
    float bound;
    int above, equal, last;
};

// The n-th largest of the groups' maxima; by one wave.
__device__ __forceinline__ float nth_largest(const Shared& sh, int n) {
    const float mine = sh.group[__lane_id()];
    int larger = 0;
#pragma unroll
    for (int i = 0; i < kGroups; i++)
        larger += __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), i)) > mine;
    return -wave_max(larger < n ? -mine : -INFINITY);  // (-inf only where that is a maximum)
}

// The first `need` elements of the slice, in order, for which f holds, into best from `at` on.  By one wave.
template <typename T, typename F>
__device__ __forceinline__ void fill(const Slice<T>& sl, Shared& sh, int at, int need, F f) {
    const int lane = __lane_id();
    int got = 0;
    for (int e0 = 0; e0 < sl.n && got < need; e0 += 64) {
        const int e = e0 + lane;
        const float x = e < sl.n ? (float)gptr(sl.x)[e] : 0.f;
        const bool take = e < sl.n && f(x);
        const uint64_t all = __builtin_amdgcn_ballot_w64(take);
        const int place = got + __builtin_popcountll(all & ((1ull << lane) - 1));
        if (take && place < need) sh.best[at + place] = key_of(x, sl.begin + e);
        got += __builtin_popcountll(all);
    }
}

// The n best of `count` candidates in LDS; the threads have met behind their writing.
__device__ __forceinline__ void rank_listed(Shared& sh, int first, int count, int at, int n) {
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const Key mine = sh.key[first + i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < count; j++) rank += sh.key[first + j] > mine;
        if (rank < n) sh.best[at + rank] = mine;
    }
}

// The n best of a slice into best, whoever reads them having met the others afterwards; sh.group holds the groups'
// maxima.  Places that the slice is too short for hold (NaN, INT32_MAX).
// `all`(f) calls f(value, element) for what the wave's threads that have something to offer hold.
template <typename T, typename All>
__device__ __forceinline__ void top_of_slice(const Slice<T>& sl, Shared& sh, int n, All all) {
    const int tid = threadIdx.x;
    if (tid < 64) {
        const float b = nth_largest(sh, n);
        if (tid == 0) {
            sh.bound = b;
            sh.above = sh.equal = 0;
        }
        if (tid < n) sh.best[tid] = key_of(NAN, INT32_MAX);
    }
    __syncthreads();
    const float bound = sh.bound;
    all([&](float x, int e) {
        if (x > bound) {
            const int i = atomicAdd(&sh.above, 1);
            if (i < kAbove) sh.key[i] = key_of(x, sl.begin + e);
        } else if (x == bound) {
            const int i = atomicAdd(&sh.equal, 1);
            if (i < kEqual) sh.key[kAbove + i] = key_of(x, sl.begin + e);
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
    Key last = ~(Key)0;
    for (int r = 0; r < n; r++) {
        if (tid == 0) sh.next = 0;
        __syncthreads();
        Key mine = 0;
        sl.each(tid, [&](float x, int e) {
            const Key k = key_of(x, sl.begin + e);
            if (k < last && k > mine) mine = k;
        });
        atomicMax(&sh.next, mine);
        __syncthreads();
        last = sh.next;
        if (tid == 0) sh.best[r] = last;
        __syncthreads();
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads, 8) void logprobs_kernel(LogprobsArgs p) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, row = blockIdx.x / p.splits, part = blockIdx.x - row * p.splits, n = p.top;
    const T* x = (const T*)p.logits + (int64_t)row * p.stride;
    const Slice<T> sl(x, min((int64_t)p.vocab, (int64_t)part * p.each), min((int64_t)p.vocab, (part + 1ll) * p.each));
    constexpr int U = 16 / Slice<T>::V, N = U * Slice<T>::V;

    Sums sum;
    auto add = [&](auto& y) {  // returns the largest
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
            sum.t = fmaf(e, fmaxf(d, kFarthest), sum.t);  // (a masked token adds 0)
        }
        return top;
    };
    float y[N];
    // the thread's groups of U lines with the largest values, and the largest of the others
    float top[3] = {-INFINITY, -INFINITY, -INFINITY};
    int at[2] = {tid, tid};
    for (int k = tid; k < sl.lines; k += U * kThreads) {
        sl.template load<U>(k, y);
        const float x = add(y);
        const bool first = x > top[0], second = x > top[1];
        top[2] = fmaxf(top[2], second ? top[1] : x);
        top[1] = first ? top[0] : second ? x : top[1];
        at[1] = first ? at[0] : second ? k : at[1];
        top[0] = first ? x : top[0];
        at[0] = first ? k : at[0];
    }
    if (sl.before(tid) >= 0 || sl.behind(tid) >= 0) {
        float z[2];
        z[0] = sl.before(tid) >= 0 ? (float)gptr(sl.x)[sl.before(tid)] : -INFINITY;
        z[1] = sl.behind(tid) >= 0 ? (float)gptr(sl.x)[sl.behind(tid)] : -INFINITY;
        add(z);
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
        top_of_slice(sl, sh, n, [&](auto f) {
            const float bound = sh.bound;
            auto offer = [&](int k) {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int line = k + i / Slice<T>::V * kThreads;
                    if (line < sl.lines) f(y[i], sl.head + line * Slice<T>::V + i % Slice<T>::V);
                }
            };
            if (sl.lines <= U * kThreads) {  // still in registers
                if (tid < sl.lines && mine >= bound) offer(tid);
                if (mine >= bound) sl.ends(tid, f);
                return;
            }
            const bool whole = top[2] >= bound;
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (!whole && top[i] >= bound && (i == 0 || at[1] != at[0])) {
                    sl.template load<U>(at[i], y);
                    offer(at[i]);
                }
            if (!whole && mine >= bound) sl.ends(tid, f);
            sl.each_of(whole, f);
        });
        __syncthreads();
    }
    if (p.splits > 1) {
        float* const at = p.parts + (int64_t)row * p.splits * kPart;
        float* const to = at + part * kPart;
        if (tid < n) put2(to + 4 + 2 * tid, __uint_as_float((uint32_t)sh.best[tid]), __uint_as_float((uint32_t)(sh.best[tid] >> 32)));
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
            sh.key[i] = (Key)__float_as_uint(y.y) << 32 | __float_as_uint(y.x);
        }
        __syncthreads();
        sum.m = sh.m[0];
        sum.s = sh.s[0];
        sum.t = sh.t[0];
        if (n) {
            // the parts' tokens are in order: a bound from the first ones of each
            if (tid < kGroups) {
                const int s = tid % p.splits, r = tid / p.splits;
                sh.group[tid] = r < n ? fmaxf(-INFINITY, value_of(sh.key[s * n + r])) : -INFINITY;
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
            Key mine[PER];
#pragma unroll
            for (int k = 0; k < PER; k++) {
                const int i = tid + k * kThreads;
                mine[k] = i < listed ? sh.key[i] : 0;
            }
            const float bound = sh.bound;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PER; k++)
                if (tid + k * kThreads < listed && (value_of(mine[k]) >= bound || bound == -INFINITY))
                    sh.key[atomicAdd(&sh.above, 1)] = mine[k];
            __syncthreads();
            rank_listed(sh, 0, sh.above, 0, n);
            __syncthreads();
        }
    }
    const float log_s = logf(sum.s);
    if (tid < n) {
        gptr(p.top_tokens)[(int64_t)row * n + tid] = token_of(sh.best[tid]);
        gptr(p.top_logprobs)[(int64_t)row * n + tid] = (value_of(sh.best[tid]) - sum.m) - log_s;
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
