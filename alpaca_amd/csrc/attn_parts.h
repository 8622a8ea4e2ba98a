// What the attention kernels over caches of their own layout share: pairs and
// second terms of f16, a division by a number that the host knows, and the joining of
// the results of key ranges.
#pragma once

#include "common.h"

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2P = 14.f;   // P enters the products as P 2^14: what is far below the largest stays above f16's subnormals

__device__ __forceinline__ uint32_t bits(f16x2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ f16x2 pair(uint32_t u) { return __builtin_bit_cast(f16x2, u); }
__device__ __forceinline__ f16x2 round2(float a, float b) { return __builtin_convertvector((f32x2){a, b}, f16x2); }
// e minus the low (high) half of a pair, in one instruction; exact where the half is e rounded.
__device__ __forceinline__ float rest_low(f16x2 h, float e) {
    float d;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(bits(h)), "v"(e));
    return d;
}
__device__ __forceinline__ float rest_high(f16x2 h, float e) {
    float d;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(bits(h)), "v"(e));
    return d;
}
__device__ __forceinline__ f16x8 frag(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Division of 0 <= n < 2^31 by a divisor that the host knows: with 2^s >= d,
// m = floor(2^(31 + s) / d) + 1 has m d = 2^(31 + s) + e, 0 < e <= d <= 2^s, so
// n m / 2^(31 + s) exceeds n / d by less than n / 2^31 / d < 1 / d and has its floor.
struct Divisor {
    unsigned d = 1, m = 0, s = 0;
    Divisor() = default;
    explicit Divisor(unsigned v) : d(v) {
        while ((1u << s) < d) s++;
        m = (unsigned)((1ull << (31 + s)) / d + 1);  // (d = 1: 2^31 + 1)
    }
    __device__ __forceinline__ int operator()(int n) const { return (int)(__umulhi((unsigned)n << 1, m) >> s); }
};

// Part i of `parts` of n: [share(n, i, parts), share(n, i + 1, parts)).
__device__ __forceinline__ int share(int n, int i, const Divisor& parts) {
    const int q = parts(n);
    return q * i + min(i, n - q * (int)parts.d);
}

// ------------------------------------------------------------------ joining the splits
// A split leaves (maximum, sum, unnormalised output) of its columns in the
// workspace, and the last workgroup of a group of columns to arrive joins them in the
// same launch, 3 us of GPU time and as much on the host less than a second one.  The
// partial results are written and read with agent-scope accesses, which the L2 caches
// of all XCDs see; each thread waits for its own to be acknowledged before the count,
// and the last sets the counter back to zero for the next call.
struct Joined {
    float m = -INFINITY, l = 0.f, a = 0.f, b = 0.f;
};
// (top is the larger: a maximum that no score has reached weighs 1 where no other
// has either, so that a NaN is not lost)
__device__ __forceinline__ float join_weight(float m, float top) { return m == top ? 1.f : __builtin_amdgcn_exp2f(m - top); }
__device__ __forceinline__ void join_add(Joined& j, float m, float l, float a, float b) {
    const float top = fmaxf(j.m, m), f = join_weight(j.m, top), w = join_weight(m, top);
    j.m = top;
    j.l = j.l * f + l * w;
    j.a = j.a * f + a * w;
    j.b = j.b * f + b * w;
}
// Two floats past the caches of an XCD, and back.
__device__ __forceinline__ void put2(float* p, float a, float b) {
    const uint64_t u = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    __hip_atomic_store(gptr((uint64_t*)p), u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get2(const float* p) {
    const uint64_t u = __hip_atomic_load(gptr((const uint64_t*)p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)u), __uint_as_float((uint32_t)(u >> 32)));
}
// Splits first, first + step, ... < splits of the row at pp, for dims d and d + 1;
// J of them in a round trip to memory.
template <int J>
__device__ __forceinline__ Joined join(const float* pp, int hd, int d, int first, int step, int splits) {
    Joined j;
    for (int s0 = first; s0 < splits; s0 += J * step) {
        float2 ml[J], o[J];
#pragma unroll
        for (int i = 0; i < J; i++) {  // (past the last: that one again, unused)
            const float* x = pp + (int64_t)min(s0 + i * step, splits - 1) * (hd + 2);
            ml[i] = get2(x);
            o[i] = get2(x + 2 + d);
        }
        float top = j.m;
#pragma unroll
        for (int i = 0; i < J; i++)
            if (s0 + i * step < splits) top = fmaxf(top, ml[i].x);
        const float f = join_weight(j.m, top);
        j.l *= f;
        j.a *= f;
        j.b *= f;
#pragma unroll
        for (int i = 0; i < J; i++) {
            if (s0 + i * step >= splits) continue;
            const float w = join_weight(ml[i].x, top);
            j.l += w * ml[i].y;
            j.a += w * o[i].x;
            j.b += w * o[i].y;
        }
        j.m = top;
    }
    return j;
}
// Groups of threads with every groups-th split each, met in LDS (a float4 a thread):
// item i of `items` in thread i of each group; the result is group 0's.
template <int J>
__device__ __forceinline__ Joined join_groups(const float* pp, int hd, int d, int group, int groups, int items, int i,
                                              int splits, float4* js) {
    Joined j;
    if (group < groups) j = join<J>(pp, hd, d, group, groups, splits);
    js[threadIdx.x] = make_float4(j.m, j.l, j.a, j.b);
    __syncthreads();
    if (group == 0)
        for (int g = 1; g < groups; g++) {
            const float4 o = js[i + g * items];
            join_add(j, o.x, o.y, o.z, o.w);
        }
    return j;
}

// What comes off the exponents of a step: kLog2P - mref, mref the maximum so far in base 2
// (0 for none), mx the step's own largest score.  A maximum is the rounded product of a
// score with `sc`, and x sc - mref, rounded once, keeps what that rounding left: the same
// for every key, so that it cancels, but past kLargeScore it would take P out of f16's
// range.  From there on the scores are taken from the step's largest first, exactly 0 for
// that one, and only the maxima are rounded.  (log2p: what P is scaled by, if not kLog2P.)
constexpr float kLargeScore = 8388608.f;  // 2^23: half a step is 2^-1
template <int N, typename V>
__device__ __forceinline__ float exponent_base(V (&x)[N], float mx, float mref, float sc, float log2p = kLog2P) {
#pragma clang fp contract(off)
    float base = log2p - mref;
    const bool large = fabsf(mref) > kLargeScore;
    if (__builtin_amdgcn_ballot_w64(large)) {
        const float top = large && mx != -INFINITY ? mx : 0.f;  // (a step of masked keys: 0)
#pragma unroll
        for (int i = 0; i < N; i++) x[i] -= top;
        if (large) base = log2p + (top * sc - mref);
    }
    return base;
}
