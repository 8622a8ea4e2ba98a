// Causal grouped-query attention over a KV cache held in 4 bits (kv_q4.h).
//
// Query token t at position start + t sees positions 0..start + t; query head h
// reads KV head h / G, G = heads / kv_heads.  The (token, head of the group)
// pairs of a KV head are its query columns c = t G + g: 16 of them are the
// columns of the products S^T = K Q^T and O^T = V^T P^T, whose rows are keys
// and dims, so that a lane owns one column: its softmax needs two cross-lane
// moves, and its probabilities lie where the second product takes them.
#include "attn_parts.h"
#include "kv_q4.h"

#include <algorithm>

namespace {

// An f16 value times e, in one instruction (the product with 0 added, which no product of a
// number differs from but -0).  Not written as assembly: e comes from a matrix product or an
// exponential, whose waits the compiler places only before instructions that it knows.
__device__ __forceinline__ float times(f16 h, float e) { return fmaf((float)h, e, 0.f); }

// n - 8 of a word's nibbles 0 and 4 (low) or 1 and 5 (high), exactly: 1024 + n
// and 1024 + 16 n are f16 values with the nibble in their last bits.  The
// constants in registers (Nibbles(): a scalar and a vector one) let the mask and
// the bias be one instruction.
struct Nibbles {
    uint32_t low = 0x000F000Fu, high = 0x00F000F0u, bias = 0x64006400u;
    f16x2 sixteenth = {(f16)0.0625f, (f16)0.0625f};
    __device__ __forceinline__ Nibbles() {
        asm("" : "+s"(low));
        asm("" : "+s"(high));
        asm("" : "+v"(bias));
    }
    __device__ __forceinline__ f16x2 lo(uint32_t w) const {
        return pair((w & low) | bias) - (f16x2){(f16)1032.f, (f16)1032.f};
    }
    __device__ __forceinline__ f16x2 hi(uint32_t w) const {
        return __builtin_elementwise_fma(pair((w & high) | bias), sixteenth, (f16x2){(f16)-72.f, (f16)-72.f});
    }
};

struct SplitArgs {
    Q4Attention a;
    Q4Cache c;
    int G, splits;
    Divisor by_group, by_heads, by_splits, by_cus;
    float scale_log2;
};

// A tile's quants and scales as a lane holds them.
template <int NB>
struct Tile {
    uint32_t k[2][NB];    // keys: 16 tokens each
    uint2 ks[2][NB];      // their scales: 4 tokens
    uint2 v[NB];          // values: 8 tokens of a pair of dims
    uint2 vs[2][NB];
    __device__ __forceinline__ void load(const uint8_t* kt, const uint8_t* vt, int lane) {
        const int g = lane >> 4;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint32_t* kw = (const uint32_t*)(kt + (s * 64 + lane) * 4 * NB);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                k[s][b] = gptr(kw)[b];
                ks[s][b] = load2(kt + q4_scales_at(NB) + ((s * 4 + g) * NB + b) * 8);
                vs[s][b] = load2(vt + q4_scales_at(NB) + ((s * 4 + g) * NB + b) * 8);
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b++) v[b] = load2(vt + b * 512 + lane * 8);
    }
    static __device__ __forceinline__ uint2 load2(const uint8_t* p) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 x = *(const AS_GLOBAL u32x2*)p;
        return make_uint2(x[0], x[1]);
    }
};

// Where column `col` of KV head kvh leaves split 0 (then split by split).
template <int HD>
__device__ __forceinline__ float* partial(const SplitArgs& p, int kvh, int col) {
    const int t = p.by_group(col), h = kvh * p.G + col - t * p.G;
    return p.a.partials + ((int64_t)t * p.a.heads + h) * p.splits * (HD + 2);
}

// Called by the whole workgroup once its partial results of columns [col0, col0 + n) are
// written; `lds` is free.
template <int HD, typename T>
__device__ __forceinline__ void count_and_join(const SplitArgs& p, int kvh, int col0, int n, void* lds) {
    int* last = (int*)lds;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        int* counter = p.a.counters + blockIdx.x;
        *last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.splits - 1;
        if (*last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    const bool mine = *last;
    __syncthreads();  // (*last is read; the joining uses its place)
    if (!mine) return;
    auto put = [&](int col, int d, const Joined& j) {
        const int t = p.by_group(col), h = kvh * p.G + col - t * p.G;
        T* out = (T*)p.a.out + t * p.a.out_stride + (int64_t)h * HD + d;
        out[0] = (T)(j.a / j.l);
        out[1] = (T)(j.b / j.l);
    };
    const int items = n * (HD / 2);
    if (2 * items > (int)blockDim.x) {
        for (int i = threadIdx.x; i < items; i += blockDim.x) {
            const int col = col0 + i / (HD / 2), d = 2 * (i % (HD / 2));
            put(col, d, join<8>(partial<HD>(p, kvh, col), HD, d, 0, 1, p.splits));
        }
        return;
    }
    const int groups = blockDim.x / items, group = threadIdx.x / items, i = threadIdx.x - group * items;
    const int col = col0 + i / (HD / 2), d = 2 * (i % (HD / 2));
    const Joined j = join_groups<8>(partial<HD>(p, kvh, col), HD, d, group, groups, items, i, p.splits, (float4*)lds);
    if (group == 0) put(col, d, j);
}

// T float: the queries and probabilities as two f16 terms, the quants exact and the
// values exact in two terms.  A probability below 2^-17 of its row's largest loses bits
// (half of f16's smallest step is 2^-39 of that), which shows in an output 2^-15 the size
// of that key's value.  T f16: queries and keys exact, probabilities and values one f16
// term.
//
// A column's queries as the lane takes them, at q its dims 8 g of block 0: block b,
// dims 8 g + {0, 4, 1, 5, 2, 6, 3, 7} as the keys' nibbles come.  float: scaled into
// [-1, 1] by a power of two (`over` of the largest among the lane's rows), so that two f16
// terms hold any float32 range.  Returns what the products are to be scaled by for scores in
// base 2.
struct Same {
    __device__ __forceinline__ float operator()(float x) const { return x; }
};
template <int NB, typename T, typename Over = Same>
__device__ __forceinline__ float load_queries(const T* q, float scale_log2, f16x8 (&qh)[NB],
                                              f16x8 (&ql)[sizeof(T) == 4 ? NB : 1], Over over = Same()) {
    constexpr int at[8] = {0, 4, 1, 5, 2, 6, 3, 7};
    T x[NB][8];
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int e = 0; e < 8; e++) x[b][e] = q[32 * b + e];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) qh[b][e] = x[b][at[e]];
        return scale_log2;
    } else {
        float most = 0.f;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(x[b][e]));
        most = over(xor32_combine(xor16_combine(most, MaxOp()), MaxOp()));
        // (the bounds keep the scale itself, and a masked score's product with it, a number)
        const int ex = most > 0.f && most < INFINITY ? max(-100, min(__builtin_amdgcn_frexp_expf(most), 120)) : 0;
        const float down = ldexpf(1.f, -ex);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            f16x2 hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float u = x[b][at[2 * i]] * down, v = x[b][at[2 * i + 1]] * down;
                hi[i] = round2(u, v);
                lo[i] = round2(rest_low(hi[i], u), rest_high(hi[i], v));
            }
            qh[b] = frag(hi[0], hi[1], hi[2], hi[3]);
            ql[b] = frag(lo[0], lo[1], lo[2], lo[3]);
        }
        return ldexpf(scale_log2, ex);
    }
}
// A key's four scores of a block, in the units of the block's quants, added scaled.
__device__ __forceinline__ void add_scaled(f32x4& s, f32x4 part, uint2 d) {
    const f16x2 d0 = pair(d.x), d1 = pair(d.y);
    s[0] = fmaf((float)d0[0], part[0], s[0]);
    s[1] = fmaf((float)d0[1], part[1], s[1]);
    s[2] = fmaf((float)d1[0], part[2], s[2]);
    s[3] = fmaf((float)d1[1], part[3], s[3]);
}

// Up to kMostWaves waves a workgroup, each with key tiles of its own.
constexpr int kMostWaves = 8;
template <int NB>
constexpr int lds_bytes(int waves, int cols) {
    return waves * cols * (32 * NB + 4 + 2) * 4;
}
// Joins the waves' results of columns col0.., left in LDS: outputs xo[wave][column][dim], then
// (maximum, sum) xml[wave][2][column].  `tiles`: how many the waves shared.
template <int NB, int COLS, typename T>
__device__ __forceinline__ void join_waves(const SplitArgs& p, int kvh, int sp, int col0, int cols, int tiles,
                                           uint8_t* lds) {
    constexpr int HD = 32 * NB;
    const int waves = blockDim.x >> 6, G = p.G;
    float (*xo)[COLS][HD + 4] = (float (*)[COLS][HD + 4])lds;
    float (*xml)[2][COLS] = (float (*)[2][COLS])(lds + waves * COLS * (HD + 4) * 4);
    const int n = min(COLS, cols - col0), had = max(1, min(waves, tiles));  // (a wave without a tile adds nothing)
    for (int i = threadIdx.x; i < n * (HD / 2); i += blockDim.x) {
        const int qc = i / (HD / 2), d = 2 * (i % (HD / 2));
        float mt = xml[0][0][qc];
        for (int w = 1; w < had; w++) mt = fmaxf(mt, xml[w][0][qc]);
        float lt = 0.f, oa = 0.f, ob = 0.f;
        for (int w = 0; w < had; w++) {
            const float f = join_weight(xml[w][0][qc], mt);
            lt += f * xml[w][1][qc];
            oa += f * xo[w][qc][d];
            ob += f * xo[w][qc][d + 1];
        }
        if (p.splits == 1) {
            const int64_t tt = p.by_group(col0 + qc), hh = kvh * G + col0 + qc - tt * G;
            T* out = (T*)p.a.out + tt * p.a.out_stride + hh * HD + d;
            out[0] = (T)(oa / lt);
            out[1] = (T)(ob / lt);
        } else {
            float* pp = partial<HD>(p, kvh, col0 + qc) + sp * (HD + 2);
            put2(pp + 2 + d, oa, ob);
            if (d == 0) put2(pp, mt, lt);
        }
    }
    if (p.splits > 1) count_and_join<HD, T>(p, kvh, col0, n, lds);
}

template <int NB, int CT, typename T>
__global__ __launch_bounds__(64 * kMostWaves) void q4_attention_kernel(SplitArgs p) {
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int HD = 32 * NB, COLS = 16 * CT;
    extern __shared__ __align__(16) uint8_t lds[];
    const int waves = blockDim.x >> 6;
    float (*xo)[COLS][HD + 4] = (float (*)[COLS][HD + 4])lds;
    float (*xml)[2][COLS] = (float (*)[2][COLS])(lds + waves * COLS * (HD + 4) * 4);
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Nibbles nib;
    const int id = p.by_heads(blockIdx.x), kvh = blockIdx.x - id * p.c.kv_heads;
    const int sp = blockIdx.y, col0 = id * COLS;
    const int G = p.G, cols = p.a.tokens * G;
    const int start = p.a.start_dev ? *p.a.start_dev : p.a.start;
    const bool inside = start >= 0 && start <= p.c.capacity - p.a.tokens;
    // the tiles of this column group, and this split's share of them
    const int first_seen = start + p.by_group(col0), last_seen = start + p.by_group(min(col0 + COLS - 1, cols - 1));
    const int tiles = inside ? last_seen / kQ4Tile + 1 : 0;
    const int t0 = share(tiles, sp, p.by_splits), t1 = share(tiles, sp + 1, p.by_splits);

    const uint8_t* kt = p.c.k + (int64_t)kvh * q4_head_bytes(p.c.capacity, NB);
    const uint8_t* vt = p.c.v + (int64_t)kvh * q4_head_bytes(p.c.capacity, NB);
    constexpr int64_t B = q4_tile_bytes(NB);
    constexpr bool AHEAD = NB <= 4;  // the next tile on its way while one is worked on, where registers allow
    int j = t0 + wave;
    Tile<NB> xa, xb;
    auto load = [&](Tile<NB>& x, int tile) {
        const int64_t at = min(tile, t1 - 1) * B;  // (past the split's last tile: that one, unused)
        x.load(kt + at, vt + at, lane);
    };
    if (j < t1) load(xa, j);

    f16x8 qh[CT][NB], ql[CT][EXACT ? NB : 1];
    float sc[CT], m[CT];
    int seen[CT];  // a column's last position
    f32x4 o[CT][NB][2], l[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int col = min(col0 + 16 * ct + c16, cols - 1), t = p.by_group(col), h = kvh * G + col - t * G;
        seen[ct] = start + t;
        sc[ct] = load_queries<NB, T>((const T*)p.a.q + (int64_t)t * p.a.q_stride + (int64_t)h * HD + 8 * g, p.scale_log2,
                                     qh[ct], ql[ct]);
        m[ct] = -INFINITY;
        l[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NB; b++) o[ct][b][0] = o[ct][b][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const f16x2 one2 = {(f16)1.f, (f16)1.f};
    const f16x8 ones = frag(one2, one2, one2, one2);
    auto step = [&](Tile<NB>& x, int tile) {
        // S^T(key 16 s + 4 g + r, column c16)
        f32x4 sa[CT][2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++) sa[ct][s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t w = x.k[s][b], w8 = w >> 8;
                const f16x8 kf = frag(nib.lo(w), nib.hi(w), nib.lo(w8), nib.hi(w8));
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    f32x4 part = mfma(kf, qh[ct][b], f32x4{0.f, 0.f, 0.f, 0.f});
                    if constexpr (EXACT) part = mfma(kf, ql[ct][b], part);
                    add_scaled(sa[ct][s], part, x.ks[s][b]);
                }
            }
        }
        const int key0 = tile * kQ4Tile;
        if (key0 + kQ4Tile - 1 > first_seen) {
#pragma unroll
            for (int s = 0; s < 2; s++) {
                uint32_t keep[2] = {0u, 0u};
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int key = key0 + 16 * s + 4 * g + r;
#pragma unroll
                    for (int ct = 0; ct < CT; ct++)
                        if (key > seen[ct]) sa[ct][s][r] = -INFINITY;
                    if (key <= last_seen) keep[r >> 1] |= 0xFFFFu << (16 * (r & 1));
                }
                // positions that may never have been written: values of 0, since 0 times what lies there may be NaN
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    x.vs[s][b].x &= keep[0];
                    x.vs[s][b].y &= keep[1];
                }
            }
        }
        f16x8 pf[CT], pg[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            f32x4(&x)[2] = sa[ct];
            float mx = x[0][0];
#pragma unroll
            for (int i = 1; i < 8; i++) mx = fmaxf(mx, x[i >> 2][i & 3]);
            mx = xor32_combine(xor16_combine(mx, MaxOp()), MaxOp());
            const float mn = fmaxf(m[ct], mx * sc[ct]);  // (sc > 0)
            const float mref = mn == -INFINITY ? 0.f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m[ct] - mref), eref = exponent_base(x, mx, mref, sc[ct]);
            f16x2 ph[4], pl[EXACT ? 4 : 1];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float e0 = __builtin_amdgcn_exp2f(fmaf(x[i >> 1][2 * (i & 1)], sc[ct], eref));
                const float e1 = __builtin_amdgcn_exp2f(fmaf(x[i >> 1][2 * (i & 1) + 1], sc[ct], eref));
                ph[i] = round2(e0, e1);
                if constexpr (EXACT) pl[i] = round2(rest_low(ph[i], e0), rest_high(ph[i], e1));
            }
            if (__builtin_amdgcn_ballot_w64(m[ct] != mn)) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    o[ct][b][0] *= alpha;
                    o[ct][b][1] *= alpha;
                }
                l[ct] *= alpha;
                m[ct] = mn;
            }
            pf[ct] = frag(ph[0], ph[1], ph[2], ph[3]);
            l[ct] = mfma(ones, pf[ct], l[ct]);
            if constexpr (EXACT) {
                pg[ct] = frag(pl[0], pl[1], pl[2], pl[3]);
                l[ct] = mfma(ones, pg[ct], l[ct]);
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint32_t w0 = x.v[b].x, w1 = x.v[b].y;
            const f16x2 d[4] = {pair(x.vs[0][b].x), pair(x.vs[0][b].y), pair(x.vs[1][b].x), pair(x.vs[1][b].y)};
#pragma unroll
            for (int par = 0; par < 2; par++) {
                f16x2 n[4], hi[4], lo[4];
                n[0] = par ? nib.hi(w0) : nib.lo(w0);
                n[1] = par ? nib.hi(w0 >> 8) : nib.lo(w0 >> 8);
                n[2] = par ? nib.hi(w1) : nib.lo(w1);
                n[3] = par ? nib.hi(w1 >> 8) : nib.lo(w1 >> 8);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    hi[i] = n[i] * d[i];
                    // what the rounding left: 15 bits in all, exact
                    if constexpr (EXACT) lo[i] = __builtin_elementwise_fma(n[i], d[i], -hi[i]);
                }
                const f16x8 vh = frag(hi[0], hi[1], hi[2], hi[3]);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    f32x4& y = o[ct][b][par];
                    y = mfma(vh, pf[ct], y);
                    if constexpr (EXACT) {
                        y = mfma(vh, pg[ct], y);
                        y = mfma(frag(lo[0], lo[1], lo[2], lo[3]), pf[ct], y);
                    }
                }
            }
        }
    };
    if constexpr (AHEAD) {
        if (j + waves < t1) load(xb, j + waves);
        for (; j < t1; j += 2 * waves) {
            step(xa, j);
            if (j + waves >= t1) break;
            load(xa, j + 2 * waves);
            step(xb, j + waves);
            load(xb, j + 3 * waves);
        }
    } else {
        for (; j < t1; j += waves) {
            step(xa, j);
            load(xa, j + waves);
        }
    }

    // o[ct][b][par][r] = O(column 16 ct + c16, dim 32 b + 2 (4 g + r) + par)
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int c = 16 * ct + c16;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(float2*)&xo[wave][c][32 * b + 2 * (4 * g + r)] = make_float2(o[ct][b][0][r], o[ct][b][1][r]);
        if (g == 0) {
            xml[wave][0][c] = m[ct];
            xml[wave][1][c] = l[ct][0];
        }
    }
    __syncthreads();
    join_waves<NB, COLS, T>(p, kvh, sp, col0, cols, t1 - t0, lds);
}

// ------------------------------------------------------------------ few columns
// Single tokens: up to few_columns(NB) = CP query columns, and all blocks of the head in
// the 16 columns of a product.  Column CP b + c holds query c's block b, zeros standing
// for the other blocks, so that one accumulator takes all blocks' scores, a lane scales
// its own block's only, and a sum over the columns CP apart gives the score.  The
// values' scales go into the probabilities the same way (a column has one block's), so
// that values enter as n - 8, exactly, and of the products with each block's values a
// lane keeps its own block's.  Bound by the vector instructions, over half of them the
// unpacking, close to memory: 131,072 positions, 32/8 heads of 128, 31.8 to 36 us over
// cards in float32 (4.2 to 4.7 TB/s) and 29.0 to 31.0 in f16; on one card 35.7 and 31.0
// against 41.9 and 35 with a column a query, and 37.2 in float32 with three tiles ahead
// instead of two; 8,000 positions, 9/3 heads of 64, 8.2 us against 10.3.
// The probabilities times scales are held as P 2^14 d / 2^E, E kept as the maximum of
// the softmax is, so that the largest of the block's so far lies in [2^13, 2^15) and
// f16's smallest step is 2^-37 of it or less, whatever the scales of tokens that have no
// weight.  (E as the largest scale's exponent is known before the exponentials, but costs
// as much, within 1%, and with values of 1e-5 beside one of 6e4 at a weight of e^-60 it
// loses 6e-3 of a float32 output.)
constexpr int kLeastE = -80;  // a sum of weights over any cache stays a number
constexpr int few_columns(int nb) { return nb == 1 ? 16 : nb == 2 ? 8 : nb <= 4 ? 4 : 2; }

template <int N>
__device__ __forceinline__ float row_rotated(float x) {  // of 16 lanes
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 | N, 0xf, 0xf, true));
}
// Over the lanes of a row that are CP apart; the same bits in each.
template <int CP, typename Op>
__device__ __forceinline__ float over_slots(float x, Op op) {
    if constexpr (CP <= 8) x = op(x, row_rotated<8>(x));
    if constexpr (CP <= 4) x = op(x, row_rotated<4>(x));
    if constexpr (CP <= 2) x = op(x, row_rotated<2>(x));
    return x;
}

template <int NB>
struct FewTile {
    uint32_t k[2][NB];
    uint2 v[NB], ks[2], vs[2];  // (the scales: of the lane's own block)
    __device__ __forceinline__ void load(const uint8_t* kt, const uint8_t* vt, int lane, int scales_at) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const uint32_t* kw = (const uint32_t*)(kt + (s * 64 + lane) * 4 * NB);
#pragma unroll
            for (int b = 0; b < NB; b++) k[s][b] = gptr(kw)[b];
            ks[s] = Tile<NB>::load2(kt + scales_at + s * 32 * NB);
            vs[s] = Tile<NB>::load2(vt + scales_at + s * 32 * NB);
        }
#pragma unroll
        for (int b = 0; b < NB; b++) v[b] = Tile<NB>::load2(vt + b * 512 + lane * 8);
    }
};

template <int NB, typename T>
__global__ __launch_bounds__(64 * kMostWaves) void q4_attention_few_kernel(SplitArgs p) {
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int HD = 32 * NB, CP = few_columns(NB);
    extern __shared__ __align__(16) uint8_t lds[];
    const int waves = blockDim.x >> 6;
    const int lane = threadIdx.x & 63, g = lane >> 4, slot = (lane & 15) / CP, cc = lane % CP, own = min(slot, NB - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Nibbles nib;
    const int kvh = blockIdx.x, sp = blockIdx.y, G = p.G, cols = p.a.tokens * G;  // (at most CP)
    const int start = p.a.start_dev ? *p.a.start_dev : p.a.start;
    const bool inside = start >= 0 && start <= p.c.capacity - p.a.tokens;
    const int col = min(cc, cols - 1), t = p.by_group(col), h = kvh * G + col - t * G;
    const int seen = start + t, last_seen = start + p.a.tokens - 1;
    const int tiles = inside ? last_seen / kQ4Tile + 1 : 0;
    const int t0 = share(tiles, sp, p.by_splits), t1 = share(tiles, sp + 1, p.by_splits);

    const uint8_t* kt = p.c.k + (int64_t)kvh * q4_head_bytes(p.c.capacity, NB);
    const uint8_t* vt = p.c.v + (int64_t)kvh * q4_head_bytes(p.c.capacity, NB);
    const int scales_at = q4_scales_at(NB) + (g * NB + own) * 8;
    constexpr int AHEAD = 2;  // tiles on their way or at work
    FewTile<NB> x[AHEAD];
    auto load = [&](FewTile<NB>& y, int tile) {
        const int64_t at = min(tile, t1 - 1) * q4_tile_bytes(NB);  // (past the split's last tile: that one, unused)
        y.load(kt + at, vt + at, lane, scales_at);
    };
    int j = t0 + wave;
    if (j < t1)
#pragma unroll
        for (int i = 0; i < AHEAD - 1; i++) load(x[i], j + i * waves);

    f16x8 qh[NB], ql[EXACT ? NB : 1], mine[2][1];
    const float sc = load_queries<1, T>((const T*)p.a.q + (int64_t)t * p.a.q_stride + (int64_t)h * HD + 32 * own + 8 * g,
                                        p.scale_log2, mine[0], mine[1],
                                        [](float most) { return over_slots<CP>(most, MaxOp()); });
    const f16x8 zero = {};
#pragma unroll
    for (int b = 0; b < NB; b++) {
        qh[b] = slot == b ? mine[0][0] : zero;
        if constexpr (EXACT) ql[b] = slot == b ? mine[1][0] : zero;
    }

    float m = -INFINITY, l = 0.f;
    int E = 0;         // the exponent that P 2^14 d is held against,
    float peak = 0.f;  // and its largest when E was last chosen, in [2^13, 2^14); from 2^15 on E is chosen again
    f32x4 o[NB][2];
#pragma unroll
    for (int b = 0; b < NB; b++) o[b][0] = o[b][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto step = [&](FewTile<NB>& y, int tile) {
        f32x4 sa[2];
#pragma unroll
        for (int s = 0; s < 2; s++) sa[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const uint32_t w = y.k[s][b], w8 = w >> 8;
                const f16x8 kf = frag(nib.lo(w), nib.hi(w), nib.lo(w8), nib.hi(w8));
                sa[s] = mfma(kf, qh[b], sa[s]);
                if constexpr (EXACT) sa[s] = mfma(kf, ql[b], sa[s]);
            }
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const f16x2 d0 = pair(y.ks[s].x), d1 = pair(y.ks[s].y);
            sa[s] = f32x4{times(d0[0], sa[s][0]), times(d0[1], sa[s][1]), times(d1[0], sa[s][2]), times(d1[1], sa[s][3])};
#pragma unroll
            for (int r = 0; r < 4; r++) sa[s][r] = over_slots<CP>(sa[s][r], AddOp());
        }
        const int key0 = tile * kQ4Tile;
        if (key0 + kQ4Tile - 1 > start) {
#pragma unroll
            for (int s = 0; s < 2; s++) {
                uint32_t keep[2] = {0u, 0u};
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int key = key0 + 16 * s + 4 * g + r;
                    if (key > seen) sa[s][r] = -INFINITY;
                    if (key <= last_seen) keep[r >> 1] |= 0xFFFFu << (16 * (r & 1));
                }
                // positions that may never have been written: values of 0
                y.vs[s].x &= keep[0];
                y.vs[s].y &= keep[1];
            }
        }
        float mx = sa[0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) mx = fmaxf(mx, sa[i >> 2][i & 3]);
        mx = xor32_combine(xor16_combine(mx, MaxOp()), MaxOp());
        const float mn = fmaxf(m, mx * sc);
        const float mref = mn == -INFINITY ? 0.f : mn;
        const float eref = exponent_base(sa, mx, mref, sc) - (float)E;
        const uint32_t dv[4] = {y.vs[0].x, y.vs[0].y, y.vs[1].x, y.vs[1].y};
        float w[8], sum = 0.f, top = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float e = __builtin_amdgcn_exp2f(fmaf(sa[i >> 2][i & 3], sc, eref));
            sum += e;
            w[i] = times(pair(dv[i >> 1])[i & 1], e);
            top = fmaxf(top, fabsf(w[i]));  // (a NaN is not taken)
        }
        if (__builtin_amdgcn_ballot_w64(m != mn || top > 32768.f)) {
            const float down = __builtin_amdgcn_exp2f(m - mref);
            peak = fmaxf(peak * down, top);
            peak = xor32_combine(xor16_combine(peak, MaxOp()), MaxOp());
            const int by = peak > 0.f ? max(__builtin_amdgcn_frexp_expf(peak) - 14, kLeastE - E) : 0;
            const float f = ldexpf(1.f, -by), alpha = down * f;
            E += by;
            peak *= f;
            sum *= f;
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] *= f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                o[b][0] *= alpha;
                o[b][1] *= alpha;
            }
            l *= alpha;
            m = mn;
        }
        l += sum;
        f16x2 ph[4], pl[EXACT ? 4 : 1];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            ph[i] = round2(w[2 * i], w[2 * i + 1]);
            if constexpr (EXACT) pl[i] = round2(rest_low(ph[i], w[2 * i]), rest_high(ph[i], w[2 * i + 1]));
        }
        const f16x8 pf = frag(ph[0], ph[1], ph[2], ph[3]);
        f16x8 pg;
        if constexpr (EXACT) pg = frag(pl[0], pl[1], pl[2], pl[3]);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint32_t w0 = y.v[b].x, w1 = y.v[b].y, w08 = w0 >> 8, w18 = w1 >> 8;
            const f16x8 even = frag(nib.lo(w0), nib.lo(w08), nib.lo(w1), nib.lo(w18));
            const f16x8 odd = frag(nib.hi(w0), nib.hi(w08), nib.hi(w1), nib.hi(w18));
            o[b][0] = mfma(even, pf, o[b][0]);
            o[b][1] = mfma(odd, pf, o[b][1]);
            if constexpr (EXACT) {
                o[b][0] = mfma(even, pg, o[b][0]);
                o[b][1] = mfma(odd, pg, o[b][1]);
            }
        }
    };
    for (; j < t1; j += AHEAD * waves) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (j + i * waves >= t1) break;
            load(x[(i + AHEAD - 1) % AHEAD], j + (i + AHEAD - 1) * waves);
            step(x[i], j + i * waves);
        }
    }

    // o[own][par][r] = O(column cc, dim 32 own + 2 (4 g + r) + par) / 2^E
    float (*xo)[16][HD + 4] = (float (*)[16][HD + 4])lds;
    float (*xml)[2][16] = (float (*)[2][16])(lds + waves * 16 * (HD + 4) * 4);
    l = xor32_combine(xor16_combine(l, AddOp()), AddOp());
#pragma unroll
    for (int b = 1; b < NB; b++)
        if (slot == b) {
            o[0][0] = o[b][0];
            o[0][1] = o[b][1];
        }
    if (slot < NB) {
        const float up = ldexpf(1.f, E);
#pragma unroll
        for (int r = 0; r < 4; r++)
            *(float2*)&xo[wave][cc][32 * slot + 2 * (4 * g + r)] = make_float2(o[0][0][r] * up, o[0][1][r] * up);
        if (lane < CP) {
            xml[wave][0][cc] = m;
            xml[wave][1][cc] = l * up;
        }
    }
    __syncthreads();
    join_waves<NB, 16, T>(p, kvh, sp, 0, cols, t1 - t0, lds);
}

// ------------------------------------------------------------------ many columns
// A workgroup takes 64 CT query columns, 16 CT a wave; the tiles of keys and
// values are unpacked once for all its waves, into LDS as the fragments that the
// products read (16 bytes a lane in lane order, so no bank conflicts either
// way).  NSET (1, 2 or 4) sets of four waves take consecutive ranges of the keys and join
// through LDS at the end.  Two buffers a set: while the waves work on one, they
// unpack the next tile's words, loaded a step earlier, into the other; one
// barrier a step.
//
// The keys' fragments hold n - 8 and the products are scaled block by block, which keeps
// the keys exact; rounded to f16 in the fragments, d (n - 8) costs no vector instruction
// a score and is a fifth faster (2,048 f16 queries, 32/8 heads of 128: 54 us against 67),
// but doubles the error of the f16 outputs (4e-4 of the norm against 2.8e-4, of which
// the output's own rounding is 2e-4; queries of 3 times the keys' size).  The values'
// fragments hold d (n - 8), T f16 rounded to f16, T float with a second fragment of
// what the first one's rounding left.
template <int NB, int CT, int NSET, typename T>
struct Wide {
    static constexpr bool EXACT = sizeof(T) == 4;
    static constexpr int TPS = NB <= 4 && !EXACT ? 2 : 1;    // tiles a step
    static constexpr int KF = 2 * NB * TPS;                  // fragments of keys in a buffer,
    static constexpr int VT = EXACT ? 2 : 1;                 // and of values, in VT terms
    static constexpr int SCALES = (KF + KF * VT) * 1024;     // the keys' scales, a tile's as in the cache
    static constexpr int BUF = SCALES + TPS * 64 * NB;
    static constexpr int COLS = 64 * CT;
    static constexpr int JOIN = COLS * (32 * NB + 4) * 4 + COLS * 8;  // a set's outputs and statistics
    static constexpr int LDS = 2 * NSET * BUF > JOIN ? 2 * NSET * BUF : JOIN;
    static constexpr bool FITS = LDS <= 160 << 10;
};

template <int NB, int CT, int NSET, typename T>
__global__ __launch_bounds__(256 * NSET) __attribute__((amdgpu_waves_per_eu(NSET == 4 ? 4 : 2, NSET == 4 ? 4 : 2))) void q4_attention_wide_kernel(SplitArgs p) {
    typedef Wide<NB, CT, NSET, T> W;
    constexpr bool EXACT = W::EXACT;
    constexpr int TPS = W::TPS, HD = 32 * NB, STEP = TPS * kQ4Tile;
    constexpr int ITEMS = NB * TPS;  // (tile, block)
    constexpr int PER = (ITEMS + 3) / 4;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), set = wave / 4, wl = wave % 4;
    const int G = p.G, cols = p.a.tokens * G, groups = (cols + W::COLS - 1) / W::COLS;
    const Nibbles nib;
    // The longest (last) columns first.  One set: the chip holds two workgroups a CU and hands CU c
    // the workgroups c and c + CUs first, so every other CUs' worth comes in reverse, short beside long.
    int bx = blockIdx.x;
    if constexpr (NSET == 1) {
        const int cus = p.by_cus.d, from = p.by_cus(bx) * cus;
        if (p.by_cus(bx) & 1) bx = from + min(cus, (int)gridDim.x - from) - 1 - (bx - from);
    }
    const int id = p.by_heads(bx), kvh = bx - id * p.c.kv_heads;
    const int col0 = (groups - 1 - id) * W::COLS;
    const int start = p.a.start_dev ? *p.a.start_dev : p.a.start;
    const bool inside = start >= 0 && start <= p.c.capacity - p.a.tokens;
    const int wcol0 = col0 + wl * 16 * CT;  // the wave's columns
    const int last_seen = start + p.by_group(min(col0 + W::COLS - 1, cols - 1));
    const int w_first = start + p.by_group(min(wcol0, cols - 1));
    const int w_last = start + p.by_group(min(wcol0 + 16 * CT - 1, cols - 1));
    const int tiles = inside ? last_seen / kQ4Tile + 1 : 0;
    const int all = (tiles + TPS - 1) / TPS;  // steps over all the keys
    const int per = (all + NSET - 1) / NSET, f0 = set * per;  // this set's steps: [f0, f0 + count)
    const int count = max(0, min(all - f0, per));

    f16x8 q[CT][NB], ql[CT][EXACT ? NB : 1];
    int seen[CT];
    float sc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int col = min(wcol0 + 16 * ct + c16, cols - 1), t = p.by_group(col), h = kvh * G + col - t * G;
        seen[ct] = start + t;
        sc[ct] = load_queries<NB, T>((const T*)p.a.q + (int64_t)t * p.a.q_stride + (int64_t)h * HD + 8 * g, p.scale_log2,
                                     q[ct], ql[ct]);
    }
    float m[CT];
    f32x4 o[CT][NB][2], l[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        m[ct] = -INFINITY;
        l[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < NB; b++) o[ct][b][0] = o[ct][b][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const f16x2 one2 = {(f16)1.f, (f16)1.f};
    const f16x8 ones = frag(one2, one2, one2, one2);
    const uint8_t* kt = p.c.k + (int64_t)kvh * q4_head_bytes(p.c.capacity, NB);
    const uint8_t* vt = p.c.v + (int64_t)kvh * q4_head_bytes(p.c.capacity, NB);
    uint8_t* const buf0 = lds + set * 2 * W::BUF;

    // The set's four waves share the (tile, block) items of a step, of the keys and of the values.
    uint32_t rk[PER][4], rv[PER][6];
    const uint32_t k_at = lane * 4 * NB, ks_at = q4_scales_at(NB) + ((c16 >> 2) * NB * 4 + (c16 & 3)) * 2;
    const uint32_t v_at = lane * 8, vs_at = q4_scales_at(NB) + g * NB * 8;
    auto item = [&](int k, int* tt, int* b) {
        const int i = wl + 4 * k;
        *tt = i / NB;
        *b = i - *tt * NB;
        return ITEMS % 4 == 0 || i < ITEMS;
    };
    auto fetch = [&](int step) {
#pragma unroll
        for (int k = 0; k < PER; k++) {
            int tt, b;
            if (!item(k, &tt, &b)) continue;
            // past the last tile: that one again, its columns masked
            const int64_t at = (int64_t)min(step * TPS + tt, tiles - 1) * q4_tile_bytes(NB);
            const uint8_t *x = kt + at + b * 4, *y = vt + at + b * 512;
            const uint8_t *xs = kt + at + b * 8, *ys = vt + at + b * 8;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                rk[k][s] = *(const AS_GLOBAL uint32_t*)(x + (k_at + s * 256 * NB));
                rk[k][2 + s] = *(const AS_GLOBAL uint16_t*)(xs + (ks_at + s * 32 * NB));
                const uint2 d = Tile<NB>::load2(ys + (vs_at + s * 32 * NB));
                rv[k][2 + 2 * s] = d.x;
                rv[k][3 + 2 * s] = d.y;
            }
            const uint2 w = Tile<NB>::load2(y + v_at);
            rv[k][0] = w.x;
            rv[k][1] = w.y;
        }
    };
    auto unpack = [&](int step, uint8_t* buf) {
#pragma unroll
        for (int k = 0; k < PER; k++) {
            int tt, b;
            if (!item(k, &tt, &b)) continue;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const uint32_t w = rk[k][s], w8 = w >> 8;
                if (g == 0)
                    *(uint16_t*)(buf + W::SCALES + (((tt * 2 + s) * 4 + (c16 >> 2)) * NB + b) * 8 + (c16 & 3) * 2) =
                        (uint16_t)rk[k][2 + s];
                *(f16x8*)(buf + ((tt * 2 + s) * NB + b) * 1024 + lane * 16) =
                    frag(nib.lo(w), nib.hi(w), nib.lo(w8), nib.hi(w8));
            }
            const int key0 = (step * TPS + tt) * kQ4Tile;
            if (key0 + kQ4Tile - 1 > last_seen) {
                // positions that may never have been written: values of 0
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (key0 + 16 * (e >> 2) + 4 * g + (e & 3) > last_seen)
                        rv[k][2 + (e >> 1)] &= e & 1 ? 0xFFFFu : 0xFFFF0000u;
            }
            const uint32_t w[4] = {rv[k][0], rv[k][0] >> 8, rv[k][1], rv[k][1] >> 8};
            uint8_t* v = buf + (W::KF + (tt * NB + b) * 2 * W::VT) * 1024 + lane * 16;
#pragma unroll
            for (int par = 0; par < 2; par++) {
                f16x2 hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const f16x2 n = par ? nib.hi(w[i]) : nib.lo(w[i]), d = pair(rv[k][2 + i]);
                    hi[i] = n * d;
                    if constexpr (EXACT) lo[i] = __builtin_elementwise_fma(n, d, -hi[i]);
                }
                *(f16x8*)(v + par * W::VT * 1024) = frag(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (EXACT) *(f16x8*)(v + (par * W::VT + 1) * 1024) = frag(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    };
    auto work = [&](int step, const uint8_t* buf) {
        const int key0 = step * STEP;
        if (key0 > w_last) return;
        f32x4 sa[CT][TPS * 2];
        // fragments are read a group of NB ahead of the products that take them
        f16x8 fr[2][NB];
        auto read = [&](int group) {
#pragma unroll
            for (int b = 0; b < NB; b++) fr[group & 1][b] = *(const f16x8*)(buf + (group * NB + b) * 1024 + lane * 16);
        };
        read(0);
        // a group's products are scaled while the next group's run, where registers allow
        constexpr int LAG = NB <= 3 && !EXACT ? 1 : 0;
        // heads of 256: the first values only behind the softmax, ahead of which 39 registers spill
        // (4,000 queries of 16/8 heads: 287 us against 444)
        constexpr bool LATE = NB == 8;
        f32x4 part[2][CT][NB];
        uint2 d[2][NB];
        auto scale = [&](int u) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                sa[ct][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < NB; b++) add_scaled(sa[ct][u], part[u & 1][ct][b], d[u & 1][b]);
            }
        };
#pragma unroll
        for (int u = 0; u < 2 * TPS; u++) {
            if (!LATE || u + 1 < 2 * TPS) read(u + 1);  // (after the last keys: the first values)
#pragma unroll
            for (int b = 0; b < NB; b++) d[u & 1][b] = *(const uint2*)(buf + W::SCALES + ((u * 4 + g) * NB + b) * 8);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    part[u & 1][ct][b] = mfma(fr[u & 1][b], q[ct][b], f32x4{0.f, 0.f, 0.f, 0.f});
                    if constexpr (EXACT) part[u & 1][ct][b] = mfma(fr[u & 1][b], ql[ct][b], part[u & 1][ct][b]);
                }
            if (u >= LAG) scale(u - LAG);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (LAG) scale(2 * TPS - 1);
        if (key0 + STEP - 1 > w_first) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int u = 0; u < 2 * TPS; u++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (key0 + 16 * u + 4 * g + r > seen[ct]) sa[ct][u][r] = -INFINITY;
        }
        f16x8 pf[CT][TPS], pg[CT][EXACT ? TPS : 1];
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            float mx = sa[ct][0][0];
#pragma unroll
            for (int i = 1; i < 8 * TPS; i++) mx = fmaxf(mx, sa[ct][i >> 2][i & 3]);
            mx = xor32_combine(xor16_combine(mx, MaxOp()), MaxOp());
            const float mn = fmaxf(m[ct], mx * sc[ct]);
            const float mref = mn == -INFINITY ? 0.f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m[ct] - mref), eref = exponent_base(sa[ct], mx, mref, sc[ct]);
#pragma unroll
            for (int tt = 0; tt < TPS; tt++) {
                f16x2 e[4], r[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const f32x4& x = sa[ct][2 * tt + (i >> 1)];
                    const float a = __builtin_amdgcn_exp2f(fmaf(x[2 * (i & 1)], sc[ct], eref));
                    const float b = __builtin_amdgcn_exp2f(fmaf(x[2 * (i & 1) + 1], sc[ct], eref));
                    e[i] = round2(a, b);
                    if constexpr (EXACT) r[i] = round2(rest_low(e[i], a), rest_high(e[i], b));
                }
                pf[ct][tt] = frag(e[0], e[1], e[2], e[3]);
                if constexpr (EXACT) pg[ct][tt] = frag(r[0], r[1], r[2], r[3]);
            }
            if (__builtin_amdgcn_ballot_w64(m[ct] != mn)) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    o[ct][b][0] *= alpha;
                    o[ct][b][1] *= alpha;
                }
                l[ct] *= alpha;
                m[ct] = mn;
            }
#pragma unroll
            for (int tt = 0; tt < TPS; tt++) {
                l[ct] = mfma(ones, pf[ct][tt], l[ct]);
                if constexpr (EXACT) l[ct] = mfma(ones, pg[ct][tt], l[ct]);
            }
        }
        if (LATE) read(2 * TPS);
        constexpr int VG = 2 * TPS * W::VT;  // groups of the values' fragments: (tile, block, parity, term)
#pragma unroll
        for (int u = 0; u < VG; u++) {
            if (u + 1 < VG) read(2 * TPS + u + 1);
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const int at = u * NB + i, f = at / W::VT, tt = f / (2 * NB), d = f % (2 * NB);
                const f16x8 v = fr[(2 * TPS + u) & 1][i];
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    f32x4& x = o[ct][d >> 1][d & 1];
                    x = mfma(v, pf[ct][tt], x);
                    if constexpr (EXACT)
                        if (at % W::VT == 0) x = mfma(v, pg[ct][tt], x);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (tiles > 0) {  // (the same for the whole workgroup)
        const int lastf = all - 1;
        fetch(min(f0, lastf));
        unpack(min(f0, lastf), buf0);
        fetch(min(f0 + 1, lastf));
        __syncthreads();
        auto next = [&](int j) {
            if (j + 1 >= per) return;
            unpack(min(f0 + j + 1, lastf), buf0 + ((j + 1) & 1) * W::BUF);
            fetch(min(f0 + j + 2, lastf));
        };
        auto now = [&](int j) {
            if (j < count) work(f0 + j, buf0 + (j & 1) * W::BUF);
        };
        // Of two sets one unpacks while the other, on the same SIMDs, is at its products (2,048 float32
        // queries, 32/8 heads of 128: 103.6 us against 107.0, of f16 64.9 against 65.5; 4,000 of f16, 16/8
        // heads of 256: 288 against 298); of four sets it costs (37.4 against 38.9 so).
        if (NSET == 2 && set) {
            for (int j = 0; j < per; j++) {
                now(j);
                next(j);
                __syncthreads();
            }
        } else {
            for (int j = 0; j < per; j++) {
                next(j);
                now(j);
                __syncthreads();
            }
        }
    }
    // the other sets' results through LDS
    float* xo = (float*)lds;
    float* xml = xo + W::COLS * (HD + 4);
    auto put_set = [&]() {
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const int c = wl * 16 * CT + 16 * ct + c16;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float* x = xo + c * (HD + 4) + 32 * b + 8 * g;
                *(float4*)x = make_float4(o[ct][b][0][0], o[ct][b][1][0], o[ct][b][0][1], o[ct][b][1][1]);
                *(float4*)(x + 4) = make_float4(o[ct][b][0][2], o[ct][b][1][2], o[ct][b][0][3], o[ct][b][1][3]);
            }
            if (g == 0) {
                xml[2 * c] = m[ct];
                xml[2 * c + 1] = l[ct][0];
            }
        }
    };
    for (int s = 1; s < NSET; s++) {
        if (s > 1) __syncthreads();
        if (set == s) put_set();
        __syncthreads();
        if (set == 0) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const int c = wl * 16 * CT + 16 * ct + c16;
                const float mo = xml[2 * c], mn = fmaxf(m[ct], mo), fa = join_weight(m[ct], mn), fb = join_weight(mo, mn);
                m[ct] = mn;
                const float lo = xml[2 * c + 1];
#pragma unroll
                for (int r = 0; r < 4; r++) l[ct][r] = l[ct][r] * fa + lo * fb;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const float* x = xo + c * (HD + 4) + 32 * b + 8 * g;
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int par = 0; par < 2; par++)
                            o[ct][b][par][r] = o[ct][b][par][r] * fa + x[2 * r + par] * fb;
                }
            }
        }
    }
    if (set) return;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const int col = wcol0 + 16 * ct + c16;
        if (col >= cols) continue;
        const int t = p.by_group(col), h = kvh * G + col - t * G;
        T* out = (T*)p.a.out + t * p.a.out_stride + (int64_t)h * HD + 8 * g;
        const float inv = 1.0f / l[ct][0];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                out[32 * b + 2 * r] = (T)(o[ct][b][0][r] * inv);
                out[32 * b + 2 * r + 1] = (T)(o[ct][b][1][r] * inv);
            }
    }
}

// Whether workgroups of the many-column kernel may have one set of waves, and of 64 columns four, as
// LDS and registers allow.
constexpr bool one_set(int nb) { return nb <= 6; }
constexpr bool four_sets(int nb, bool exact) { return nb <= 2 && !exact; }

template <int NB, int CT, int NSET, typename T>
hipError_t launch_wide(const SplitArgs& p, int64_t cols, hipStream_t st) {
    typedef Wide<NB, CT, NSET, T> W;
    static_assert(W::FITS, "LDS");
    auto* kernel = q4_attention_wide_kernel<NB, CT, NSET, T>;
    static OncePerDevice once;
    if (hipError_t e = allow_whole_lds(once, (const void*)kernel)) return e;
    const dim3 grid((unsigned)((cols + W::COLS - 1) / W::COLS * p.c.kv_heads));
    kernel<<<grid, 256 * NSET, W::LDS, st>>>(p);
    return hipGetLastError();
}

template <auto* kernel, int NB, int COLS>
hipError_t launch_waves(const SplitArgs& p, const Q4Plan& plan, int64_t cols, hipStream_t st) {
    static OncePerDevice once;
    if (hipError_t e = allow_whole_lds(once, (const void*)kernel)) return e;
    const dim3 grid((unsigned)((cols + COLS - 1) / COLS * p.c.kv_heads), p.splits);
    kernel<<<grid, 64 * plan.waves, lds_bytes<NB>(plan.waves, COLS), st>>>(p);
    return hipGetLastError();
}

// Columns of a workgroup of the wide kernel at most, for nb blocks a head: as registers and LDS allow,
// and in float32, where its barriers cost small heads more than unpacking does (512 queries at 3,584
// positions, 32/32 heads of 64: 78 us against 65 with a wave's tiles its own), from head dimension 128.
constexpr int wide_columns(int nb, bool exact) {
    return exact ? (nb == 4 ? 128 : nb > 4 && nb <= 6 ? 64 : 16) : nb <= 4 ? 128 : 64;
}

template <int NB, typename T>
hipError_t launch_nb(const SplitArgs& p, const Q4Plan& plan, hipStream_t st) {
    const int64_t cols = (int64_t)p.a.tokens * p.G;
    constexpr int most = wide_columns(NB, sizeof(T) == 4);
    if constexpr (most >= 128)
        if (plan.cols == 128)
            return plan.waves == 4 ? launch_wide<NB, 2, 1, T>(p, cols, st) : launch_wide<NB, 2, 2, T>(p, cols, st);
    if constexpr (most >= 64)
        if (plan.cols == 64) {
            if constexpr (one_set(NB) && most == 64)
                if (plan.waves == 4) return launch_wide<NB, 1, 1, T>(p, cols, st);
            if constexpr (four_sets(NB, sizeof(T) == 4))
                if (plan.waves == 16) return launch_wide<NB, 1, 4, T>(p, cols, st);
            return launch_wide<NB, 1, 2, T>(p, cols, st);
        }
    if constexpr (NB <= 3 && sizeof(T) == 4)
        if (plan.cols == 32) return launch_waves<q4_attention_kernel<NB, 2, T>, NB, 32>(p, plan, cols, st);
    if (cols <= few_columns(NB)) return launch_waves<q4_attention_few_kernel<NB, T>, NB, 16>(p, plan, cols, st);
    return launch_waves<q4_attention_kernel<NB, 1, T>, NB, 16>(p, plan, cols, st);
}

template <typename T>
hipError_t launch(const SplitArgs& p, const Q4Plan& plan, hipStream_t st) {
    switch (p.c.nb) {
    case 1: return launch_nb<1, T>(p, plan, st);
    case 2: return launch_nb<2, T>(p, plan, st);
    case 3: return launch_nb<3, T>(p, plan, st);
    case 4: return launch_nb<4, T>(p, plan, st);
    case 5: return launch_nb<5, T>(p, plan, st);
    case 6: return launch_nb<6, T>(p, plan, st);
    case 7: return launch_nb<7, T>(p, plan, st);
    default: return launch_nb<8, T>(p, plan, st);
    }
}

}  // namespace

// How a call runs.  Columns of a workgroup: 16 or 32 (every wave key tiles of its own)
// until workgroups of 64 fill the chip (half of it, f16 heads of 96 and 128), 64 or 128
// from there, where unpacking a tile once for all of them pays, us with 64 or 128 and 16:
// f16, 32/32 heads of 64, 512 queries at 3,584 37.9 and 49.7, 300 at 1,000 16.7 and 15.9;
// 32/8 heads of 128, 512 queries 13.5 and 18.4, 300 10.7 and 12.5, 100 7.0 and 6.0; 16/8
// heads of 192, 400 queries 16.1 and 13.3; float32, 32/8 heads of 128, 2,048 queries 105
// and 143, 1,024 37.5 and 49, 512 18.8 and 20.9.
//
// Splits, up to a workgroup a CU over all.  A workgroup alone costs about 4 us and
// nb / 18 us a tile of its keys; joining costs 1.5 us (4 with 16 full columns).  A split
// has a tile a wave until there are 16 splits (one token at 4,000, 32/8 heads of 128: 9.3
// us in 8 and in 16, 11.5 in 32; at 8,000, 9/3 heads of 64: 9.6 in 8, 7.7 in 16, 9.2 in 48;
// 37 at 1,021, 15/5 heads of 64: 8.5 in one, 8.0 in 7), then 32 tiles, which hide the
// waits of 32 splits and more, or 16 of more than 4 blocks (4/2 heads of 256, 30,000
// positions: 15.4 us in 64, 17.5 in 32).
// Two or three splits pay over long caches only (64 queries of 32/8 heads of 128 at
// 1,000: 13.9 in two, 13.5 in one; 37 of 15/5 heads of 64 at 8,000: 22.6 and 34.6).
Q4Plan q4_attention_plan(bool f16_rows, int tokens, int heads, int kv_heads, int hd, int length) {
    Q4Plan r;
    const int64_t cols = (int64_t)tokens * (heads / kv_heads);
    if (cols <= 0) return r;  // (nothing runs)
    const int cus = device_cus(), nb = hd / 32, tiles = q4_tiles(length), work = tiles * nb;
    auto groups = [&](int tile) { return (cols + tile - 1) / tile * kv_heads; };
    auto up = [](int64_t a, int64_t b) { return (int)((a + b - 1) / b); };
    const int wide = wide_columns(nb, !f16_rows);
    if (cols > 64 && wide > 16 && groups(64) >= (f16_rows && (nb == 3 || nb == 4) ? cus / 2 : cus)) {
        // 128 columns where workgroups of 128 fill the chip and the longest does not outlast a CU's
        // share of the work by half (the columns see `length` positions at most, half of their tokens
        // fewer on average): f16, 32/8 heads of 128, us with 128 and 64: 2,048 queries 67 and 87, 1,500
        // 44.7 and 56.0, 1,024 at 1,000 57 and 61, 1,024 32.6 and 27.9; 4,096 of 9/3 heads of 64 66.6
        // and 55.7.
        const int64_t seen = length - tokens / 2;
        const bool even = 2 * 128 * cus * (int64_t)length <= 3 * cols * kv_heads * seen;
        r.cols = wide == 128 && groups(128) >= cus && even ? 128 : 64;
        // One set of waves, two workgroups a CU, which do not wait for each other, at the greatest
        // width where enough of the columns keep the last CU's second one at work (f16, 32/8 heads of
        // 128, us with one and two sets: 8,192 queries 691 and 842, 4,000 189 and 225, 2,400 84 and 100,
        // 2,048 71 and 67; float32: 3,000 182 and 222).  Four sets of 64 columns where each has many
        // steps (32/32 heads of 64: 512 queries at 3,584 37.9 us against 45.6; 300 at 300 of 9/3 heads
        // 10.8 against 9.9).
        if (one_set(nb) && r.cols == wide && 8 * groups(r.cols) * seen >= 9 * cus * (int64_t)length) r.waves = 4;
        else r.waves = r.cols == 64 && four_sets(nb, !f16_rows) && seen / kQ4Tile >= 48 ? 16 : 8;
        return r;
    }
    // 32 a workgroup, its waves unpacking a tile for both halves, where they are four times the CUs:
    // 4,000 float32 queries of 15/5 heads of 64 108 us against 122, 2,048 40.1 against 41.1, 777 14.7
    // against 12.4; at most 3 blocks a head (registers).
    r.cols = !f16_rows && nb <= 3 && groups(32) >= 4 * cus ? 32 : 16;
    const int most = groups(r.cols) <= kQ4Counters ? std::max(1, (int)(cus / groups(r.cols))) : 1;
    r.splits = work <= 40 ? 1 : std::min(most, std::max(std::min(16, up(tiles, 4)), up(tiles, nb > 4 ? 16 : 32)));
    if (r.splits < 4 && work <= 200) r.splits = 1;
    // Eight waves where each still has many tiles (131,072 positions in 32 splits: 33.1 us against
    // 36.6 with four, one card; 1,000 in 8: 7.4 against 6.9) and the chip is not full without them (512
    // float32 queries, 32/8 heads of 128, in this kernel: 31.9 against 23.1), or for the threads that
    // join (16 queries of 32/8 heads of 128 at 4,000 in 8 splits: 14.2 against 15.8).
    const int64_t here = groups(r.cols) * r.splits;
    r.waves = (up(tiles, r.splits) >= 16 && here <= cus) || (r.splits > 1 && cols * (hd / 2) > 256) ? 8 : 4;
    return r;
}

int64_t q4_attention_workspace(int tokens, int heads, int hd, const Q4Plan& plan) {
    return plan.splits > 1 ? kQ4Counters * 4 + (int64_t)tokens * heads * plan.splits * (hd + 2) * 4 : 0;
}

void q4_set_workspace(Q4Attention& a, void* workspace) {
    a.counters = (int*)workspace;
    a.partials = (float*)((uint8_t*)workspace + kQ4Counters * 4);
}

hipError_t launch_q4_attention(bool f16_rows, const Q4Attention& a, const Q4Cache& c, const Q4Plan& plan,
                               hipStream_t st) {
    if (a.tokens <= 0) return hipSuccess;
    SplitArgs p;
    p.a = a;
    p.c = c;
    p.G = a.heads / c.kv_heads;
    p.splits = plan.splits;
    p.by_group = Divisor(p.G);
    p.by_heads = Divisor(c.kv_heads);
    p.by_splits = Divisor(plan.splits);
    p.by_cus = Divisor(device_cus());
    p.scale_log2 = 1.4426950408889634f / sqrtf(32.f * c.nb);
    return f16_rows ? launch<f16>(p, plan, st) : launch<float>(p, plan, st);
}
