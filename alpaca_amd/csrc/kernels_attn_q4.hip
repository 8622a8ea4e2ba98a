// Causal grouped-query attention over a KV cache held in 4 bits (kv_q4.h).
//
// Query token t at position start + t sees positions 0..start + t; query head h
// reads KV head h / G, G = heads / kv_heads.  The (token, head of the group)
// pairs of a KV head are its query columns c = t G + g: 16 of them are the
// columns of the products S^T = K Q^T and O^T = V^T P^T, whose rows are keys
// and dims, so that a lane owns one column: its softmax needs two cross-lane
// moves, and its probabilities lie where the second product takes them.
#include "kv_q4.h"

#include <algorithm>

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;        // of a workgroup, each with key tiles of its own
constexpr float kLog2P = 14.f;   // P enters the products as P 2^14: what is far below the largest stays above f16's subnormals

__device__ __forceinline__ uint32_t bits(f16x2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ f16x2 pair(uint32_t u) { return __builtin_bit_cast(f16x2, u); }
__device__ __forceinline__ f16x2 round2(float a, float b) { return __builtin_convertvector((f32x2){a, b}, f16x2); }
__device__ __forceinline__ f16x8 frag(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
    return {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// n - 8 of a word's nibbles 0 and 4 (low) or 1 and 5 (high), exactly: 1024 + n
// and 1024 + 16 n are f16 values with the nibble in their last bits.
__device__ __forceinline__ f16x2 low_pair(uint32_t w) {
    return pair((w & 0x000F000Fu) | 0x64006400u) - (f16x2){(f16)1032.f, (f16)1032.f};
}
__device__ __forceinline__ f16x2 high_pair(uint32_t w) {
    const f16x2 x = pair((w & 0x00F000F0u) | 0x64006400u);
    return __builtin_elementwise_fma(x, (f16x2){(f16)0.0625f, (f16)0.0625f}, (f16x2){(f16)-72.f, (f16)-72.f});
}

struct SplitArgs {
    Q4Attention a;
    Q4Cache c;
    int G, splits;
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

// T float: the scores and outputs to float32 accuracy (the queries and
// probabilities as two f16 terms, the quants exact and the values exact in two
// terms).  T f16: queries exact, probabilities and values one f16 term.
template <int NB, typename T>
__global__ __launch_bounds__(64 * kWaves, 2) void q4_attention_kernel(SplitArgs p) {
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int HD = 32 * NB;
    __shared__ float xo[kWaves][16][HD + 4];
    __shared__ float xml[kWaves][2][16];
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sp = blockIdx.x % p.splits, kvh = blockIdx.y, col0 = blockIdx.x / p.splits * 16;
    const int G = p.G, cols = p.a.tokens * G;
    const int start = p.a.start_dev ? *p.a.start_dev : p.a.start;
    const bool inside = start >= 0 && start <= p.c.capacity - p.a.tokens;
    const int col = min(col0 + c16, cols - 1), t = col / G, h = kvh * G + col - t * G;
    const int seen = start + t;  // the column's last position
    // the tiles of this column group, and this split's share of them
    const int first_seen = start + col0 / G, last_seen = start + min(col0 + 15, cols - 1) / G;
    const int tiles = inside ? last_seen / kQ4Tile + 1 : 0;
    const int t0 = (int)((int64_t)tiles * sp / p.splits), t1 = (int)((int64_t)tiles * (sp + 1) / p.splits);

    // queries: block b, dims 8 g + {0, 4, 1, 5, 2, 6, 3, 7} as the keys' nibbles come
    f16x8 qh[NB], ql[EXACT ? NB : 1];
    float sc = p.scale_log2;
    {
        const T* q = (const T*)p.a.q + (int64_t)t * p.a.q_stride + (int64_t)h * HD + 8 * g;
        T x[NB][8];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[b][e] = q[32 * b + e];
        constexpr int at[8] = {0, 4, 1, 5, 2, 6, 3, 7};
        if constexpr (EXACT) {
            // the column scaled into [-1, 1] by a power of two, so that its two terms hold any float32 range
            float most = 0.f;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(x[b][e]));
            most = xor32_combine(xor16_combine(most, MaxOp()), MaxOp());
            // (the bounds keep the scale itself, and a masked score's product with it, a number)
            const int ex = most > 0.f && most < INFINITY ? max(-100, min(__builtin_amdgcn_frexp_expf(most), 120)) : 0;
            sc = ldexpf(sc, ex);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float v = ldexpf(x[b][at[e]], -ex);
                    qh[b][e] = (f16)v;
                    ql[b][e] = (f16)(v - (float)qh[b][e]);
                }
        } else {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 8; e++) qh[b][e] = x[b][at[e]];
        }
    }

    float m = -INFINITY;
    f32x4 o[NB][2], l = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NB; b++) o[b][0] = o[b][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    const f16x2 one2 = {(f16)1.f, (f16)1.f};
    const f16x8 ones = frag(one2, one2, one2, one2);
    const uint8_t* kt = p.c.k + (int64_t)kvh * q4_head_bytes(p.c.capacity, NB);
    const uint8_t* vt = p.c.v + (int64_t)kvh * q4_head_bytes(p.c.capacity, NB);

    auto step = [&](Tile<NB>& x, int tile) {
        // S^T(key 16 s + 4 g + r, column c16)
        f32x4 sa[2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
            sa[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint32_t w = x.k[s][b], w8 = w >> 8;
                const f16x8 kf = frag(low_pair(w), high_pair(w), low_pair(w8), high_pair(w8));
                f32x4 part = mfma(kf, qh[b], f32x4{0.f, 0.f, 0.f, 0.f});
                if constexpr (EXACT) part = mfma(kf, ql[b], part);
                const f16x2 d0 = pair(x.ks[s][b].x), d1 = pair(x.ks[s][b].y);
                sa[s][0] = fmaf((float)d0[0], part[0], sa[s][0]);
                sa[s][1] = fmaf((float)d0[1], part[1], sa[s][1]);
                sa[s][2] = fmaf((float)d1[0], part[2], sa[s][2]);
                sa[s][3] = fmaf((float)d1[1], part[3], sa[s][3]);
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
                    if (key > seen) sa[s][r] = -INFINITY;
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
        float mx = sa[0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) mx = fmaxf(mx, sa[i >> 2][i & 3]);
        mx = xor32_combine(xor16_combine(mx, MaxOp()), MaxOp());
        const float mn = fmaxf(m, mx * sc);  // (sc > 0)
        const float mref = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - mref), eref = kLog2P - mref;
        f16x2 ph[4], pl[EXACT ? 4 : 1];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float e0 = __builtin_amdgcn_exp2f(fmaf(sa[i >> 1][2 * (i & 1)], sc, eref));
            const float e1 = __builtin_amdgcn_exp2f(fmaf(sa[i >> 1][2 * (i & 1) + 1], sc, eref));
            ph[i] = round2(e0, e1);
            if constexpr (EXACT) pl[i] = round2(e0 - (float)ph[i][0], e1 - (float)ph[i][1]);
        }
        if (__builtin_amdgcn_ballot_w64(m != mn)) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                o[b][0] *= alpha;
                o[b][1] *= alpha;
            }
            l *= alpha;
            m = mn;
        }
        const f16x8 pf = frag(ph[0], ph[1], ph[2], ph[3]);
        f16x8 pg;
        l = mfma(ones, pf, l);
        if constexpr (EXACT) {
            pg = frag(pl[0], pl[1], pl[2], pl[3]);
            l = mfma(ones, pg, l);
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const uint32_t w0 = x.v[b].x, w1 = x.v[b].y;
            const f16x2 d[4] = {pair(x.vs[0][b].x), pair(x.vs[0][b].y), pair(x.vs[1][b].x), pair(x.vs[1][b].y)};
#pragma unroll
            for (int par = 0; par < 2; par++) {
                f16x2 n[4], hi[4], lo[4];
                n[0] = par ? high_pair(w0) : low_pair(w0);
                n[1] = par ? high_pair(w0 >> 8) : low_pair(w0 >> 8);
                n[2] = par ? high_pair(w1) : low_pair(w1);
                n[3] = par ? high_pair(w1 >> 8) : low_pair(w1 >> 8);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    hi[i] = n[i] * d[i];
                    // what the rounding left: 15 bits in all, exact
                    if constexpr (EXACT) lo[i] = __builtin_elementwise_fma(n[i], d[i], -hi[i]);
                }
                const f16x8 vh = frag(hi[0], hi[1], hi[2], hi[3]);
                o[b][par] = mfma(vh, pf, o[b][par]);
                if constexpr (EXACT) {
                    o[b][par] = mfma(vh, pg, o[b][par]);
                    o[b][par] = mfma(frag(lo[0], lo[1], lo[2], lo[3]), pf, o[b][par]);
                }
            }
        }
    };
    {
        constexpr int64_t B = q4_tile_bytes(NB);
        Tile<NB> x;
        int j = t0 + wave;
        if (j < t1) x.load(kt + j * B, vt + j * B, lane);
        for (; j < t1; j += kWaves) {
            if constexpr (NB <= 4) {
                // the next tile on its way while this one is worked on
                Tile<NB> y = x;
                const int nx = min(j + kWaves, t1 - 1);
                x.load(kt + nx * B, vt + nx * B, lane);
                step(y, j);
            } else {
                step(x, j);
                if (j + kWaves < t1) x.load(kt + (j + kWaves) * B, vt + (j + kWaves) * B, lane);
            }
        }
    }

    // o[b][par][r] = O(column c16, dim 32 b + 2 (4 g + r) + par)
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            *(float2*)&xo[wave][c16][32 * b + 2 * (4 * g + r)] = make_float2(o[b][0][r], o[b][1][r]);
    if (g == 0) {
        xml[wave][0][c16] = m;
        xml[wave][1][c16] = l[0];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * HD; i += 64 * kWaves) {
        const int qc = i / HD, d = i % HD;
        if (col0 + qc >= cols) break;
        const int tt = (col0 + qc) / G;
        const int64_t hh = kvh * G + col0 + qc - tt * G;
        float mt = xml[0][0][qc];
#pragma unroll
        for (int w = 1; w < kWaves; w++) mt = fmaxf(mt, xml[w][0][qc]);
        float lt = 0.f, ot = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            const float mw = xml[w][0][qc];
            const float f = mw == -INFINITY ? (mt == -INFINITY ? 1.f : 0.f) : exp2f(mw - mt);
            lt += f * xml[w][1][qc];
            ot += f * xo[w][qc][d];
        }
        if (p.splits == 1) {
            ((T*)p.a.out)[tt * p.a.out_stride + hh * HD + d] = (T)(ot / lt);
        } else {
            float* pp = p.a.partials + ((tt * (int64_t)p.a.heads + hh) * p.splits + sp) * (HD + 2);
            pp[2 + d] = ot;
            if (d == 0) {
                pp[0] = mt * 0.69314718055994531f;
                pp[1] = lt;
            }
        }
    }
}

// Joins the splits' (maximum, sum, unnormalised output): one workgroup a query and head.
constexpr int kMostSplits = 256;
template <typename T>
__global__ __launch_bounds__(256) void q4_merge_kernel(const float* partials, int heads, int hd, int splits, T* out,
                                                       int64_t stride) {
    __shared__ float w[kMostSplits];
    __shared__ float red[4];
    const int64_t th = blockIdx.x, t = th / heads, h = th - t * heads;
    const float* pp = partials + th * splits * (hd + 2);
    const int s = threadIdx.x;
    const float ms = s < splits ? pp[(int64_t)s * (hd + 2)] : -INFINITY;
    const float ls = s < splits ? pp[(int64_t)s * (hd + 2) + 1] : 0.f;
    const float wm = wave_max(ms);
    if ((s & 63) == 0) red[s >> 6] = wm;
    __syncthreads();
    const float mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    // (a split of no key, or of keys without a score, counts for nothing but its NaN)
    const float f = ms == -INFINITY ? (mx == -INFINITY ? 1.f : 0.f) : expf(ms - mx);
    w[s] = f;
    __syncthreads();
    const float wl = wave_sum(s < splits ? ls * f : 0.f);
    if ((s & 63) == 0) red[s >> 6] = wl;
    __syncthreads();
    const float l = (red[0] + red[1]) + (red[2] + red[3]);
    for (int d = s; d < hd; d += 256) {
        float o = 0.f;
        for (int i = 0; i < splits; i++) o += pp[(int64_t)i * (hd + 2) + 2 + d] * w[i];
        out[t * stride + h * hd + d] = (T)(o / l);
    }
}

template <typename T>
void launch(const SplitArgs& p, dim3 grid, hipStream_t st) {
    switch (p.c.nb) {
    case 1: q4_attention_kernel<1, T><<<grid, 64 * kWaves, 0, st>>>(p); break;
    case 2: q4_attention_kernel<2, T><<<grid, 64 * kWaves, 0, st>>>(p); break;
    case 3: q4_attention_kernel<3, T><<<grid, 64 * kWaves, 0, st>>>(p); break;
    case 4: q4_attention_kernel<4, T><<<grid, 64 * kWaves, 0, st>>>(p); break;
    case 5: q4_attention_kernel<5, T><<<grid, 64 * kWaves, 0, st>>>(p); break;
    case 6: q4_attention_kernel<6, T><<<grid, 64 * kWaves, 0, st>>>(p); break;
    case 7: q4_attention_kernel<7, T><<<grid, 64 * kWaves, 0, st>>>(p); break;
    default: q4_attention_kernel<8, T><<<grid, 64 * kWaves, 0, st>>>(p); break;
    }
}

}  // namespace

int q4_attention_splits(int tokens, int heads, int kv_heads, int hd, int length) {
    const int64_t groups = ((int64_t)tokens * (heads / kv_heads) + 15) / 16 * kv_heads;
    const int tiles = (length + kQ4Tile - 1) / kQ4Tile;
    // about two workgroups a CU, and a tile at least for each wave
    const int64_t want = 2 * (int64_t)device_cus() / groups, most = (tiles + kWaves - 1) / kWaves;
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kMostSplits}));
}

int64_t q4_attention_partials(int tokens, int heads, int hd, int splits) {
    return splits > 1 ? (int64_t)tokens * heads * splits * (hd + 2) : 0;
}

hipError_t launch_q4_attention(bool f16_rows, const Q4Attention& a, const Q4Cache& c, int splits, hipStream_t st) {
    if (a.tokens <= 0) return hipSuccess;
    SplitArgs p;
    p.a = a;
    p.c = c;
    p.G = a.heads / c.kv_heads;
    p.splits = splits;
    const int hd = 32 * c.nb;
    p.scale_log2 = 1.4426950408889634f / sqrtf((float)hd);
    const int64_t groups = ((int64_t)a.tokens * p.G + 15) / 16;
    const dim3 grid((unsigned)(groups * splits), c.kv_heads);
    if (f16_rows) launch<f16>(p, grid, st);
    else launch<float>(p, grid, st);
    if (splits > 1) {
        const unsigned rows = (unsigned)((int64_t)a.tokens * a.heads);
        if (f16_rows) q4_merge_kernel<f16><<<rows, 256, 0, st>>>(a.partials, a.heads, hd, splits, (f16*)a.out, a.out_stride);
        else q4_merge_kernel<float><<<rows, 256, 0, st>>>(a.partials, a.heads, hd, splits, (float*)a.out, a.out_stride);
    }
    return hipGetLastError();
}
