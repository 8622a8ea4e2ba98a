// Writing and reading back a KV cache held in 4 bits (kv_q4.h), and the
// per-head RMS norm of queries and keys with their rotation.
#include "kv_q4.h"

namespace {

constexpr int kBlock = 256;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// N elements in one access, wherever an element may lie.
template <typename T, int N>
struct Vec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

// ------------------------------------------------------------------ store
// Four waves take a 32-token tile of one KV head: 16 tokens of the keys or of the
// values each.  Lane 16 g + c holds the values 8 g .. 8 g + 7 of a block of token c,
// which is the word of the keys' layout it writes.  A block's largest value is
// found among its four lanes; the values' bytes of four neighbouring tokens, a word
// of their layout, change places within a quad of lanes.  All of a wave's rows are
// read before the first is used, so it waits for memory once; LDS holds only which
// tokens have no form.
//
// The value of largest magnitude, the first of equals, of a lane's eight and then of
// the block's four lanes.
__device__ __forceinline__ float larger(float a, float b) { return fabsf(b) > fabsf(a) ? b : a; }  // (b comes after a)
__device__ __forceinline__ float block_peak(const float (&v)[8], int g) {
    const float m = larger(larger(larger(v[0], v[1]), larger(v[2], v[3])), larger(larger(v[4], v[5]), larger(v[6], v[7])));
    const float o = xor_partner16(m), p = g & 1 ? larger(o, m) : larger(m, o);
    const float q = xor_partner32(p);
    return g & 2 ? larger(q, p) : larger(p, q);
}
struct Block {
    uint32_t nibbles;  // nibble i: value i
    uint32_t scale;    // f16 bits
    bool odd;          // a value of this lane without a form
};
__device__ __forceinline__ Block quantise(const float (&v)[8], int g) {
#pragma clang fp contract(off)
    Block r;
    r.odd = false;
#pragma unroll
    for (int e = 0; e < 8; e++) r.odd |= !(fabsf(v[e]) <= kQ4Most);
    const float d = block_peak(v, g) / -8.0f;
    const float id = d != 0.f ? 1.0f / d : 0.f;
    r.nibbles = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float p = v[e] * id;
        const float s = p + 8.5f;
        // (bounds for the values without a form, whose scale says so)
        r.nibbles |= (uint32_t)(int)fminf(fmaxf(s, 0.f), 15.f) << (4 * e);
    }
    r.scale = __builtin_bit_cast(uint16_t, (f16)d);
    return r;
}
// A word's bytes j and the quad's lanes: lane r gets byte r of the words of lanes 0, 2, 1, 3
// (the order of the values' bytes).
__device__ __forceinline__ uint32_t quad_bytes(uint32_t w, int r) {
    const uint32_t x1 = dpp_mov_i<0xB1>(w), x2 = dpp_mov_i<0x4E>(w), x3 = dpp_mov_i<0x1B>(w);  // of lanes r ^ 1, ^ 2, ^ 3
    const int sh = 8 * r;
    const uint32_t b[4] = {(w >> sh) & 255, (x1 >> sh) & 255, (x2 >> sh) & 255, (x3 >> sh) & 255};  // of lane r ^ i
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int from = r ^ i;  // the token; its byte:
        out |= b[i] << (8 * (((from & 1) << 1) | (from >> 1)));
    }
    return out;
}

// ROPE: a session's [q | k | v] rows.  The keys are rotated on the way in (pairs
// (2 i, 2 i + 1), evaluated as rope_store_kernel does), and workgroups past the KV
// heads rotate a query head of the tile's tokens each, in place or into f16.
template <int NB, typename T, bool ROPE>
__global__ __launch_bounds__(kBlock) void q4_store_kernel(HeadRows kr, HeadRows vr, int tokens, int start,
                                                          const int* start_dev, Q4Cache c, Q4Queries qr) {
#pragma clang fp contract(off)
    constexpr int HD = 32 * NB, BYTES = q4_tile_bytes(NB);
    __shared__ int without[kQ4Tile];  // tokens without a form
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15, h = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), s = wave & 1;
    const bool val = wave >> 1;
    if (start_dev) start = *start_dev;
    if (start < 0 || start > c.capacity - tokens) return;
    const int tile = start / kQ4Tile + blockIdx.x, at = tile * kQ4Tile;
    const int k0 = max(start - at, 0), k1 = min(start + tokens - at, kQ4Tile);
    if (k0 >= k1) return;  // (the same for the whole workgroup, as is all above)
    if constexpr (ROPE) {
        if (h >= c.kv_heads) {
            const int y = h - c.kv_heads, half = HD / 2;
            for (int i = k0 * half + threadIdx.x; i < k1 * half; i += kBlock) {
                const int pos = at + i / half, e = i % half;
                const int64_t t = pos - start;
                float* x = qr.q + t * qr.stride + (int64_t)y * HD + 2 * e;
                const float2 cs = qr.rope[(int64_t)pos * half + e];
                const float a = x[0], b = x[1];
                const float ac = a * cs.x, bs = b * cs.y, as = a * cs.y, bc = b * cs.x;
                if (qr.q16) {
                    f16* o = qr.q16 + (t * qr.heads + y) * HD + 2 * e;
                    o[0] = (f16)(ac - bs);
                    o[1] = (f16)(as + bc);
                } else {
                    x[0] = ac - bs;
                    x[1] = as + bc;
                }
            }
            return;
        }
    }
    uint8_t* out = (val ? c.v : c.k) + (int64_t)h * q4_head_bytes(c.capacity, NB) + (int64_t)tile * BYTES;
    const int k = 16 * s + c16;
    const bool live = k >= k0 && k < k1;
    const bool busy = 16 * s < k1 && 16 * s + 16 > k0;  // this wave has a token to write
    if (threadIdx.x < kQ4Tile) without[threadIdx.x] = 0;
    uint32_t words[NB], scales[NB];
    bool odd = false;
    if (busy) {
        typedef typename Vec<T, 8>::type vec;
        const HeadRows& rows = val ? vr : kr;
        // (a token that is not written: the row of the first that is, unused)
        const int64_t t = max(at + k0 - start, 0) + (live ? k - k0 : 0);
        const T* x = (const T*)rows.p + t * rows.stride + (int64_t)h * HD + 8 * g;
        vec in[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) in[b] = *(const vec*)(x + 32 * b);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = (float)in[b][e];
            if constexpr (ROPE) {
                if (!val) {
                    const float2* cs = qr.rope + (t + start) * (HD / 2) + 16 * b + 4 * g;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float2 w = cs[e / 2];
                        const float ac = v[e] * w.x, bs = v[e + 1] * w.y, as = v[e] * w.y, bc = v[e + 1] * w.x;
                        v[e] = ac - bs;
                        v[e + 1] = as + bc;
                    }
                }
            }
            const Block q = quantise(v, g);
            words[b] = val ? quad_bytes(q.nibbles, c16 & 3) : q.nibbles;
            scales[b] = q.scale;
            odd |= q.odd;
        }
    }
    __syncthreads();
    if (busy && live && odd) without[k] = 1;
    __syncthreads();
    if (!busy) return;
    if (!val) {
        if (live) {
            uint32_t* p = (uint32_t*)(out + q4_key_word(k, NB, 0, g));
#pragma unroll
            for (int b = 0; b < NB; b++) p[b] = words[b];
        }
    } else {
        // the word of pair 4 g + c16 % 4 of the four tokens from t0
        const int t0 = 16 * s + (c16 & 12);
        uint8_t* p = out + ((c16 >> 2) * 16 + 4 * g + (c16 & 3)) * 8 + 4 * s;
        if (t0 >= k0 && t0 + 4 <= k1) {
#pragma unroll
            for (int b = 0; b < NB; b++) *(uint32_t*)(p + b * 512) = words[b];
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (t0 + r < k0 || t0 + r >= k1) continue;
                const int e = ((r & 1) << 1) | (r >> 1);
#pragma unroll
                for (int b = 0; b < NB; b++) p[b * 512 + e] = (uint8_t)(words[b] >> (8 * e));
            }
        }
    }
    if (!live) return;
    const bool none = without[k];
#pragma unroll
    for (int b = 0; b < NB; b++)
        if (g == (b & 3)) *(uint16_t*)(out + q4_scale(k, NB, b)) = !none ? (uint16_t)scales[b] : val ? 0 : 0x7E00;
}

// ------------------------------------------------------------------ load
// Four waves a tile: two take the keys of 16 tokens each, lane 16 g + c the words of
// token c, two the values, lane 16 g + c pair c of eight tokens.
template <typename T, int N>
__device__ __forceinline__ void put(T* p, const float (&v)[N]) {
    typename Vec<T, N>::type r;
#pragma unroll
    for (int e = 0; e < N; e++) r[e] = (T)v[e];
    *(typename Vec<T, N>::type*)p = r;
}

template <int NB, typename T>
__global__ __launch_bounds__(kBlock) void q4_load_kernel(Q4Cache c, int start, int tokens, T* ko, int64_t ks, T* vo,
                                                         int64_t vs) {
    constexpr int HD = 32 * NB, BYTES = q4_tile_bytes(NB);
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = start / kQ4Tile + blockIdx.x, h = blockIdx.y, at = tile * kQ4Tile;
    const int k0 = max(start - at, 0), k1 = min(start + tokens - at, kQ4Tile);
    const uint8_t* kt = c.k + (int64_t)h * q4_head_bytes(c.capacity, NB) + (int64_t)tile * BYTES;
    const uint8_t* vt = c.v + (int64_t)h * q4_head_bytes(c.capacity, NB) + (int64_t)tile * BYTES;
    auto value = [](uint32_t d, int n) { return (float)__builtin_bit_cast(f16, (uint16_t)d) * (float)(n - 8); };
    if (wave < 2) {
        const int k = 16 * wave + c16;
        if (!ko || k < k0 || k >= k1) return;
        T* out = ko + (int64_t)(at + k - start) * ks + (int64_t)h * HD + 8 * g;
        uint32_t w[NB], d[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            w[b] = *(const uint32_t*)(kt + q4_key_word(k, NB, b, g));
            d[b] = *(const uint16_t*)(kt + q4_scale(k, NB, b));
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = value(d[b], (w[b] >> (4 * e)) & 15);
            put(out + 32 * b, x);
        }
        return;
    }
    if (!vo) return;
    constexpr int HALF = (NB + 1) / 2;
    const int b0 = wave == 2 ? 0 : HALF, b1 = wave == 2 ? HALF : NB;
    T* out = vo + (int64_t)h * HD + 2 * c16;
    u32x2 kd[2], w[HALF], d[2][HALF];
#pragma unroll
    for (int s = 0; s < 2; s++) kd[s] = *(const u32x2*)(kt + q4_scale(16 * s + 4 * g, NB, 0));
#pragma unroll
    for (int i = 0; i < HALF; i++) {
        const int b = min(b0 + i, NB - 1);
        w[i] = *(const u32x2*)(vt + b * 512 + lane * 8);
#pragma unroll
        for (int s = 0; s < 2; s++) d[s][i] = *(const u32x2*)(vt + q4_scale(16 * s + 4 * g, NB, b));
    }
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int k = 16 * s + 4 * g + r;
            if (k < k0 || k >= k1) continue;
            // a key scale of NaN: the token has no form
            const uint32_t none = (kd[s][r >> 1] >> (16 * (r & 1))) & 0x7FFF;
            T* p = out + (int64_t)(at + k - start) * vs;
#pragma unroll
            for (int i = 0; i < HALF; i++) {
                if (b0 + i >= b1) continue;
                const uint32_t q = (w[i][s] >> (8 * (((r & 1) << 1) | (r >> 1)))) & 255;
                const uint32_t sc = none > 0x7C00 ? 0x7E00 : (d[s][i][r >> 1] >> (16 * (r & 1))) & 0xFFFF;
                const float x[2] = {value(sc, q & 15), value(sc, q >> 4)};
                put(p + 32 * (b0 + i), x);
            }
        }
}

template <int N>
struct Int {
    static constexpr int value = N;
};
// f(Int<nb>()) for 1 to 8 blocks a head.
template <typename F>
void by_blocks(int nb, F f) {
    switch (nb) {
    case 1: f(Int<1>()); break;
    case 2: f(Int<2>()); break;
    case 3: f(Int<3>()); break;
    case 4: f(Int<4>()); break;
    case 5: f(Int<5>()); break;
    case 6: f(Int<6>()); break;
    case 7: f(Int<7>()); break;
    default: f(Int<8>()); break;
    }
}

// ------------------------------------------------------------------ norm and rotation
// One pass over the rows.  A lane holds the values [i V, (i + 1) V) of a head's
// first half and of its second, V the values of 16 bytes, so that both kinds of
// pairs, (2 p, 2 p + 1) and (p, p + hd / 2), lie in one lane; L lanes (a power of
// two, the last ones idle where hd / 2 is none) hold a head and sum its squares
// among themselves.
template <typename T, int L, bool ALIGNED>
__global__ __launch_bounds__(kBlock) void norm_rope_kernel(ahip_norm_rope a) {
    constexpr int V = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    const int64_t row = (int64_t)blockIdx.x * (kBlock / L) + threadIdx.x / L;
    const unsigned all = a.heads + a.kv_heads;
    if (row >= (int64_t)a.tokens * all) return;  // (whole groups of L lanes)
    const unsigned t = (unsigned)row / all, y = (unsigned)row - t * all;  // (at most 2^30 rows)
    const int i0 = (threadIdx.x % L) * V, half = a.head_dim / 2;
    const bool key = y >= (unsigned)a.heads, mine = i0 < half;
    const int h = key ? y - a.heads : y;
    const T* x = (const T*)(key ? a.k : a.q) + t * (key ? a.k_stride : a.q_stride) + (int64_t)h * 2 * half;
    T* out = (T*)(key ? a.k_out : a.q_out) + t * (key ? a.k_out_stride : a.q_out_stride) + (int64_t)h * 2 * half;
    const float* gain = key ? a.k_gain : a.q_gain;
    float v[2][V];
#pragma unroll
    for (int s = 0; s < 2; s++) {
        vec r = {};
        if (mine) {
            if constexpr (ALIGNED) {
                r = *(const vec*)(x + s * half + i0);
            } else {
#pragma unroll
                for (int e = 0; e < V; e++) r[e] = x[s * half + i0 + e];
            }
        }
#pragma unroll
        for (int e = 0; e < V; e++) v[s][e] = (float)r[e];
    }
    float f[2][V];  // what each value is scaled by
    if (gain) {
        if (mine)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int e = 0; e < V; e++) f[s][e] = gain[s * half + i0 + e];
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < V; e++) ss += v[0][e] * v[0][e] + v[1][e] * v[1][e];
        const float scale = 1.0f / sqrtf(lane_sum<L>(ss) / (float)(2 * half) + a.eps);
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int e = 0; e < V; e++) v[s][e] = v[s][e] * scale * f[s][e];
    }
    if (!mine) return;
    if (a.rope) {
        const int pos = a.positions ? a.positions[t] : a.start + (int)t;
        const bool known = pos >= 0 && pos < a.rope_positions;
        const float2* cs = (const float2*)a.rope + (int64_t)(known ? pos : 0) * half;
        auto turn = [&](float& p, float& q, float2 c) {
            if (!known) c = {NAN, NAN};  // a position outside the table
            const float r = p * c.x - q * c.y;
            q = p * c.y + q * c.x;
            p = r;
        };
        if (a.interleaved) {
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int e = 0; e < V; e += 2) turn(v[s][e], v[s][e + 1], cs[(s * half + i0 + e) / 2]);
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) turn(v[0][e], v[1][e], cs[i0 + e]);
        }
    }
#pragma unroll
    for (int s = 0; s < 2; s++) {
        if constexpr (ALIGNED) {
            vec r;
#pragma unroll
            for (int e = 0; e < V; e++) r[e] = (T)v[s][e];
            *(vec*)(out + s * half + i0) = r;
        } else {
#pragma unroll
            for (int e = 0; e < V; e++) out[s * half + i0 + e] = (T)v[s][e];
        }
    }
}

template <typename T, int L>
void run_norm_rope(const ahip_norm_rope& a, hipStream_t st) {
    auto odd = [](const void* p, int64_t stride) { return ((uintptr_t)p | (uintptr_t)(stride * sizeof(T))) & 15; };
    const bool aligned = !((a.heads ? odd(a.q, a.q_stride) | odd(a.q_out, a.q_out_stride) : 0) |
                           (a.kv_heads ? odd(a.k, a.k_stride) | odd(a.k_out, a.k_out_stride) : 0));
    const int64_t rows = (int64_t)a.tokens * (a.heads + a.kv_heads);
    const unsigned grid = (unsigned)((rows + kBlock / L - 1) / (kBlock / L));
    if (aligned) norm_rope_kernel<T, L, true><<<grid, kBlock, 0, st>>>(a);
    else norm_rope_kernel<T, L, false><<<grid, kBlock, 0, st>>>(a);
}

}  // namespace

static int tile_span(int start, int tokens) { return (start % kQ4Tile + tokens + kQ4Tile - 1) / kQ4Tile; }

// Tiles (a start known only on the device may lie anywhere in its own) by heads.
static dim3 store_grid(int tokens, int start, const int* start_dev, int heads) {
    return dim3(start_dev ? (tokens + 2 * kQ4Tile - 2) / kQ4Tile : tile_span(start, tokens), heads);
}

hipError_t launch_q4_store(bool f16_rows, HeadRows k, HeadRows v, int tokens, int start, const int* start_dev,
                           const Q4Cache& c, hipStream_t st) {
    if (tokens <= 0) return hipSuccess;
    const dim3 grid = store_grid(tokens, start, start_dev, c.kv_heads);
    by_blocks(c.nb, [&](auto nb) {
        constexpr int NB = decltype(nb)::value;
        if (f16_rows) q4_store_kernel<NB, f16, false><<<grid, kBlock, 0, st>>>(k, v, tokens, start, start_dev, c, Q4Queries());
        else q4_store_kernel<NB, float, false><<<grid, kBlock, 0, st>>>(k, v, tokens, start, start_dev, c, Q4Queries());
    });
    return hipGetLastError();
}

hipError_t launch_q4_append(const Q4Queries& q, int tokens, int start, const int* start_dev, const Q4Cache& c,
                            hipStream_t st) {
    if (tokens <= 0) return hipSuccess;
    const dim3 grid = store_grid(tokens, start, start_dev, c.kv_heads + q.heads);
    const float* k = q.q + (int64_t)q.heads * 32 * c.nb;
    const float* v = k + (int64_t)c.kv_heads * 32 * c.nb;
    by_blocks(c.nb, [&](auto nb) {
        q4_store_kernel<decltype(nb)::value, float, true><<<grid, kBlock, 0, st>>>(
            {k, q.stride}, {v, q.stride}, tokens, start, start_dev, c, q);
    });
    return hipGetLastError();
}

hipError_t launch_q4_load(bool f16_rows, const Q4Cache& c, int start, int tokens, void* ko, int64_t ks, void* vo,
                          int64_t vs, hipStream_t st) {
    if (tokens <= 0) return hipSuccess;
    const dim3 grid(tile_span(start, tokens), c.kv_heads);
    by_blocks(c.nb, [&](auto nb) {
        constexpr int NB = decltype(nb)::value;
        if (f16_rows) q4_load_kernel<NB, f16><<<grid, kBlock, 0, st>>>(c, start, tokens, (f16*)ko, ks, (f16*)vo, vs);
        else q4_load_kernel<NB, float><<<grid, kBlock, 0, st>>>(c, start, tokens, (float*)ko, ks, (float*)vo, vs);
    });
    return hipGetLastError();
}

hipError_t launch_norm_rope(bool f16_rows, const ahip_norm_rope& a, hipStream_t st) {
    if ((int64_t)a.tokens * (a.heads + a.kv_heads) <= 0) return hipSuccess;
    const int lanes = a.head_dim / 2 / (f16_rows ? 8 : 4);  // 2 to 32
    auto go = [&](auto zero) {
        typedef decltype(zero) T;
        if (lanes <= 2) run_norm_rope<T, 2>(a, st);
        else if (lanes <= 4) run_norm_rope<T, 4>(a, st);
        else if (lanes <= 8) run_norm_rope<T, 8>(a, st);
        else if (lanes <= 16) run_norm_rope<T, 16>(a, st);
        else run_norm_rope<T, 32>(a, st);
    };
    if (f16_rows) go((f16)0);
    else go(0.f);
    return hipGetLastError();
}
