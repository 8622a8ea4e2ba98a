// Writing and reading back a KV cache held in 4 bits (kv_q4.h), and the
// per-head RMS norm of queries and keys with their rotation.
#include "kv_q4.h"

namespace {

constexpr int kBlock = 256;

template <typename T>
__device__ __forceinline__ float4 load4f(const T* p);
template <>
__device__ __forceinline__ float4 load4f<float>(const float* p) { return {p[0], p[1], p[2], p[3]}; }
template <>
__device__ __forceinline__ float4 load4f<f16>(const f16* p) { return {(float)p[0], (float)p[1], (float)p[2], (float)p[3]}; }

// ------------------------------------------------------------------ store
// A workgroup takes the tokens of one 32-token tile of one KV head: 8 lanes a
// block of 32 values, 4 values a lane.  The tile's bytes are put together in LDS
// and leave as whole words where all 32 tokens are written; the tokens of a tile
// that are not written keep their bytes.
template <typename T>
__global__ __launch_bounds__(kBlock) void q4_store_kernel(HeadRows kr, HeadRows vr, int tokens, int start,
                                                          const int* start_dev, Q4Cache c) {
#pragma clang fp contract(off)
    extern __shared__ __align__(16) uint8_t lds[];  // key tile, value tile
    __shared__ int bad[kQ4Tile];
    const int nb = c.nb, hd = 32 * nb, bytes = q4_tile_bytes(nb), tid = threadIdx.x;
    if (start_dev) start = *start_dev;
    if (start < 0 || start > c.capacity - tokens) return;
    const int tile = start / kQ4Tile + blockIdx.x, h = blockIdx.y;
    const int k0 = max(start - tile * kQ4Tile, 0), k1 = min(start + tokens - tile * kQ4Tile, kQ4Tile);
    if (k0 >= k1) return;
    const int n = k1 - k0;
    if (tid < kQ4Tile) bad[tid] = 0;
    __syncthreads();
    // (rounds of whole 8-lane groups: the lanes of a block reduce together)
    for (int i = tid; i < n * nb * 2 * 8; i += kBlock) {
        const int j = i & 7, blk = i >> 3;  // blocks: [value?][token][b]
        const int b = blk % nb, row = blk / nb;
        const bool val = row >= n;
        const int k = k0 + (val ? row - n : row);
        const int64_t t = (int64_t)tile * kQ4Tile + k - start;
        const T* x = (const T*)(val ? vr.p : kr.p) + t * (val ? vr.stride : kr.stride) + (int64_t)h * hd + 32 * b + 4 * j;
        const float4 f = load4f(x);
        const float v[4] = {f.x, f.y, f.z, f.w};
        // the value of largest magnitude, the first of equals: the larger magnitude wins, then the lower index
        float m = v[0];
        bool odd = !(fabsf(v[0]) <= kQ4Most);
#pragma unroll
        for (int e = 1; e < 4; e++) {
            if (fabsf(v[e]) > fabsf(m)) m = v[e];
            odd |= !(fabsf(v[e]) <= kQ4Most);
        }
#pragma unroll
        for (int s = 1; s < 8; s <<= 1) {
            const float o = __shfl_xor(m, s, 64);
            const bool lower = (j & s) == 0;  // this lane's values come before its partner's
            if (fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && !lower)) m = o;
        }
        if (odd) bad[k] = 1;
        const float d = m / -8.0f;
        const float id = d != 0.f ? 1.0f / d : 0.f;
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float p = v[e] * id;
            const float s = p + 8.5f;
            // (bounds for the values without a form, whose scale says so)
            w |= (uint32_t)(int)fminf(fmaxf(s, 0.f), 15.f) << (4 * e);
        }
        uint8_t* img = lds + (val ? bytes : 0);
        if (val) {
            img[q4_value_byte(k, b, 2 * j)] = (uint8_t)(w & 255);
            img[q4_value_byte(k, b, 2 * j + 1)] = (uint8_t)(w >> 8);
        } else {
            *(uint16_t*)(img + q4_key_word(k, nb, b, j >> 1) + 2 * (j & 1)) = (uint16_t)w;
        }
        if (j == 0) *(f16*)(img + q4_scale(k, nb, b)) = (f16)d;
    }
    __syncthreads();
    const int64_t at = (int64_t)h * q4_head_bytes(c.capacity, nb) + (int64_t)tile * bytes;
    uint8_t* kd = c.k + at;
    uint8_t* vd = c.v + at;
    if (n == kQ4Tile) {
        for (int i = tid * 16; i < q4_scales_at(nb); i += kBlock * 16) {
            *(int4*)(kd + i) = *(const int4*)(lds + i);
            *(int4*)(vd + i) = *(const int4*)(lds + bytes + i);
        }
    } else {
        for (int i = tid; i < n * nb * 4; i += kBlock) {
            const int o = q4_key_word(k0 + i / (4 * nb), nb, i / 4 % nb, i & 3);
            *(uint32_t*)(kd + o) = *(const uint32_t*)(lds + o);
        }
        for (int i = tid; i < n * nb * 16; i += kBlock) {
            const int o = q4_value_byte(k0 + i / (16 * nb), i / 16 % nb, i & 15);
            vd[o] = lds[bytes + o];
        }
    }
    for (int i = tid; i < n * nb; i += kBlock) {
        const int k = k0 + i / nb, o = q4_scale(k, nb, i % nb);
        *(uint16_t*)(kd + o) = bad[k] ? 0x7E00 : *(const uint16_t*)(lds + o);
        *(uint16_t*)(vd + o) = bad[k] ? 0 : *(const uint16_t*)(lds + bytes + o);
    }
}

// ------------------------------------------------------------------ load
// 8 values a thread, the 32 tokens of a tile a workgroup.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) p[e] = (T)v[e];
}

template <typename T>
__global__ __launch_bounds__(kBlock) void q4_load_kernel(Q4Cache c, int start, int tokens, T* ko, int64_t ks, T* vo,
                                                         int64_t vs) {
    const int nb = c.nb, hd = 32 * nb, bytes = q4_tile_bytes(nb);
    const int tile = start / kQ4Tile + blockIdx.x, h = blockIdx.y;
    const int k0 = max(start - tile * kQ4Tile, 0), k1 = min(start + tokens - tile * kQ4Tile, kQ4Tile);
    const int64_t at = (int64_t)h * q4_head_bytes(c.capacity, nb) + (int64_t)tile * bytes;
    const uint8_t* kd = c.k + at;
    const uint8_t* vd = c.v + at;
    for (int i = threadIdx.x; i < (k1 - k0) * nb * 4; i += kBlock) {
        const int k = k0 + i / (4 * nb), b = i / 4 % nb, g = i & 3;
        const int64_t t = (int64_t)tile * kQ4Tile + k - start, o = (int64_t)h * hd + 32 * b + 8 * g;
        const float dk = (float)*(const f16*)(kd + q4_scale(k, nb, b));
        float x[8];
        if (ko) {
            const uint32_t w = *(const uint32_t*)(kd + q4_key_word(k, nb, b, g));
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = dk * (float)((int)((w >> (4 * e)) & 15) - 8);
            store8(ko + t * ks + o, x);
        }
        if (vo) {
            // a key scale of NaN: the token has no form
            const float dv = dk != dk ? dk : (float)*(const f16*)(vd + q4_scale(k, nb, b));
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int w = vd[q4_value_byte(k, b, 4 * g + e)];
                x[2 * e] = dv * (float)((w & 15) - 8);
                x[2 * e + 1] = dv * (float)((w >> 4) - 8);
            }
            store8(vo + t * vs + o, x);
        }
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

hipError_t launch_q4_store(bool f16_rows, HeadRows k, HeadRows v, int tokens, int start, const int* start_dev,
                           const Q4Cache& c, hipStream_t st) {
    if (tokens <= 0) return hipSuccess;
    // a start known only on the device may lie anywhere in its tile
    const dim3 grid(start_dev ? (tokens + 2 * kQ4Tile - 2) / kQ4Tile : tile_span(start, tokens), c.kv_heads);
    const size_t lds = 2 * (size_t)q4_tile_bytes(c.nb);
    if (f16_rows) q4_store_kernel<f16><<<grid, kBlock, lds, st>>>(k, v, tokens, start, start_dev, c);
    else q4_store_kernel<float><<<grid, kBlock, lds, st>>>(k, v, tokens, start, start_dev, c);
    return hipGetLastError();
}

hipError_t launch_q4_load(bool f16_rows, const Q4Cache& c, int start, int tokens, void* ko, int64_t ks, void* vo,
                          int64_t vs, hipStream_t st) {
    if (tokens <= 0) return hipSuccess;
    const dim3 grid(tile_span(start, tokens), c.kv_heads);
    if (f16_rows) q4_load_kernel<f16><<<grid, kBlock, 0, st>>>(c, start, tokens, (f16*)ko, ks, (f16*)vo, vs);
    else q4_load_kernel<float><<<grid, kBlock, 0, st>>>(c, start, tokens, (float*)ko, ks, (float*)vo, vs);
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
