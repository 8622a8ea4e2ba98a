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
// A wave per (token, head) row: lane l holds pairs l, l + 64 (head_dim up to 256).
template <typename T>
__global__ __launch_bounds__(kBlock) void norm_rope_kernel(NormRope a) {
    const int64_t row = (int64_t)blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, all = a.heads + a.kv_heads, half = a.hd / 2;
    if (row >= (int64_t)a.tokens * all) return;
    const int64_t t = row / all;
    const int y = (int)(row - t * all);
    const bool key = y >= a.heads;
    const int h = key ? y - a.heads : y;
    const T* x = (const T*)(key ? a.k.p : a.q.p) + t * (key ? a.k.stride : a.q.stride) + (int64_t)h * a.hd;
    T* out = (T*)(key ? a.k_out : a.q_out) + t * (key ? a.k_out_stride : a.q_out_stride) + (int64_t)h * a.hd;
    const float* gain = key ? a.k_gain : a.q_gain;
    float u[2] = {0.f, 0.f}, w[2] = {0.f, 0.f};
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int p = lane + 64 * i;
        if (p < half) {
            u[i] = (float)x[a.interleaved ? 2 * p : p];
            w[i] = (float)x[a.interleaved ? 2 * p + 1 : p + half];
            ss += u[i] * u[i] + w[i] * w[i];
        }
    }
    float scale = 1.f;
    if (gain) scale = 1.0f / sqrtf(wave_sum(ss) / (float)a.hd + a.eps);
    const int pos = a.position ? a.position[t] : a.start + (int)t;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int p = lane + 64 * i;
        if (p >= half) continue;
        const int ia = a.interleaved ? 2 * p : p, ib = a.interleaved ? 2 * p + 1 : p + half;
        float f = u[i], s = w[i];
        if (gain) {
            f = f * scale * gain[ia];
            s = s * scale * gain[ib];
        }
        if (a.rope) {
            float2 cs = {NAN, NAN};  // a position outside the table
            if (pos >= 0 && pos < a.positions) cs = a.rope[(int64_t)pos * half + p];
            const float ra = f * cs.x - s * cs.y;
            s = f * cs.y + s * cs.x;
            f = ra;
        }
        out[ia] = (T)f;
        out[ib] = (T)s;
    }
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

hipError_t launch_norm_rope(bool f16_rows, const NormRope& a, hipStream_t st) {
    const int64_t rows = (int64_t)a.tokens * (a.heads + a.kv_heads);
    if (rows <= 0) return hipSuccess;
    const unsigned grid = (unsigned)((rows + kBlock / 64 - 1) / (kBlock / 64));
    if (f16_rows) norm_rope_kernel<f16><<<grid, kBlock, 0, st>>>(a);
    else norm_rope_kernel<float><<<grid, kBlock, 0, st>>>(a);
    return hipGetLastError();
}
