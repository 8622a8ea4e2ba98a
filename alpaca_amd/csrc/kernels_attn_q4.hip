// Causal grouped-query attention over a KV cache held in 4 bits (kv_q4.h).
#include "kv_q4.h"

namespace {

// One wave per (query, head): a tile of 32 keys at a time, the score of a key in
// two lanes (the halves of the dims), an online softmax, then each lane's dims.
template <typename T>
__global__ __launch_bounds__(64) void q4_attention_kernel(Q4Attention a, Q4Cache c) {
    __shared__ float qs[256], ps[kQ4Tile], ds[kQ4Tile * 8];
    const int lane = threadIdx.x, h = blockIdx.y, nb = c.nb, hd = 32 * nb;
    const int64_t t = blockIdx.x;
    const int start = a.start_dev ? *a.start_dev : a.start;
    const int h_kv = h / (a.heads / c.kv_heads);
    T* out = (T*)a.out + t * a.out_stride + (int64_t)h * hd;
    const bool inside = start >= 0 && start <= c.capacity - a.tokens;
    const int end = inside ? start + (int)t + 1 : 0;
    const T* q = (const T*)a.q + t * a.q_stride + (int64_t)h * hd;
    const float scale = 1.0f / sqrtf((float)hd);
    for (int d = lane; d < hd; d += 64) qs[d] = (float)q[d] * scale;
    __syncthreads();
    const uint8_t* kt = c.k + (int64_t)h_kv * q4_head_bytes(c.capacity, nb);
    const uint8_t* vt = c.v + (int64_t)h_kv * q4_head_bytes(c.capacity, nb);
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < end; k0 += kQ4Tile, kt += q4_tile_bytes(nb), vt += q4_tile_bytes(nb)) {
        const int k = lane & 31;
        float s = 0.f;
        for (int b = 0; b < nb; b++) {
            float p = 0.f;
            for (int g = 2 * (lane >> 5); g < 2 * (lane >> 5) + 2; g++) {
                const uint32_t w = *(const uint32_t*)(kt + q4_key_word(k, nb, b, g));
                for (int e = 0; e < 8; e++) p += qs[32 * b + 8 * g + e] * (float)((int)((w >> (4 * e)) & 15) - 8);
            }
            s += p * (float)*(const f16*)(kt + q4_scale(k, nb, b));
            if (lane < kQ4Tile) ds[k * 8 + b] = (float)*(const f16*)(vt + q4_scale(k, nb, b));
        }
        s += __shfl_xor(s, 32, 64);
        if (k0 + k >= end) s = -INFINITY;
        const float mn = fmaxf(m, wave_max(s));
        const float mref = mn == -INFINITY ? 0.f : mn, alpha = expf(m - mref), p = expf(s - mref);
        l = l * alpha + lane_sum<32>(p);
        m = mn;
        if (lane < kQ4Tile) ps[k] = p;
        __syncthreads();
        for (int i = 0; 64 * i < hd; i++) {
            const int d = lane + 64 * i;
            o[i] *= alpha;
            if (d < hd)
                for (int j = 0; j < kQ4Tile; j++) {
                    const int w = vt[q4_value_byte(j, d / 32, d % 32 / 2)];
                    if (k0 + j < end) o[i] += ps[j] * ds[j * 8 + d / 32] * (float)((d & 1 ? w >> 4 : w & 15) - 8);
                }
        }
        __syncthreads();
    }
    for (int i = 0; 64 * i < hd; i++)
        if (lane + 64 * i < hd) out[lane + 64 * i] = (T)(o[i] / l);
}

}  // namespace

int q4_attention_splits(int tokens, int heads, int kv_heads, int hd, int length) { return 1; }

int64_t q4_attention_partials(int tokens, int heads, int hd, int splits) {
    return splits > 1 ? (int64_t)tokens * heads * splits * (hd + 2) : 0;
}

hipError_t launch_q4_attention(bool f16_rows, const Q4Attention& a, const Q4Cache& c, int splits, hipStream_t st) {
    if (a.tokens <= 0) return hipSuccess;
    const dim3 grid(a.tokens, a.heads);
    if (f16_rows) q4_attention_kernel<f16><<<grid, 64, 0, st>>>(a, c);
    else q4_attention_kernel<float><<<grid, 64, 0, st>>>(a, c);
    return hipGetLastError();
}
