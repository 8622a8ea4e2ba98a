// A KV cache held in 4 bits: the format, the layout and the launchers.
//
// Values.  Q4_0 blocks of 32 values along the head dimension, with the nibbles
// and f16 scales ahip_quantize gives: d = m / -8 (m the value of largest
// magnitude, the first of equals), n = trunc(x * (1 / d) + 8.5) at most 15, and
// a value reads back as d * (n - 8).  A token whose keys or values of a KV head
// hold a NaN, an infinity or a magnitude past 65,504 has no such form: its key
// scales of that head are NaN and its value scales 0, so that a query that sees
// it gets NaN through its score, one that does not is untouched (0 * finite),
// and both rows read back as NaN.
//
// Layout.  Keys and values in a buffer each: [kv_heads][tiles] tiles of 32
// tokens, the last one padded; nb = head_dim / 32; 576 nb bytes a tile, 18 for
// each 32 values.  The quants of a tile lie in the order in which a wave's lanes
// take them as operands of v_mfma_f32_16x16x32_f16 (lane = 16 g + c), so that the
// attention loads whole tiles without a gap and unpacks them in place:
//   keys    [2 halves of 16 tokens][lane: c the token, g a chunk of 8 dims][nb]
//           words; nibble i of word b is dim 32 b + 8 g + i
//   values  [nb][lane: c a pair of dims, g a group of 4 tokens][8] bytes; byte e
//           of (b, g, c) holds dims 32 b + 2 c (low nibble) and + 1 of token
//           16 (e / 4) + 4 g + {0, 2, 1, 3}[e % 4]
// (a mask picks nibbles 0 and 4, 1 and 5, ... of a word as pairs of 16 bits; the
// byte order of the values makes such pairs neighbouring tokens), then
//   scales  [2 halves][4 groups of 4 tokens][nb][4 tokens] f16
#pragma once

#include "../../include/alpaca_hip.h"
#include "common.h"

constexpr int kQ4Tile = 32;  // tokens
constexpr float kQ4Most = 65504.f;

__host__ __device__ constexpr int64_t q4_tile_bytes(int nb) { return 576 * nb; }  // (64 bits: a tile index times it may need them)
__host__ __device__ constexpr int q4_scales_at(int nb) { return 512 * nb; }
__host__ __device__ inline int q4_tiles(int capacity) { return (int)(((int64_t)capacity + kQ4Tile - 1) / kQ4Tile); }
__host__ __device__ inline int64_t q4_head_bytes(int capacity, int nb) {
    return (int64_t)q4_tiles(capacity) * q4_tile_bytes(nb);
}
// Byte offsets inside a tile of token k (0..31).
__host__ __device__ inline int q4_key_word(int k, int nb, int b, int g) {
    return 4 * (((k >> 4) * 64 + g * 16 + (k & 15)) * nb + b);
}
__host__ __device__ inline int q4_scale(int k, int nb, int b) {
    return q4_scales_at(nb) + 2 * ((((k >> 4) * 4 + ((k >> 2) & 3)) * nb + b) * 4 + (k & 3));
}

// One layer's cache.
struct Q4Cache {
    uint8_t* k = nullptr;
    uint8_t* v = nullptr;
    int kv_heads = 0, capacity = 0, nb = 0;
};

// Rows of `heads` vectors a token, `stride` elements from one token to the next.
struct HeadRows {
    const void* p = nullptr;
    int64_t stride = 0;
};

// Writes `tokens` rows at positions start.. (*start_dev when set; a range
// outside the cache then writes nothing).
hipError_t launch_q4_store(bool f16_rows, HeadRows k, HeadRows v, int tokens, int start, const int* start_dev,
                           const Q4Cache& c, hipStream_t st);
// A session's rows [q | k | v] (interleaved pairs): q rotated in place or, with q16 set, into
// f16 rows [heads][hd]; k rotated and v written at positions start.. .
struct Q4Queries {
    float* q = nullptr;
    int64_t stride = 0;
    int heads = 0;
    const float2* rope = nullptr;  // (cos, sin) [positions][hd / 2]
    f16* q16 = nullptr;
};
hipError_t launch_q4_append(const Q4Queries& q, int tokens, int start, const int* start_dev, const Q4Cache& c,
                            hipStream_t st);
// Reads them back; k_out or v_out may be null.
hipError_t launch_q4_load(bool f16_rows, const Q4Cache& c, int start, int tokens, void* k_out, int64_t k_stride,
                          void* v_out, int64_t v_stride, hipStream_t st);

// Per-head RMS norm and rotation of q and k rows (ahip_qk_norm_rope's arguments, checked).
hipError_t launch_norm_rope(bool f16_rows, const ahip_norm_rope& a, hipStream_t st);

// Causal attention of `tokens` queries at positions start.. (*start_dev when
// set) over the cache; where splits > 1 with a workspace of q4_attention_workspace()
// bytes: kQ4Counters words, zero before and after every launch, and the parts' results.
struct Q4Attention {
    const void* q = nullptr;
    void* out = nullptr;
    int64_t q_stride = 0, out_stride = 0;
    int tokens = 0, heads = 0, start = 0;
    const int* start_dev = nullptr;
    float* partials = nullptr;
    int* counters = nullptr;
};
constexpr int kQ4Counters = 512;
// How a call runs: query columns of a workgroup, its waves, and parts the keys are split into.
// `length`: the positions that the call may see.  A call's workspace does not shrink as it grows.
struct Q4Plan {
    int cols = 16, waves = 4, splits = 1;
};
Q4Plan q4_attention_plan(bool f16_rows, int tokens, int heads, int kv_heads, int hd, int length);
// Bytes of a launch's workspace, the counters first; 0 for one part.
int64_t q4_attention_workspace(int tokens, int heads, int hd, const Q4Plan& plan);
void q4_set_workspace(Q4Attention& a, void* workspace);
hipError_t launch_q4_attention(bool f16_rows, const Q4Attention& a, const Q4Cache& c, const Q4Plan& plan,
                               hipStream_t st);
