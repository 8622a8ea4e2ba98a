// A KV cache in pages that a table gives to many sequences: the layout and the
// launchers.
//
// Values are f16, as a session's f16 cache holds them.  A token whose keys or
// values of a KV head hold a NaN, an infinity or a magnitude past 65,504 keeps
// NaN keys and zero values in that head: a query that sees it gets NaN through
// its score, one that does not is untouched (0 * finite), and both rows read back
// as NaN.
//
// Layout.  Keys and values in a buffer each, [page][kv_head][tile] of tiles of 16
// tokens (32 head_dim bytes), in the order in which a wave's lanes take them as
// operands of both shapes of f16 matrix products, so that tiles go from memory to
// registers or LDS without being rearranged:
//   keys    [head_dim / 8][16 slots][8 dims]; token t lies in slot
//           8 ((t >> 2) & 1) + 4 (t >> 3) + (t & 3)
//   values  [2 halves of 8 tokens][head_dim][8 tokens]
// With the keys' slots as rows of S^T = K Q^T, a lane of v_mfma_f32_32x32x16 holds
// the scores of 8 consecutive tokens in 8 consecutive registers, and one of
// v_mfma_f32_16x16x32 those of 8 consecutive tokens in its two results' 4 + 4: the
// 8 values of a row of P that the second product takes, beside 8 tokens of a value.
#pragma once

#include "../../include/alpaca_hip.h"
#include "common.h"

constexpr int kPagedTile = 16;  // tokens

__host__ __device__ constexpr int paged_tile_bytes(int hd) { return 32 * hd; }
__host__ __device__ constexpr int paged_key_slot(int t) { return 8 * ((t >> 2) & 1) + 4 * ((t >> 3) & 1) + (t & 3); }

struct PagedKV {
    uint8_t* k = nullptr;
    uint8_t* v = nullptr;
    int kv_heads = 0, hd = 0, pages = 0;
    int tiles_log2 = 0;  // of a page
};

// The batch of a step (ahip_paged_batch): what its arrays hold is read by the kernels only, which
// take any content: row ranges are cut to the rows, positions below 0 or past the table have no page.
struct PagedSteps {
    const int* row_starts = nullptr;
    const int* lengths = nullptr;
    const int* table = nullptr;
    int sequences = 0, table_stride = 0, rows = 0;
};

struct PagedRows {
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    void* q_out = nullptr;
    int64_t q_stride = 0, k_stride = 0, v_stride = 0, q_out_stride = 0;
    const float2* rope = nullptr;
    int rope_positions = 0, heads = 0, interleaved = 0;
};
hipError_t launch_paged_append(bool f16_rows, const PagedRows& r, const PagedSteps& b, const PagedKV& c, hipStream_t st);
hipError_t launch_paged_load(bool f16_rows, const PagedSteps& b, const PagedKV& c, void* k, int64_t k_stride, void* v,
                             int64_t v_stride, hipStream_t st);

struct PagedAttention {
    const void* q = nullptr;
    void* out = nullptr;
    int64_t q_stride = 0, out_stride = 0;
    int heads = 0, window = 0, sinks = 0, max_rows = 0;
    void* workspace = nullptr;
};
constexpr int kPagedCounters = 1024;  // words at the front of a workspace, zero before and after every launch
int64_t paged_attention_workspace(int hd);
hipError_t launch_paged_attention(bool f16_rows, const PagedAttention& a, const PagedSteps& b, const PagedKV& c,
                                  hipStream_t st);

// ------------------------------------------------------------------ on the device

// One sequence of a batch.
struct PagedSeq {
    int row0, n;      // its rows
    int length;       // tokens with the new ones; row i has position length - n + i
};
constexpr int kPagedMost = 1 << 30;  // positions
__device__ __forceinline__ PagedSeq paged_seq(const PagedSteps& b, int s) {
    const int a = min(max(gptr(b.row_starts)[s], 0), b.rows);
    const int e = min(max(gptr(b.row_starts)[s + 1], a), b.rows);
    return {a, e - a, min(max(gptr(b.lengths)[s], 0), kPagedMost)};
}

// Sums of a wave's lanes 0..l in lane l.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return x;
}

// The sequence that has item `w` where one of rows q has items(q) of them, in order, and w - those before; s = -1 past
// the last.  By a whole wave, the same in all lanes.
struct PagedItem {
    int s, i;
    PagedSeq seq;
};
template <typename F>
__device__ __forceinline__ PagedItem paged_find(const PagedSteps& b, int w, F items) {
    const int lane = __lane_id();
    for (int s0 = 0; s0 < b.sequences; s0 += 64) {
        PagedSeq q{0, 0, 0};
        if (s0 + lane < b.sequences) q = paged_seq(b, s0 + lane);
        const int mine = q.n ? items(q) : 0, upto = wave_scan(mine);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > w);
        if (past) {
            const int l = __builtin_ctzll(past);
            auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
            return {s0 + l, w - of(upto - mine), {of(q.row0), of(q.n), of(q.length)}};
        }
        w -= __builtin_amdgcn_readlane(upto, 63);
    }
    return {-1, 0, {0, 0, 0}};
}

// The page that holds tile `tile` (positions 16 tile ..) of sequence s, or -1; and the tile's place among all tiles
// of KV head kvh.
__device__ __forceinline__ int paged_page(const PagedSteps& b, const PagedKV& c, int s, int tile) {
    const int p = tile >> c.tiles_log2;
    if (tile < 0 || p >= b.table_stride) return -1;
    const int id = gptr(b.table)[(int64_t)s * b.table_stride + p];
    return (unsigned)id < (unsigned)c.pages ? id : -1;
}
__device__ __forceinline__ int64_t paged_tile(const PagedKV& c, int page, int kvh, int tile) {
    return (((int64_t)page * c.kv_heads + kvh) << c.tiles_log2) + (tile & ((1 << c.tiles_log2) - 1));
}
