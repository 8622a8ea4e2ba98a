// Writing a batch's keys and values into a cache in pages (paged.h), rotated to
// their positions on the way, with its queries' rotation; and reading them back.
//
// A pair of dims (a, b) of a head at position p becomes (a cos - b sin, a sin + b cos)
// with the table's angle of (p, pair); pairs are adjacent dims or halves of the head.
//
// A workgroup of 256 threads takes as many heads as have 16 lanes of 16 dims a token: KV
// heads of one tile of 16 positions of a sequence, or query heads of 16 rows (once or
// twice that many).  A thread rotates 16 dims of one token, its 8 angles in registers, and
// turns 8 tokens by 2 dims of the values.  Keys of a tile's 16 tokens are written 256
// bytes at a time, values 16 bytes where all 8 tokens are new and 2 where a group is
// only partly so.
//
// Bound by memory: 4,096 f16 tokens of 32/8 heads of 128 with what reads them back 33 us (4.1
// TB/s over both launches).  Few rows: a chain of five round trips to memory, the batch, the
// page, the angles, the rows and the stores, 4.5 us for one token of 9/3 heads of 64.
#include "paged.h"

namespace {

constexpr int kThreads = 256;

template <typename T>
struct Lines;  // 8 dims at once
template <>
struct Lines<float> {
    static __device__ __forceinline__ void load(const float* p, float (&x)[8], bool whole) {
        if (whole) {
            const int4 a = gload_i4(p), b = gload_i4(p + 4);
            const int u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = __int_as_float(u[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = gptr(p)[e];
        }
    }
    static __device__ __forceinline__ void store(float* p, const float (&x)[8], bool whole) {
        if (whole) {
            *(AS_GLOBAL f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
            *(AS_GLOBAL f32x4*)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) gptr(p)[e] = x[e];
        }
    }
};
__device__ __forceinline__ f16x8 rounded(const float (&x)[8]) {
    return {(f16)x[0], (f16)x[1], (f16)x[2], (f16)x[3], (f16)x[4], (f16)x[5], (f16)x[6], (f16)x[7]};
}
template <>
struct Lines<f16> {
    static __device__ __forceinline__ void load(const f16* p, float (&x)[8], bool whole) {
        if (whole) {
            const f16x8 h = *(const AS_GLOBAL f16x8*)p;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = (float)h[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = (float)gptr(p)[e];
        }
    }
    static __device__ __forceinline__ void store(f16* p, const float (&x)[8], bool whole) {
        if (whole) {
            *(AS_GLOBAL f16x8*)p = rounded(x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) gptr(p)[e] = (f16)x[e];
        }
    }
};
// Two dims.
template <typename T>
__device__ __forceinline__ float2 load_two(const T* p, bool whole) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    if (whole) {
        const T2 x = *(const AS_GLOBAL T2*)p;
        return make_float2((float)x[0], (float)x[1]);
    }
    return make_float2((float)gptr(p)[0], (float)gptr(p)[1]);
}
template <typename T>
__device__ __forceinline__ void store_two(T* p, float a, float b, bool whole) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    if (whole) {
        *(AS_GLOBAL T2*)p = T2{(T)a, (T)b};
    } else {
        gptr(p)[0] = (T)a;
        gptr(p)[1] = (T)b;
    }
}
// An f16 that is a NaN or an infinity.
__device__ __forceinline__ bool odd16(f16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7C00u) == 0x7C00u; }

// What a workgroup works on: the tile, and its thread's token of it.
struct Place {
    PagedSeq seq;
    int s, tile, pos0;  // pos0: the position of the sequence's first row
    __device__ __forceinline__ int row(int pos) const {  // of a position, -1 where it is not new
        const int i = pos - pos0;
        return i >= 0 && i < seq.n ? seq.row0 + i : -1;
    }
};
__device__ __forceinline__ bool find_place(const PagedSteps& b, int tile, Place& p) {
    const PagedItem it = paged_find(b, tile, [&](const PagedSeq& q) {
        // (>> rounds down: rows of negative positions have tiles too)
        return ((q.length - 1) >> 4) - ((q.length - q.n) >> 4) + 1;
    });
    if (it.s < 0) return false;
    p.s = it.s;
    p.seq = it.seq;
    p.pos0 = p.seq.length - p.seq.n;
    p.tile = (p.pos0 >> 4) + it.i;
    return true;
}

struct AppendArgs {
    PagedRows r;
    PagedSteps b;
    PagedKV c;
    int tiles, kv_slices;  // workgroups: KV heads of tiles of positions, then
    int blocks, q_slices;  // query heads of blocks of 16 rows
    bool together;         // those of the same tokens on one XCD, whose cache then has their angles
    int lanes, at_once;    // 16-dim lanes of a head, heads at once
    bool q_whole, k_whole, v_whole, out_whole, rope_whole;  // rows that lie on 16 bytes
};

// The two runs of 8 dims that lane `u` of a head rotates.
__device__ __forceinline__ void runs(int u, int hd, int interleaved, int (&d)[2]) {
    d[0] = interleaved ? 16 * u : 8 * u;
    d[1] = interleaved ? 16 * u + 8 : hd / 2 + 8 * u;
}
__device__ __forceinline__ void rotate(float (&x)[2][8], const float2 (&cs)[8], int interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float& a = interleaved ? x[i >> 2][2 * (i & 3)] : x[0][i];
        float& b = interleaved ? x[i >> 2][2 * (i & 3) + 1] : x[1][i];
        const float y = a * cs[i].x - b * cs[i].y, z = a * cs[i].y + b * cs[i].x;
        a = y;
        b = z;
    }
}

// The position of each lane's row, 16 lanes a row; INT_MIN for a row of no sequence.
__device__ __forceinline__ int position_of(const PagedSteps& b, int row) {
    const int lane = __lane_id();
    int pos = INT32_MIN;
    for (int s0 = 0; s0 < b.sequences; s0 += 64) {
        PagedSeq q{0, 0, 0};
        if (s0 + lane < b.sequences) q = paged_seq(b, s0 + lane);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int r = __builtin_amdgcn_readlane(row, 16 * t);
            const uint64_t has = __builtin_amdgcn_ballot_w64(r >= q.row0 && r < q.row0 + q.n);
            if (!has) continue;
            const int p = __builtin_amdgcn_readlane(q.length - q.n - q.row0, __builtin_ctzll(has)) + r;
            if (lane >> 4 == t) pos = p;
        }
    }
    return pos;
}

template <typename T, bool INTERLEAVED, int PASSES>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(AppendArgs p) {
    __shared__ uint32_t odd[16];  // a bit a head of the slice: tokens that have no form
    int unit, slice;
    bool queries;
    if (p.together) {  // workgroups go round the 8 XCDs
        const int slices = p.kv_slices + p.q_slices, eight = blockIdx.x / (8 * slices), i = blockIdx.x - eight * 8 * slices;
        unit = 8 * eight + (i & 7), slice = i >> 3;
        queries = slice >= p.kv_slices;
        if (queries) slice -= p.kv_slices;
    } else {
        const int kv = p.tiles * p.kv_slices, units = (int)blockIdx.x < kv ? p.tiles : p.blocks;
        queries = (int)blockIdx.x >= kv;
        const int w = blockIdx.x - (queries ? kv : 0);
        slice = w / units, unit = w - slice * units;
    }
    // queries: the lanes of a token side by side, as their rows lie; keys: the tokens, as the pages do
    const int hd = p.c.hd, lo = threadIdx.x & 15, hi = threadIdx.x >> 4, tok = queries ? hi : lo, u = queries ? lo : hi;
    const int lane = u % p.lanes, sub = u / p.lanes;
    Place at;
    int pos, row;
    if (queries) {
        row = unit * 16 + tok;
        pos = position_of(p.b, row);
        if (pos == INT32_MIN) row = -1;
    } else {
        if (!find_place(p.b, unit, at)) return;
        pos = at.tile * 16 + tok;
        row = at.row(pos);
    }
    int d[2];
    runs(lane, hd, INTERLEAVED, d);
    float2 cs[8];
    const bool turned = p.r.rope != nullptr;
    if (turned) {
        if (pos >= 0 && pos < p.r.rope_positions) {
            const float2* t = p.r.rope + (int64_t)pos * (hd / 2) + 8 * lane;
            if (p.rope_whole) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int4 y = gload_i4(t + 2 * i);
                    cs[2 * i] = make_float2(__int_as_float(y.x), __int_as_float(y.y));
                    cs[2 * i + 1] = make_float2(__int_as_float(y.z), __int_as_float(y.w));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) cs[i] = gload_f2(t + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) cs[i] = make_float2(NAN, NAN);
        }
    }
    if (queries) {
        if (row < 0 || sub >= p.at_once) return;
        const int h = slice * p.at_once * PASSES + sub;
        const T* q = (const T*)p.r.q + row * p.r.q_stride + (int64_t)h * hd;
        T* out = (T*)p.r.q_out + row * p.r.q_out_stride + (int64_t)h * hd;
        const int64_t next = (int64_t)p.at_once * hd;
        float x[PASSES][2][8];
#pragma unroll
        for (int i = 0; i < PASSES; i++)
            if (h + i * p.at_once < p.r.heads) {
                Lines<T>::load(q + i * next + d[0], x[i][0], p.q_whole);
                Lines<T>::load(q + i * next + d[1], x[i][1], p.q_whole);
            }
#pragma unroll
        for (int i = 0; i < PASSES; i++)
            if (h + i * p.at_once < p.r.heads) {
                if (turned) rotate(x[i], cs, INTERLEAVED);
                Lines<T>::store(out + i * next + d[0], x[i][0], p.out_whole);
                Lines<T>::store(out + i * next + d[1], x[i][1], p.out_whole);
            }
        return;
    }
    const int page = paged_page(p.b, p.c, at.s, at.tile);  // (the same for the whole workgroup)
    if (page < 0) return;
    if (threadIdx.x < 16) odd[threadIdx.x] = 0;
    __syncthreads();
    const int h0 = slice * p.at_once, kvh = h0 + sub;
    const bool mine = row >= 0 && sub < p.at_once && kvh < p.c.kv_heads;
    // values: 2 dims of 8 tokens a thread
    const int pairs = hd / 2, vi = threadIdx.x;
    const int vsub = vi / (2 * pairs), half = (vi / pairs) & 1, dim = 2 * (vi % pairs);
    const int vh = h0 + vsub, vpos = at.tile * 16 + 8 * half;
    const bool values = vsub < p.at_once && vh < p.c.kv_heads;
    float2 v[8];
    int fresh = 0;
    if (values) {
#pragma unroll
        for (int e = 0; e < 8; e++) {  // (a token that is not new: another's row, unused)
            const int i = vpos + e - at.pos0, r = at.seq.row0 + min(max(i, 0), at.seq.n - 1);
            fresh |= (i >= 0 && i < at.seq.n) << e;
            v[e] = load_two((const T*)p.r.v + r * p.r.v_stride + (int64_t)vh * hd + dim, p.v_whole);
        }
    }
    f16x8 key[2];
    if (mine) {
        const T* k = (const T*)p.r.k + row * p.r.k_stride + (int64_t)kvh * hd;
        float x[2][8];
        Lines<T>::load(k + d[0], x[0], p.k_whole);
        Lines<T>::load(k + d[1], x[1], p.k_whole);
        if (turned) rotate(x, cs, INTERLEAVED);
        key[0] = rounded(x[0]);
        key[1] = rounded(x[1]);
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 8; e++) bad = bad || odd16(key[0][e]) || odd16(key[1][e]);
        if (bad) atomicOr(&odd[tok], 1u << sub);
    }
    f16x8 va = {}, vb = {};
    if (values) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (!(fresh >> e & 1)) continue;
            va[e] = (f16)v[e].x;
            vb[e] = (f16)v[e].y;
            if (odd16(va[e]) || odd16(vb[e])) atomicOr(&odd[8 * half + e], 1u << vsub);
        }
    }
    __syncthreads();
    if (mine) {
        if (odd[tok] >> sub & 1) {
#pragma unroll
            for (int e = 0; e < 8; e++) key[0][e] = key[1][e] = (f16)NAN;
        }
        uint8_t* t = p.c.k + paged_tile(p.c, page, kvh, at.tile) * paged_tile_bytes(hd) + paged_key_slot(tok) * 16;
        *(AS_GLOBAL f16x8*)(t + d[0] / 8 * 256) = key[0];
        *(AS_GLOBAL f16x8*)(t + d[1] / 8 * 256) = key[1];
    }
    if (values && fresh) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (odd[8 * half + e] >> vsub & 1) va[e] = vb[e] = (f16)0.f;
        f16* t = (f16*)(p.c.v + paged_tile(p.c, page, vh, at.tile) * paged_tile_bytes(hd)) + (half * hd + dim) * 8;
        if (fresh == 255) {
            *(AS_GLOBAL f16x8*)t = va;
            *(AS_GLOBAL f16x8*)(t + 8) = vb;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (fresh >> e & 1) {
                    gptr(t)[e] = va[e];
                    gptr(t)[8 + e] = vb[e];
                }
        }
    }
}

struct LoadArgs {
    PagedSteps b;
    PagedKV c;
    void *k, *v;
    int64_t k_stride, v_stride;
    int lanes, at_once;
    bool k_whole, v_whole;
};

// Back into rows: a tile a workgroup as above, all its loads under way before the first is used; 4,096 tokens of 8 heads of
// 128 into f16 8.4 us, the bytes of 6.7.
template <typename T>
__global__ __launch_bounds__(kThreads) void paged_load_kernel(LoadArgs p) {
    __shared__ uint32_t odd[16];  // a bit a head of the slice: tokens without a form, whose keys are NaN
    Place at;
    if (!find_place(p.b, blockIdx.x, at)) return;
    const int hd = p.c.hd, tok = threadIdx.x & 15, u = threadIdx.x >> 4;
    const int lane = u % p.lanes, sub = u / p.lanes, h0 = blockIdx.y * p.at_once;
    const int page = paged_page(p.b, p.c, at.s, at.tile);  // (-1: NaN)
    const int kvh = h0 + sub, row = at.row(at.tile * 16 + tok);
    if (threadIdx.x < 16) odd[threadIdx.x] = page < 0 ? ~0u : 0u;
    __syncthreads();
    const int pairs = hd / 2, vsub = threadIdx.x / (2 * pairs), half = (threadIdx.x / pairs) & 1;
    const int dim = 2 * (threadIdx.x % pairs), vh = h0 + vsub;
    const bool values = p.v && vsub < p.at_once && vh < p.c.kv_heads;
    f16x8 va, vb, key[2];
    if (values) {
        const uint8_t* t = p.c.v + paged_tile(p.c, max(page, 0), vh, at.tile) * paged_tile_bytes(hd);
        va = *(const AS_GLOBAL f16x8*)(t + (half * hd + dim) * 16);
        vb = *(const AS_GLOBAL f16x8*)(t + (half * hd + dim) * 16 + 16);
    }
    const bool mine = row >= 0 && sub < p.at_once && kvh < p.c.kv_heads;
    if (mine) {
        const uint8_t* t = p.c.k + paged_tile(p.c, max(page, 0), kvh, at.tile) * paged_tile_bytes(hd) + paged_key_slot(tok) * 16;
#pragma unroll
        for (int i = 0; i < 2; i++) key[i] = *(const AS_GLOBAL f16x8*)(t + (2 * lane + i) * 256);
        if (lane == 0 && odd16(key[0][0])) atomicOr(&odd[tok], 1u << sub);
    }
    __syncthreads();
    if (mine && p.k) {
        T* out = (T*)p.k + row * p.k_stride + (int64_t)kvh * hd + 16 * lane;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = page < 0 ? NAN : (float)key[i][e];
            Lines<T>::store(out + 8 * i, x, p.k_whole);
        }
    }
    if (!values) return;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int r = at.row(at.tile * 16 + 8 * half + e);
        if (r < 0) continue;
        const bool no = odd[8 * half + e] >> vsub & 1;
        store_two((T*)p.v + r * p.v_stride + (int64_t)vh * hd + dim, no ? NAN : (float)va[e], no ? NAN : (float)vb[e],
                  p.v_whole);
    }
}

bool whole(const void* p, int64_t stride, int size) { return !(((uintptr_t)p | (uint64_t)stride * size) & 15); }

// Tiles that the batch can touch: a sequence of n new tokens lies in (n + 30) / 16 at most, and in n.
unsigned tiles_bound(const PagedSteps& b) {
    const int64_t t = ((int64_t)b.rows + 30ll * b.sequences) / 16;
    return (unsigned)(t < b.rows ? t : b.rows);
}

// Two query heads a thread (f16), their angles read once and their rows under way together, from so many values on: 2,048
// tokens of 32/8 heads of 128, written and read back, 17.9 us, of one head a thread 19.2; 4,096 of 32/32 heads of 64 46.7 and
// 46.2; four heads as two.  f32, whose rows are twice as long: 4,096 of 32/8 heads of 128 56.4 and 55.4, of 32/32 heads of 64
// 61.4 and 58.4 (four: 61.6 and 65.0); one.
constexpr int64_t kManyValues = 1 << 21;

template <typename T, int PASSES>
hipError_t launch_append(AppendArgs& p, hipStream_t st) {
    const int per = p.at_once * PASSES;
    p.tiles = (int)tiles_bound(p.b);
    p.blocks = (p.b.rows + 15) / 16;
    p.q_slices = (p.r.heads + per - 1) / per;
    // Where an XCD has several tiles of a sequence: 4,096 tokens as above 33.8 us, a tile's workgroups all over the chip
    // 35.5, f32 of 32/32 heads of 64 57.2 and 61.2.  128 single tokens, each a tile and an eighth of a block: 13.8 and 10.7.
    p.together = p.r.rope && p.blocks >= 64 && p.b.rows >= 8ll * p.b.sequences;
    // (there are at least as many tiles as blocks)
    const int64_t grid = p.together ? (p.tiles + 7ll) / 8 * 8 * (p.kv_slices + p.q_slices)
                                    : (int64_t)p.tiles * p.kv_slices + (int64_t)p.blocks * p.q_slices;
    if (grid * kThreads > UINT32_MAX) return hipErrorInvalidConfiguration;  // (a launch holds no more threads)
    if (p.r.interleaved) paged_append_kernel<T, true, PASSES><<<(unsigned)grid, kThreads, 0, st>>>(p);
    else paged_append_kernel<T, false, PASSES><<<(unsigned)grid, kThreads, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(bool f16_rows, const PagedRows& r, const PagedSteps& b, const PagedKV& c, hipStream_t st) {
    AppendArgs p;
    const int size = f16_rows ? 2 : 4;
    p.r = r;
    p.b = b;
    p.c = c;
    p.lanes = c.hd / 16;
    p.at_once = 16 / p.lanes;
    p.kv_slices = (c.kv_heads + p.at_once - 1) / p.at_once;
    p.q_whole = whole(r.q, r.q_stride, size);
    p.k_whole = whole(r.k, r.k_stride, size);
    p.v_whole = whole(r.v, r.v_stride, size);
    p.out_whole = whole(r.q_out, r.q_out_stride, size);
    p.rope_whole = whole(r.rope, 0, 8);
    if (!f16_rows) return launch_append<float, 1>(p, st);
    const bool many = r.heads > p.at_once && (int64_t)b.rows * r.heads * c.hd >= kManyValues;
    return many ? launch_append<f16, 2>(p, st) : launch_append<f16, 1>(p, st);
}

hipError_t launch_paged_load(bool f16_rows, const PagedSteps& b, const PagedKV& c, void* k, int64_t k_stride, void* v,
                             int64_t v_stride, hipStream_t st) {
    LoadArgs p;
    const int size = f16_rows ? 2 : 4;
    p.b = b;
    p.c = c;
    p.k = k;
    p.v = v;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.lanes = c.hd / 16;
    p.at_once = 16 / p.lanes;
    p.k_whole = whole(k, k_stride, size);
    p.v_whole = whole(v, v_stride, size);
    const dim3 grid(tiles_bound(b), (c.kv_heads + p.at_once - 1) / p.at_once);
    if (f16_rows) paged_load_kernel<f16><<<grid, kThreads, 0, st>>>(p);
    else paged_load_kernel<float><<<grid, kThreads, 0, st>>>(p);
    return hipGetLastError();
}
