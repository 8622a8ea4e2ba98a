// Causal grouped-query attention of a batch of sequences over a cache in pages
// (paged.h), of all positions or of a window with the first ones.
//
// A sequence's query at position p sees positions j <= p with j > p - window (where
// there is a window) or j < sinks; query head h reads KV head h / G.  The (token, head
// of the group) pairs of a KV head are its query columns c = t G + g, the columns of
// the products S^T = K Q^T and O^T = V^T P^T, so that a lane's scores are all of one
// column and its probabilities lie where the second product takes them.
//
// What is read of a batch is bounded here, whatever it holds: a step of keys ends
// with the table, and a page outside the cache is not read; a column that sees a
// position without a page gets NaN.
#include "attn_parts.h"
#include "paged.h"

#include <algorithm>

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// The batch's arrays do not change while a kernel runs: scalar loads where the address is a wave's.
template <typename T>
__device__ __forceinline__ T uniform_load(const T* p) {
    return *(const __attribute__((address_space(4))) T*)p;
}

struct AttnArgs {
    PagedAttention a;
    PagedSteps b;
    PagedKV c;
    int G, most;  // positions that the table can hold
    Divisor by_group;
    float scale_log2;
    float* partials;
    int* counters;
    int wide_grid;   // workgroups of the many-column part
    int wide_parts;  // that a group of its columns may be split into
    int few_columns; // sequences of more query columns are the many-column part's
    int target;      // workgroups that the few-column part aims for
    bool whole_q, whole_out;  // rows that lie on 16 bytes
};

constexpr int kFewCols = 16, kFewStep = 32;
constexpr int kFewLeast = 8;       // steps of a workgroup, where columns are split
constexpr int kFewWaves = 4;       // of a workgroup of the few-column part alone
constexpr int kManyColumns = 64;   // sequences of more columns take the many-column part
constexpr int kMostTarget = kPagedCounters;       // split groups of columns at most
constexpr int kMostSlots = 2 * kMostTarget + 64;  // their parts
constexpr __host__ __device__ int few_slots(int target) { return 2 * target + 64; }  // of them, the few-column part's

// The steps of `step` keys that queries at first..last see: the first tokens' ones, then a range.
struct Steps {
    int first_steps, lo, count;
    __device__ __forceinline__ int operator[](int i) const { return i < first_steps ? i : lo + i - first_steps; }
};
__device__ __forceinline__ Steps steps_of(const AttnArgs& p, int first, int last, int step) {
    Steps r{0, 0, 0};
    if (last < 0) return r;
    if (p.a.window) {
        r.lo = max(0, first - p.a.window + 1) / step;
        r.first_steps = min((int)(((int64_t)p.a.sinks + step - 1) / step), r.lo);
    }
    r.count = r.first_steps + max(0, min(last, p.most - 1) / step + 1 - r.lo);
    return r;
}
// Whether a query at `pos` sees the key, and whether queries at first..last see all of [key0, key1], or any of it.
__device__ __forceinline__ bool sees(const AttnArgs& p, int pos, int key) {
    return key <= pos && (!p.a.window || key > pos - p.a.window || key < p.a.sinks);
}
__device__ __forceinline__ bool all_see(const AttnArgs& p, int first, int last, int key0, int key1) {
    return key1 <= first && (!p.a.window || key0 > last - p.a.window || key1 < p.a.sinks);
}
__device__ __forceinline__ bool any_sees(const AttnArgs& p, int first, int last, int key0, int key1) {
    return key0 <= last && (!p.a.window || key1 > first - p.a.window || key0 < p.a.sinks);
}

// The page of a tile, the same for the whole wave (-1: none).
__device__ __forceinline__ int page_of(const AttnArgs& p, int s, int tile) {
    const int i = tile >> p.c.tiles_log2;
    if (i >= p.b.table_stride) return -1;
    const int id = uniform_load(p.b.table + (int64_t)s * p.b.table_stride + i);
    return (unsigned)id < (unsigned)p.c.pages ? id : -1;
}

// A column's queries as the lane takes them: dims of runs of 8, D apart, from q on.  float: scaled
// into [-1, 1] by a power of two of the largest among the lanes that `over` joins, in two f16 terms, which so
// hold any float32 range.  Returns what the products are to be scaled by for scores in base 2.
template <int N, int D, typename T, typename Over>
__device__ __forceinline__ float load_queries(const T* q, float scale_log2, bool whole, f16x8 (&qh)[N],
                                              f16x8 (&ql)[sizeof(T) == 4 ? N : 1], Over over) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int b = 0; b < N; b++) {
            if (whole) {
                qh[b] = *(const AS_GLOBAL f16x8*)(q + D * b);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) qh[b][e] = gptr(q)[D * b + e];
            }
        }
        return scale_log2;
    } else {
        float x[N][8], most = 0.f;
#pragma unroll
        for (int b = 0; b < N; b++) {
            if (whole) {
                const f32x4 u = *(const AS_GLOBAL f32x4*)(q + D * b), v = *(const AS_GLOBAL f32x4*)(q + D * b + 4);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[b][e] = u[e];
                    x[b][4 + e] = v[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) x[b][e] = gptr(q)[D * b + e];
            }
        }
#pragma unroll
        for (int b = 0; b < N; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(x[b][e]));
        most = over(most);
        // (the bounds keep the scale itself, and a masked score's product with it, a number)
        const int ex = most > 0.f && most < INFINITY ? max(-100, min(__builtin_amdgcn_frexp_expf(most), 120)) : 0;
        const float down = ldexpf(1.f, -ex);
#pragma unroll
        for (int b = 0; b < N; b++) {
            f16x2 hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float u = x[b][2 * i] * down, v = x[b][2 * i + 1] * down;
                hi[i] = round2(u, v);
                lo[i] = round2(rest_low(hi[i], u), rest_high(hi[i], v));
            }
            qh[b] = frag(hi[0], hi[1], hi[2], hi[3]);
            ql[b] = frag(lo[0], lo[1], lo[2], lo[3]);
        }
        return ldexpf(scale_log2, ex);
    }
}
// 1 / sum of a column's probabilities, 0 where it sees nothing, NaN where it sees a position past the table.
__device__ __forceinline__ float inverse(float l, bool past) { return past ? NAN : l == 0.f ? 0.f : 1.f / l; }

// ------------------------------------------------------------------ few columns
// Sequences of a few query columns, single tokens above all: bound by the pages' bytes.  16 columns of a KV head are a
// workgroup's, the products 16x16x32 of which a single token of G query heads uses G columns: the matrix unit has room for
// that, and nothing is read twice.  Each wave has steps of 32 keys of its own, whose tiles go from memory straight into the
// products' operands, one step ahead; LDS would only add a trip.  The steps of one group of columns are split over
// workgroups, so that all of them have like shares of the batch's work whatever its lengths, and the last one to arrive
// joins the parts.
//
// 64 sequences of 32/8 heads of 128, 868 MB of pages, f16: 162 us, 5.3 TB/s (a copy reaches 5.0, a sum 5.8), matrix unit 4%
// busy; one of 131,072 positions 99 us, 5.4 TB/s; 24 sequences with windows, 126 MB: 29.1 us, 4.3 TB/s, of which 5 are the
// launch, the look for the work and the join.  A token of 9/3 heads of 64 at 2,000 positions: 8.1 us, a chain of such trips.

// A workgroup's work: a group of 16 columns of sequence s, part sp of `splits`.
struct FewItem {
    int s, kvh, group, sp, splits, counter, slot;
    PagedSeq seq;
};
struct FewCount {
    int groups, steps;  // of a sequence, of 16 columns of a KV head each
};
__device__ __forceinline__ FewCount few_count(const AttnArgs& p, const PagedSeq& q) {
    const int64_t cols = (int64_t)q.n * p.G;
    if (q.n == 0 || cols > p.few_columns) return {0, 0};
    return {(int)((cols + kFewCols - 1) / kFewCols), steps_of(p, q.length - q.n, q.length - 1, kFewStep).count};
}
// Workgroup `w` of the few-column part, by a whole wave; splits = 0 past the last.
__device__ __forceinline__ FewItem few_find(const AttnArgs& p, int w) {
    const int lane = __lane_id(), S = p.b.sequences, KVH = p.c.kv_heads;
    auto seq_of = [&](int s0) { return s0 + lane < S ? paged_seq(p.b, s0 + lane) : PagedSeq{0, 0, 0}; };
    // steps a workgroup: all the batch's over the workgroups aimed for.  (float: the same sum in every wave)
    const PagedSeq front = seq_of(0);  // (all of a batch of up to 64)
    const FewCount front_count = few_count(p, front);
    float all = (float)front_count.groups * (float)front_count.steps, groups_all = (float)front_count.groups;
    for (int s0 = 64; s0 < S; s0 += 64) {
        const FewCount f = few_count(p, seq_of(s0));
        all += (float)f.groups * (float)f.steps;
        groups_all += (float)f.groups;
    }
    all = wave_sum(all) * (float)KVH * 1.0001f;
    const float target = (float)p.target;
    int share = (int)fminf(all / target + 1.f, 1e9f);
    if (share <= kFewLeast) {
        share = kFewLeast;
    } else if (groups_all = wave_sum(groups_all) * (float)KVH; 2.f * groups_all <= target) {
        // Last parts that are not full make these up to groups_all more than aimed for, and a CU that has one more ends last.
        // So the least share that makes no more (of a batch of more than 64 sequences, one that makes no more): 8 of 32/8 heads
        // of 128 at up to 16,000 47 us and not 58, two at up to 60,000 76 and 99.  Of more groups that would leave too few to
        // split: 96 sequences of 8/4 heads of 64, 384 groups of 512, 46 and not 37.6.
        int most = max(share, (int)fminf(all / (target - groups_all) + 1.f, 1e9f));
        for (int i = 0; i < 5 && share < most && S <= 64; i++) {
            const int mid = (share + most) >> 1;
            const float parts = ceilf((float)front_count.steps * (0.999999f / (float)mid));
            const bool fits = wave_sum((float)front_count.groups * parts) * (float)KVH <= target;
            most = fits ? mid : most;
            share = fits ? share : mid + 1;
        }
        share = most;
    }
    FewItem r{0, 0, 0, 0, 0, 0, 0, {0, 0, 0}};
    for (int s0 = 0; s0 < S; s0 += 64) {
        PagedSeq q = front;
        FewCount f = front_count;
        if (s0) {
            q = seq_of(s0);
            f = few_count(p, q);
        }
        const int groups = f.groups * KVH, splits = max(1, (f.steps + share - 1) / share);
        const int mine = groups * splits, upto = wave_scan(mine);
        const int joint = splits > 1 ? groups : 0, joint_to = wave_scan(joint);
        const int parts = joint * splits, parts_to = wave_scan(parts);
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > w);
        if (past) {
            const int l = __builtin_ctzll(past);
            auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
            const int i = w - of(upto - mine);
            r.s = s0 + l;
            r.seq = {of(q.row0), of(q.n), of(q.length)};
            r.splits = of(splits);
            r.kvh = i % KVH;
            r.sp = i / KVH % r.splits;
            r.group = i / KVH / r.splits;
            const int at = r.group * KVH + r.kvh;
            r.counter += of(joint_to - joint) + at;
            r.slot += of(parts_to - parts) + at * r.splits;
            // (only row ranges that overlap could have more)
            if (r.splits > 1 && (r.counter >= p.target || r.slot + r.splits > few_slots(p.target))) r.splits = 0;
            return r;
        }
        w -= __builtin_amdgcn_readlane(upto, 63);
        r.counter += __builtin_amdgcn_readlane(joint_to, 63);
        r.slot += __builtin_amdgcn_readlane(parts_to, 63);
    }
    return r;
}

template <int NB>
struct FewTile {
    f16x8 k[2][NB], v[2 * NB];
    int none;  // bits of the step's two tiles: those that have no page
};
template <int NB>
constexpr int few_lds(int waves) {
    return waves * kFewCols * (32 * NB + 4 + 2) * 4;
}

template <int NB, typename T>
__device__ __forceinline__ void few_part(const AttnArgs& p, int w, uint8_t* lds) {
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int HD = 32 * NB, TILE = paged_tile_bytes(HD);
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15, waves = blockDim.x >> 6;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const FewItem it = few_find(p, w);
    if (it.splits == 0) return;  // (the same for the whole workgroup)
    const PagedSeq& seq = it.seq;
    const int col0 = it.group * kFewCols, cols = min(seq.n * p.G - col0, kFewCols), pos0 = seq.length - seq.n;
    const int first = pos0 + p.by_group(col0), last = pos0 + p.by_group(col0 + cols - 1);
    const Steps steps = steps_of(p, first, last, kFewStep);
    const int per = steps.count / it.splits, more = steps.count - per * it.splits;
    const int t0 = per * it.sp + min(it.sp, more), t1 = t0 + per + (it.sp < more);

    const uint8_t *kbase = p.c.k + (g * 16 + (lane & 7)) * 16, *vbase = p.c.v + ((g & 1) * HD + c16) * 16;
    constexpr bool AHEAD = NB <= 4;  // two tiles in registers, where those allow; else one, refilled as it is used
    struct Place {
        const uint8_t *k, *v;
        int none;
    };
    auto place = [&](int i) {
        const int tile = 2 * steps[min(i, t1 - 1)];  // (past the last step: that one, unused)
        const int pa = page_of(p, it.s, tile), pb = p.c.tiles_log2 ? pa : page_of(p, it.s, tile + 1);
        const int64_t a = paged_tile(p.c, max(pa, 0), it.kvh, tile) * TILE;
        const int64_t b = paged_tile(p.c, max(pb, 0), it.kvh, tile + 1) * TILE;
        return Place{kbase + (lane & 8 ? b : a), vbase + (lane & 32 ? b : a), (pa < 0) | (pb < 0) << 1};
    };
    auto load_k = [&](FewTile<NB>& x, const Place& at) {
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int c = 0; c < NB; c++) x.k[s][c] = *(const AS_GLOBAL f16x8*)(at.k + c * 1024 + s * 128);
    };
    auto load_v = [&](FewTile<NB>& x, const Place& at) {
        x.none = at.none;
#pragma unroll
        for (int d = 0; d < 2 * NB; d++) x.v[d] = *(const AS_GLOBAL f16x8*)(at.v + d * 256);
    };
    auto load = [&](FewTile<NB>& x, int i) {
        const Place at = place(i);
        load_k(x, at);
        load_v(x, at);
    };
    FewTile<NB> xa, xb;
    int j = t0 + wave;
    if (j < t1) load(xa, j);

    f16x8 qh[NB], ql[EXACT ? NB : 1];
    const int col = col0 + min(c16, cols - 1), t = p.by_group(col), pos = pos0 + t;
    const T* q = (const T*)p.a.q + (int64_t)(seq.row0 + t) * p.a.q_stride + (int64_t)(it.kvh * p.G + col - t * p.G) * HD + 8 * g;
    const float sc = load_queries<NB, 32, T>(q, p.scale_log2, p.whole_q, qh, ql, [](float x) {
        return xor32_combine(xor16_combine(x, MaxOp()), MaxOp());
    });
    float m = -INFINITY, l = 0.f;
    f32x4 o[2 * NB];
#pragma unroll
    for (int d = 0; d < 2 * NB; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto step = [&](FewTile<NB>& x, int i) {
        f32x4 sa[2];  // S(key 8 g + 4 s + r, column c16)
#pragma unroll
        for (int s = 0; s < 2; s++) {
            sa[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NB; c++) {
                sa[s] = mfma(x.k[s][c], qh[c], sa[s]);
                if constexpr (EXACT) sa[s] = mfma(x.k[s][c], ql[c], sa[s]);
            }
        }
        Place next;
        if constexpr (!AHEAD) {
            next = place(i + waves);
            load_k(x, next);
        }
        const int key0 = steps[i] * kFewStep;
        if (x.none || !all_see(p, first, last, key0, key0 + kFewStep - 1)) {
            const bool none = x.none >> (g >> 1) & 1;
            uint32_t keep[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int key = key0 + 8 * g + e;
                if (none) sa[e >> 2][e & 3] = NAN;
                if (!sees(p, pos, key)) sa[e >> 2][e & 3] = -INFINITY;
                if (!none && any_sees(p, first, last, key, key)) keep[e >> 1] |= 0xFFFFu << (16 * (e & 1));
            }
            // positions that may never have been written: values of 0, since 0 times what lies there may be NaN
#pragma unroll
            for (int d = 0; d < 2 * NB; d++) {
                typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
                u32x4 u = __builtin_bit_cast(u32x4, x.v[d]);
#pragma unroll
                for (int e = 0; e < 4; e++) u[e] &= keep[e];
                x.v[d] = __builtin_bit_cast(f16x8, u);
            }
        }
        float mx = sa[0][0];
#pragma unroll
        for (int e = 1; e < 8; e++) mx = fmaxf(mx, sa[e >> 2][e & 3]);
        mx = xor32_combine(xor16_combine(mx, MaxOp()), MaxOp());
        const float mn = fmaxf(m, mx * sc);  // (sc > 0)
        const float mref = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - mref), base = exponent_base(sa, mx, mref, sc);
        f16x2 ph[4], pl[EXACT ? 4 : 1];
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a = __builtin_amdgcn_exp2f(fmaf(sa[e >> 1][2 * (e & 1)], sc, base));
            const float b = __builtin_amdgcn_exp2f(fmaf(sa[e >> 1][2 * (e & 1) + 1], sc, base));
            sum += a + b;
            ph[e] = round2(a, b);
            if constexpr (EXACT) pl[e] = round2(rest_low(ph[e], a), rest_high(ph[e], b));
        }
        if (__builtin_amdgcn_ballot_w64(m != mn)) {
#pragma unroll
            for (int d = 0; d < 2 * NB; d++) o[d] *= alpha;
            l *= alpha;
            m = mn;
        }
        l += sum;
        const f16x8 pf = frag(ph[0], ph[1], ph[2], ph[3]);
#pragma unroll
        for (int d = 0; d < 2 * NB; d++) {
            o[d] = mfma(x.v[d], pf, o[d]);
            if constexpr (EXACT) o[d] = mfma(x.v[d], frag(pl[0], pl[1], pl[2], pl[3]), o[d]);
        }
        if constexpr (!AHEAD) load_v(x, next);
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
        for (; j < t1; j += waves) step(xa, j);
    }

    // o[d][r] = O(column c16, dim 16 d + 4 g + r); the waves' results meet in LDS
    float (*xo)[kFewCols][HD + 4] = (float (*)[kFewCols][HD + 4])lds;
    float (*xml)[2][kFewCols] = (float (*)[2][kFewCols])(lds + waves * kFewCols * (HD + 4) * 4);
    l = xor32_combine(xor16_combine(l, AddOp()), AddOp());
#pragma unroll
    for (int d = 0; d < 2 * NB; d++) *(f32x4*)&xo[wave][c16][16 * d + 4 * g] = o[d];
    if (g == 0) {
        xml[wave][0][c16] = m;
        xml[wave][1][c16] = l;
    }
    __syncthreads();
    const int items = cols * (HD / 2), had = max(1, min(waves, t1 - t0));  // (a wave without a step adds nothing)
    float* const part = p.partials + (int64_t)it.slot * kFewCols * (HD + 2);
    auto put = [&](int c, int d, float a, float b, float sum) {
        const int u = p.by_group(col0 + c), h = it.kvh * p.G + col0 + c - u * p.G;
        const float inv = inverse(sum, pos0 + u >= p.most);
        T* out = (T*)p.a.out + (int64_t)(seq.row0 + u) * p.a.out_stride + (int64_t)h * HD + d;
        gptr(out)[0] = (T)(a * inv);
        gptr(out)[1] = (T)(b * inv);
    };
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        const int c = i / (HD / 2), d = 2 * (i % (HD / 2));
        float top = xml[0][0][c];
        for (int v = 1; v < had; v++) top = fmaxf(top, xml[v][0][c]);
        float sum = 0.f, a = 0.f, b = 0.f;
        for (int v = 0; v < had; v++) {
            const float f = join_weight(xml[v][0][c], top);
            sum += f * xml[v][1][c];
            a += f * xo[v][c][d];
            b += f * xo[v][c][d + 1];
        }
        if (it.splits == 1) {
            put(c, d, a, b, sum);
        } else {
            float* x = part + (int64_t)(c * it.splits + it.sp) * (HD + 2);
            put2(x + 2 + d, a, b);
            if (d == 0) put2(x, top, sum);
        }
    }
    if (it.splits == 1) return;
    // the last part of the columns to arrive joins them all
    int* arrived = (int*)lds;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        int* counter = p.counters + it.counter;
        *arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == it.splits - 1;
        if (*arrived) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    const bool mine = *arrived;
    __syncthreads();  // (*arrived is read; the joining uses its place)
    if (!mine) return;
    auto at = [&](int c) { return part + (int64_t)c * it.splits * (HD + 2); };
    if (2 * items > (int)blockDim.x) {
        for (int i = threadIdx.x; i < items; i += blockDim.x) {
            const int c = i / (HD / 2), d = 2 * (i % (HD / 2));
            const Joined r = join<8>(at(c), HD, d, 0, 1, it.splits);
            put(c, d, r.a, r.b, r.l);
        }
        return;
    }
    const int groups = blockDim.x / items, group = threadIdx.x / items, i = threadIdx.x - group * items;
    const int c = i / (HD / 2), d = 2 * (i % (HD / 2));
    const Joined r = join_groups<8>(at(c), HD, d, group, groups, items, i, it.splits, (float4*)lds);
    if (group == 0) put(c, d, r.a, r.b, r.l);
}

template <int NB, typename T>
__global__ __launch_bounds__(64 * kFewWaves) void paged_few_kernel(AttnArgs p) {
    extern __shared__ __align__(16) uint8_t lds[];
    few_part<NB, T>(p, blockIdx.x, lds);
}

// ------------------------------------------------------------------ many columns
// 32 CW query columns a workgroup, 32 a wave, products 32x32x16; the keys' tiles go by DMA into LDS as they lie in memory and
// are read as operands without bank conflicts (16 bytes a lane in lane order).  Steps are of 32 keys, and a wave is one ahead
// with its scores: the products of step i + 1's keys run beside the exponentials of step i, those of step i's values beside the
// maximum of step i + 1's scores.  A stage of STEPS steps has one barrier; while its values and the keys of the step ahead of
// each are at work, the next one's are under way.  SETS sets of CW waves take consecutive ranges of the steps and join through
// LDS at the end; those of four sets may be workgroups' parts of the steps, which the last one to arrive joins, as the
// few-column part's are.  KV heads are the fastest index of the grid, so that the workgroups of 8 of them have an XCD's L2
// each for their pages.
//
// Bound by the two units that share a SIMD's issue.  4,096 f16 tokens of 32/8 heads of 128: 157-171 us on different cards,
// 800-870 TFLOP/s (a library product of 8,192: 1,176), matrix unit 41% busy and vector unit 44% of the cycles, 7.4 vector
// instructions a matrix one, no bank conflicts; without its LDS reads it would take 0.93 of that, without its exponentials
// 0.91, without its loads 0.85, with none of them 0.73.  float32 has two products for each of these (two f16 terms of the
// queries, two of the probabilities): three chunks of 2,500 tokens with windows of 1,024, 24/8 heads of 128, 185-199 us, 78
// GFLOP once and 156 as they are done, 790-840 TFLOP/s, matrix unit 50% busy.
template <int NB, int CW, int SETS>
struct Wide {
    static constexpr int HD = 32 * NB, TILE = paged_tile_bytes(HD), KEYS = 32, STEP = 2 * TILE;
    static constexpr int STEPS = NB <= 4 && SETS <= 2 ? 2 : 1;  // of a stage
    static constexpr int COLS = 32 * CW;
    static constexpr bool SPLIT = SETS == 4 && NB >= 3;  // the steps over workgroups, where columns make too few
    static constexpr int JOIN = SETS > 1 ? COLS * (HD + 4) * 4 + COLS * 8 : 0;  // a set's outputs and statistics
    static constexpr int SIDE = 2 * STEPS * STEP;  // two stages of keys, or of values
    static constexpr int RING = 2 * SETS * SIDE;
    static constexpr int FEW = few_lds<NB>(CW * SETS);
    static constexpr int LDS = RING > JOIN ? (RING > FEW ? RING : FEW) : (JOIN > FEW ? JOIN : FEW);
    static constexpr bool FITS = LDS <= 160 << 10;
};
// P enters the products as P 2^9 and a column's reference follows its maximum only when that is 2^6 past it, which
// few steps are.  By their difference, exact for neighbouring numbers: m + 6 rounds to m + 8 where those are 4 or 8 apart, and
// P would be past f16.  In f16 P is one term, rounded by 2^-11 at most, here and in the few-column part (2^14 there): rows of
// f16 are rounded by as much at the end, so that a prompt's error against 64 bits is 2.5e-4 of its norm where that rounding alone
// is 2.1e-4; a second term is a second product for every value.
constexpr float kWideLog2P = 9.f, kSlack = 6.f;
// Parts of the steps: a part and the joining cost about 6 us, so that 600 positions (19 steps) stay whole: 18 us, in two 25.
constexpr int kWideLeast = 16;  // steps of a part

template <int NB, int CW, int SETS, typename T>
__device__ __forceinline__ void wide_part(const AttnArgs& p, uint8_t* lds) {
    typedef Wide<NB, CW, SETS> W;
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int HD = W::HD, TILE = W::TILE, KEYS = W::KEYS, U = W::STEPS;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, half = lane >> 5, c32 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), set = wave / CW, wl = wave % CW;
    const int KVH = p.c.kv_heads, kvh = blockIdx.x % KVH, w = blockIdx.x / KVH;
    const int sp = W::SPLIT ? w % p.wide_parts : 0, item = W::SPLIT ? w / p.wide_parts : w;
    const PagedItem it = paged_find(p.b, item, [&](const PagedSeq& q) {
        const int64_t cols = (int64_t)q.n * p.G;
        return cols > p.few_columns ? (int)((cols + W::COLS - 1) / W::COLS) : 0;
    });
    if (it.s < 0) return;
    const int s = it.s;
    const PagedSeq seq = it.seq;
    const int cols = seq.n * p.G, pos0 = seq.length - seq.n;
    // a sequence's last columns first: they see the most keys
    const int col0 = ((cols + W::COLS - 1) / W::COLS - 1 - it.i) * W::COLS;
    const int first = pos0 + p.by_group(col0), last = pos0 + p.by_group(min(col0 + W::COLS, cols) - 1);
    const int wcol0 = min(col0 + wl * 32, cols - 1);  // the wave's columns
    const int w_first = pos0 + p.by_group(wcol0), w_last = pos0 + p.by_group(min(wcol0 + 31, cols - 1));
    const Steps steps = steps_of(p, first, last, KEYS);
    // the workgroup's part of the steps, and the set's of those
    const int parts = W::SPLIT ? max(1, min(p.wide_parts, steps.count / kWideLeast)) : 1;
    const int each = (steps.count + parts - 1) / parts, end = min(steps.count, (sp + 1) * each);
    if (W::SPLIT && sp >= parts) return;
    const int per = max(0, end - sp * each + SETS - 1) / SETS, f0 = sp * each + set * per;
    // the wave's steps: of its set's those that one of its columns sees
    const int count = max(0, min(min(end, steps_of(p, first, w_last, KEYS).count) - f0, per));

    const int col = min(col0 + wl * 32 + c32, cols - 1), t = p.by_group(col), pos = pos0 + t;
    f16x8 qh[2 * NB], ql[EXACT ? 2 * NB : 1];
    const T* q = (const T*)p.a.q + (int64_t)(seq.row0 + t) * p.a.q_stride + (int64_t)(kvh * p.G + col - t * p.G) * HD + 8 * half;
    const float sc = load_queries<2 * NB, 16, T>(q, p.scale_log2, p.whole_q, qh, ql, [](float x) {
        return xor32_combine(x, MaxOp());
    });
    // (the queries are here before the loop: a wait for them inside it would wait for the tiles under way)
#pragma unroll
    for (int c = 0; c < 2 * NB; c++) {
        asm volatile("" : "+v"(qh[c]));
        if constexpr (EXACT) asm volatile("" : "+v"(ql[c]));
    }
    float m = -INFINITY, l = 0.f, base = 0.f;
    f32x16 o[NB];
#pragma unroll
    for (int d = 0; d < NB; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.f;

    // Whether a position that one of the workgroup's columns sees has no page (then every step looks again).
    bool holes = false;
    if (steps.count) {
        auto missing = [&](int from, int to) {
            for (int i = (from >> 4 >> p.c.tiles_log2) + lane; i <= to >> 4 >> p.c.tiles_log2; i += 64)
                if (i < p.b.table_stride)
                    holes |= (unsigned)gptr(p.b.table)[(int64_t)s * p.b.table_stride + i] >= (unsigned)p.c.pages;
        };
        missing(p.a.window ? max(0, first - p.a.window + 1) : 0, min(last, p.most - 1));
        if (steps.first_steps) missing(0, min(p.a.sinks - 1, min(last, p.most - 1)));
        holes = __builtin_amdgcn_ballot_w64(holes);
    }
    // Whether the second tile of the step that `last` is in has none.  (Further steps are not run, and where `last` is in that
    // tile itself the search above has found it.)
    const bool behind = last >= 0 && page_of(p, s, (last / 16) | 1) < 0;
    // The set's steps i that are plain: all of i + 1 is seen by all columns of the wave, and all of i by one of the workgroup's.
    const int plain0 = holes ? INT32_MAX
                       : p.a.window ? steps.first_steps + (last >= p.a.window ? (last - p.a.window) / KEYS + 1 : 0) - steps.lo - f0
                                    : -f0;
    const int plain1 = min(count, steps.first_steps + max(0, w_first + 1) / KEYS - steps.lo - f0) - 1;

    // keys of step i at ring + ((i - 1) % 2U) STEP, values of step i at ring + SIDE + (i % 2U) STEP
    uint8_t* const ring = lds + set * 2 * W::SIDE;
    const uint32_t ring_at = lds_addr(ring);
    // the wave's share of a stage's loads: tiles u0, u0 + CW, ... and KB p0, p0 + P, ... of them
    constexpr int TILES = 2 * U, MINE = TILES > CW ? TILES / CW : 1, P = CW > TILES ? CW / TILES : 1;
    const int u0 = wl % TILES, p0 = wl / TILES;
    struct Places {
        int64_t at[MINE];
    };
    auto places = [&](int i) {  // of the stage that begins with step i (past the last step: that one, unused)
        Places r;
#pragma unroll
        for (int k = 0; k < MINE; k++) {
            const int u = u0 + CW * k, tile = 2 * steps[max(0, min(f0 + i + (u >> 1), steps.count - 1))] + (u & 1);
            r.at[k] = paged_tile(p.c, max(page_of(p, s, tile), 0), kvh, tile) * TILE;
        }
        return r;
    };
    auto fetch = [&](const uint8_t* from, const Places& r, uint32_t to) {
#pragma unroll
        for (int k = 0; k < MINE; k++)
#pragma unroll
            for (int part = 0; part < NB; part += P)
                if (P == 1 || NB % P == 0 || part + p0 < NB)
                    dma16s(from + r.at[k] + (part + p0) * 1024, lane * 16, to + (u0 + CW * k) * TILE + (part + p0) * 1024);
    };
    const uint32_t k_lane = (c32 >> 4) * TILE + (half * 16 + (c32 & 15)) * 16, v_lane = W::SIDE + (half * HD + c32) * 16;
    // S(key 16 (r / 8) + 8 half + r % 8, column c32) of step i
    auto scores = [&](int i, f32x16& x) {
        const uint8_t* kb = ring + ((i - 1) & (2 * U - 1)) * W::STEP + k_lane;
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] = 0.f;
#pragma unroll
        for (int c = 0; c < 2 * NB; c++) {
            const f16x8 a = *(const f16x8*)(kb + c * 512);
            x = mfma32(a, qh[c], x);
            if constexpr (EXACT) x = mfma32(a, ql[c], x);
        }
    };
    // Hides what a column does not see.
    auto hide = [&](int i, f32x16& x) {
        const int key0 = steps[f0 + i] * KEYS;
        if (!holes && all_see(p, w_first, w_last, key0, key0 + KEYS - 1)) return;
        if (holes) {
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (page_of(p, s, key0 / 16 + u) < 0)
#pragma unroll
                    for (int r = 0; r < 8; r++) x[8 * u + r] = NAN;
        }
        if (!p.a.window) {
            const int at = pos - key0 - 8 * half;  // the lane's key 16 u + r is seen up to this one
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (16 * (r >> 3) + (r & 7) > at) x[r] = -INFINITY;
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (!sees(p, pos, key0 + 8 * half + 16 * (r >> 3) + (r & 7))) x[r] = -INFINITY;
        }
    };
    // Values of 0 at positions that no column of the workgroup sees, where they may never have been written, be another
    // sequence's or stand for a page that there is not: 0 times what lies there may be NaN.  (The waves of a set write the
    // same.)  Positions behind `last` that are the sequence's and have a page are left: cleared too, three chunks of 2,500
    // f32 tokens with windows took 193 us and not 187.
    auto clear = [&](int i) {
        const int key0 = steps[f0 + i] * KEYS, key1 = key0 + KEYS - 1;
        if (!holes && key1 < min(seq.length, p.most) && (!p.a.window || key0 > first - p.a.window || key1 < p.a.sinks) &&
            !(behind && key1 > last))
            return;
        for (int u = 0; u < 2; u++) {
            const bool none = holes && page_of(p, s, key0 / 16 + u) < 0;
            for (int c = lane; c < 2 * HD; c += 64) {
                uint32_t keep[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int key = key0 + 16 * u + (c >= HD ? 8 : 0) + e;
                    if (!none && key < p.most && any_sees(p, first, last, key, key)) keep[e >> 1] |= 0xFFFFu << (16 * (e & 1));
                }
                u32x4* at = (u32x4*)(ring + W::SIDE + (i & (2 * U - 1)) * W::STEP + u * TILE + c * 16);
                u32x4 v = *at;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] &= keep[e];
                *at = v;
            }
        }
    };
    // The reference follows the scores to come, where they are past it.
    bool large = false;  // (a column's reference is: exponent_base has something to do)
    auto follow = [&](f32x16& x) {
#pragma clang fp contract(off)  // (mn - m of the rounded mn, as exponent_base has it)
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < 16; e++) mx = fmaxf(mx, x[e]);
        mx = xor32_combine(mx, MaxOp());
        const float mn = mx * sc;  // (sc > 0)
        if (__builtin_amdgcn_ballot_w64(mn - m > kSlack)) {
            const float top = fmaxf(m, mn), alpha = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
#pragma unroll
            for (int d = 0; d < NB; d++) o[d] *= alpha;
            l *= alpha;
            m = top;
        }
        f32x16(&y)[1] = reinterpret_cast<f32x16(&)[1]>(x);
        base = exponent_base(y, mx, m == -INFINITY ? 0.f : m, sc, kWideLog2P);
        large = __builtin_amdgcn_ballot_w64(fabsf(m) > kLargeScore && m != -INFINITY);
    };
    // Step i, its scores in x; those of step i + 1 into next.  Slots of a product (two in float32), the next operand's
    // read and what runs beside it, in this order: operands AHEAD slots before their use, exponentials beside the keys'
    // products, maxima beside the values'.
    auto step = [&](int i, f32x16& x, f32x16& next) {
        const bool plain = i >= plain0 && i < plain1;
        constexpr int SLOTS = 2 * NB, AHEAD = NB == 1 ? 2 : 4, RING = AHEAD + 1;
        f16x2 ph[8], pl[EXACT ? 8 : 1];
        float sum[2] = {0.f, 0.f}, part[5];
        uint64_t past = 0;
        auto at = [](int k) { return min(k, SLOTS - 1); };
        if (!plain) clear(i);
        const uint8_t* kb = ring + (i & (2 * U - 1)) * W::STEP + k_lane;
        const uint8_t* vb = ring + (i & (2 * U - 1)) * W::STEP + v_lane;
        f16x8 fr[RING];
        auto read = [&](int k) {  // value operands tile by tile
            fr[k % RING] = *(const f16x8*)(k < SLOTS ? kb + k * 512 : vb + (k - SLOTS) / NB * TILE + (k - SLOTS) % NB * 512);
        };
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < AHEAD; k++) read(k);
#pragma unroll
        for (int r = 0; r < 16; r++) next[r] = 0.f;
#pragma unroll
        for (int k = 0; k < SLOTS; k++) {
            read(k + AHEAD);
            next = mfma32(fr[k % RING], qh[k], next);
            if constexpr (EXACT) next = mfma32(fr[k % RING], ql[k], next);
#pragma unroll
            for (int e = k * 8 / SLOTS; e < (k + 1) * 8 / SLOTS; e++) {
                const float a = __builtin_amdgcn_exp2f(fmaf(x[2 * e], sc, base));
                const float b = __builtin_amdgcn_exp2f(fmaf(x[2 * e + 1], sc, base));
                sum[0] += a;
                sum[1] += b;
                ph[e] = round2(a, b);
                if constexpr (EXACT) pl[e] = round2(rest_low(ph[e], a), rest_high(ph[e], b));
            }
            asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int k = 0; k < SLOTS; k++) {
            const int u = k / NB, d = k % NB;
            if (k + AHEAD < SLOTS) read(SLOTS + k + AHEAD);
            const f16x8 v = fr[(SLOTS + k) % RING];
            o[d] = mfma32(v, frag(ph[4 * u], ph[4 * u + 1], ph[4 * u + 2], ph[4 * u + 3]), o[d]);
            if constexpr (EXACT) o[d] = mfma32(v, frag(pl[4 * u], pl[4 * u + 1], pl[4 * u + 2], pl[4 * u + 3]), o[d]);
            if (k == 0) l += sum[0] + sum[1];
            // the largest score, and whether it is past the reference: a part of the chain a slot
            if (k == at(1)) {
#pragma unroll
                for (int e = 0; e < 5; e++) part[e] = fmaxf(fmaxf(next[3 * e], next[3 * e + 1]), next[3 * e + 2]);
            }
            if (k == at(2)) part[0] = fmaxf(fmaxf(fmaxf(part[0], part[1]), part[2]), fmaxf(fmaxf(part[3], part[4]), next[15]));
            if (k == at(3)) part[0] = xor32_combine(part[0], MaxOp());
            if (k == at(4)) past = __builtin_amdgcn_ballot_w64(part[0] * sc - m > kSlack);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_expect(!plain || large || past, 0)) {
            if (i + 1 >= count) return;
            if (!plain) hide(i + 1, next);
            follow(next);
        }
    };
    if (per > 0) {  // (the same for the whole workgroup)
        const Places a = places(1 - U);  // keys of step 0, at the end of a stage
        fetch(p.c.k, a, ring_at + U * W::STEP);
        Places kp = places(1), vp = places(0);
        wait_stage_barrier<0>();
        fetch(p.c.k, kp, ring_at);
        fetch(p.c.v, vp, ring_at + W::SIDE);
        kp = places(1 + U);
        vp = places(U);
        f32x16 x, y;
        if (count > 0) {
            scores(0, x);
            hide(0, x);
            follow(x);
        }
        auto stage = [&](int i) {  // that begins with step i: the next one's loads on their way
            wait_stage_barrier<0>();
            if (i + U >= per) return;
            const uint32_t to = ring_at + ((i + U) & (2 * U - 1)) * W::STEP;
            fetch(p.c.k, kp, to);
            fetch(p.c.v, vp, to + W::SIDE);
            kp = places(i + 1 + 2 * U);
            vp = places(i + 2 * U);
        };
        for (int i = 0; i < per; i += 2) {
            stage(i);
            if (i < count) step(i, x, y);
            if (U == 1) {
                if (i + 1 >= per) break;
                stage(i + 1);
            }
            if (i + 1 < count) step(i + 1, y, x);
        }
    }
    // l: half the keys in either half of the wave
    l = xor32_combine(l, AddOp());
    if constexpr (SETS > 1) {
        float* xo = (float*)lds;
        float* xml = xo + W::COLS * (HD + 4);
        const int c = wl * 32 + c32;
        for (int other = 1; other < SETS; other++) {
            __syncthreads();
            if (set == other) {
#pragma unroll
                for (int d = 0; d < NB; d++)
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        *(f32x4*)&xo[c * (HD + 4) + 32 * d + 8 * u + 4 * half] =
                            f32x4{o[d][4 * u], o[d][4 * u + 1], o[d][4 * u + 2], o[d][4 * u + 3]};
                if (half == 0) {
                    xml[2 * c] = m;
                    xml[2 * c + 1] = l;
                }
            }
            __syncthreads();
            if (set == 0) {
                const float mo = xml[2 * c], top = fmaxf(m, mo), fa = join_weight(m, top), fb = join_weight(mo, top);
                m = top;
                l = l * fa + xml[2 * c + 1] * fb;
#pragma unroll
                for (int d = 0; d < NB; d++)
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const f32x4 y = *(const f32x4*)&xo[c * (HD + 4) + 32 * d + 8 * u + 4 * half];
#pragma unroll
                        for (int r = 0; r < 4; r++) o[d][4 * u + r] = o[d][4 * u + r] * fa + y[r] * fb;
                    }
            }
        }
        if (parts == 1 && set) return;
    }
    if constexpr (W::SPLIT)
        if (parts > 1) {
            // the last part of the columns to arrive joins them all
            const int group = item * KVH + kvh, here = min(cols - col0, W::COLS), c = wl * 32 + c32;
            const int64_t slot = few_slots(p.target) + (int64_t)group * p.wide_parts * (W::COLS / kFewCols);
            float* const part = p.partials + slot * kFewCols * (HD + 2);
            float* xo = (float*)lds;  // rows by way of LDS, so that a wave's stores lie side by side
            float* xml = xo + W::COLS * (HD + 4);
            if (set == 0) {
#pragma unroll
                for (int d = 0; d < NB; d++)
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        *(f32x4*)&xo[c * (HD + 4) + 32 * d + 8 * u + 4 * half] =
                            f32x4{o[d][4 * u], o[d][4 * u + 1], o[d][4 * u + 2], o[d][4 * u + 3]};
                if (half == 0) {
                    xml[2 * c] = m;
                    xml[2 * c + 1] = l;
                }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < here * (HD / 2); i += 64 * CW * SETS) {
                const int jc = i / (HD / 2), d = 2 * (i % (HD / 2));
                float* x = part + (int64_t)(jc * parts + sp) * (HD + 2);
                put2(x + 2 + d, xo[jc * (HD + 4) + d], xo[jc * (HD + 4) + d + 1]);
                if (d == 0) put2(x, xml[2 * jc], xml[2 * jc + 1]);
            }
            int* arrived = (int*)lds;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (threadIdx.x == 0) {
                int* counter = p.counters + p.target + group;
                *arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
                if (*arrived) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (!*arrived) return;
            for (int i = threadIdx.x; i < here * (HD / 2); i += 64 * CW * SETS) {
                const int jc = i / (HD / 2), d = 2 * (i % (HD / 2));
                const Joined r = join<4>(part + (int64_t)jc * parts * (HD + 2), HD, d, 0, 1, parts);
                const int u = p.by_group(col0 + jc), h = kvh * p.G + col0 + jc - u * p.G;
                const float inv = inverse(r.l, pos0 + u >= p.most);
                T* out = (T*)p.a.out + (int64_t)(seq.row0 + u) * p.a.out_stride + (int64_t)h * HD + d;
                gptr(out)[0] = (T)(r.a * inv);
                gptr(out)[1] = (T)(r.b * inv);
            }
            return;
        }
    if (col0 + wl * 32 + c32 >= cols) return;
    const float inv = inverse(l, pos >= p.most);
    T* out = (T*)p.a.out + (int64_t)(seq.row0 + t) * p.a.out_stride + (int64_t)(kvh * p.G + col - t * p.G) * HD + 4 * half;
#pragma unroll
    for (int d = 0; d < NB; d++)
#pragma unroll
        for (int u = 0; u < 4; u++) {
            typedef T T4 __attribute__((ext_vector_type(4)));
            T4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = (T)(o[d][4 * u + r] * inv);
            if (p.whole_out) {
                *(AS_GLOBAL T4*)(out + 32 * d + 8 * u) = y;
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++) gptr(out)[32 * d + 8 * u + r] = y[r];
            }
        }
}

// Waves of a SIMD: two where a half of its registers holds what a wave needs.
constexpr int wide_waves(int nb, bool exact) { return nb <= (exact ? 4 : 6) ? 2 : 1; }

// The sequences of many columns, then those of few, in one launch.
template <int NB, int CW, int SETS, typename T>
__global__ __launch_bounds__(64 * CW * SETS)
__attribute__((amdgpu_waves_per_eu(wide_waves(NB, sizeof(T) == 4), 2))) void paged_mixed_kernel(AttnArgs p) {
    extern __shared__ __align__(16) uint8_t lds[];
    if ((int)blockIdx.x < p.wide_grid) wide_part<NB, CW, SETS, T>(p, lds);
    else few_part<NB, T>(p, blockIdx.x - p.wide_grid, lds);
}

template <auto* kernel>
hipError_t launch_one(const AttnArgs& p, int64_t grid, int threads, int lds, hipStream_t st) {
    static OncePerDevice once;
    if (hipError_t e = allow_whole_lds(once, (const void*)kernel)) return e;
    if (grid <= 0) return hipSuccess;
    if (grid * threads > UINT32_MAX) return hipErrorInvalidConfiguration;  // (a launch holds no more threads)
    kernel<<<(unsigned)grid, threads, lds, st>>>(p);
    return hipGetLastError();
}

// Workgroups that the few-column part may need for sequences of up to `cols` columns each.
int64_t few_grid(const AttnArgs& p, int64_t cols) {
    const int64_t tight = ((int64_t)p.b.rows * p.G + 15ll * p.b.sequences) / kFewCols;
    const int64_t most = std::min<int64_t>((int64_t)p.b.rows * ((p.G + kFewCols - 1) / kFewCols),
                                           std::min(tight, p.b.sequences * ((cols + kFewCols - 1) / kFewCols)));
    return most * p.c.kv_heads + p.target + 1;
}

template <int NB, int CW, int SETS, typename T>
hipError_t launch_mixed(AttnArgs& p, hipStream_t st) {
    typedef Wide<NB, CW, SETS> W;
    static_assert(W::FITS, "LDS");
    p.few_columns = kManyColumns;
    // sequences of many columns are at most rows G / kManyColumns, each with a group that is not full
    const int64_t cols = (int64_t)p.b.rows * p.G;
    const int64_t groups = cols / W::COLS + std::min<int64_t>(p.b.sequences, cols / kManyColumns);
    if (groups * p.c.kv_heads > INT32_MAX) return hipErrorInvalidConfiguration;
    p.wide_grid = (int)(groups * p.c.kv_heads);
    p.wide_parts = 1;
    if constexpr (W::SPLIT)
        if (p.wide_grid > 0 && p.wide_grid <= kMostTarget - p.target) {
            const int most = (kMostSlots - few_slots(p.target)) / (W::COLS / kFewCols);
            p.wide_parts = std::max(1, std::min(device_cus(), most) / p.wide_grid);
            p.wide_grid *= p.wide_parts;
        }
    return launch_one<paged_mixed_kernel<NB, CW, SETS, T>>(p, p.wide_grid + few_grid(p, kManyColumns), 64 * CW * SETS,
                                                          W::LDS, st);
}

// How a call runs, by the workgroups that the batch's columns make; the lengths are on the device, and the shares of the
// few-column part are chosen there.  us, one card:
//
// The many-column part, where its workgroups nearly fill the chip. Of 128 columns and one set of waves, two a CU, from one a
// CU on (two sets: 1,000 tokens and 31 single ones, 32/8 heads of 128, f16: 114 and 131; 2,048 tokens 60 and 58); of 128 and
// two sets, where workgroups of 64 are more than the CUs (600 tokens at 4,096: 74, of 64 columns 96; 1,000: 82 and 98); of
// 64 and four sets from 1.6 CUs of them on, in units of 32 dims (300 tokens at 4,096: 53, the few-column part 65; 512 of
// 32/32 heads of 64: 41 and 46; but 1,000 of 9/3 heads of 64: 39 and 33); from 1.1 where heads of 96 and more have tables of
// 2,048 positions and more, whose steps are split (150 tokens at 4,096: 33, the few-column part 52, at 16,000 75 and 122;
// 100 beside 31 single ones 68 and 83; but 140 at 600: 25 and 23, and of 32/32 heads of 64, where nothing is left to split,
// 280 at 2,500: 28 and 23). 200 tokens at 4,096, in two parts: 39, in one 52. Where most workgroups are of sequences of few
// columns, one set of 128 leaves them the most room (512 tokens of 32/32 heads of 64 and 31 single ones: 97, two sets 106,
// 64 columns 125). One sequence's 256 columns, one workgroup a CU, where the short ones of their second round fill it behind
// the long ones of the first (32/8 heads of 128, f16: 4,096 tokens 159 and 168, 3,500 122 and 127; but 3,000 104 and 98,
// 5,000 256 and 242; 24/8 heads, 5,000 176 and 187). Far into a context, where all are alike long, it gains as much (4,096
// behind 28,672 others 1,947 and 2,009, 3,500 behind 29,268 1,784 and 1,890, f32 4,096 3,065 and 3,100); at twice the prompt's
// length little (4,096 of 8,192 419 and 424, f32 650 and 651), and of many KV heads it may lose there (3,800 of 7,600, 32/32
// heads of 96, f16 330 and 317; 1,700 of 3,400, 64/64 of 128, f32 290 and 275).
//
// The few-column part alone: four waves a workgroup (one token of 9/3 heads of 64 at 2,000 positions 8.1, eight waves 8.6),
// a workgroup a CU, or two where groups of columns are half as many (64 sequences of 32/8 heads of 128: 162 and 178; 24 at
// up to 4,000 39 and 45; 12 at up to 12,000, 96 groups, 50 and 50; two at up to 60,000 78.6 and 76.3; one at 131,072 102 and
// 99, of 16/8 heads of 256 at 30,000 54 and 51).
template <int NB, typename T>
hipError_t launch_nb(AttnArgs& p, hipStream_t st) {
    const int64_t cus = device_cus(), cols = (int64_t)p.b.rows * p.G, KVH = p.c.kv_heads;
    const int64_t max_rows = p.a.max_rows > 0 ? std::min(p.a.max_rows, p.b.rows) : p.b.rows;
    auto groups = [&](int width) { return (cols + width - 1) / width * KVH; };
    p.target = (int)std::min<int64_t>(cus, kMostTarget);
    if (max_rows * p.G > kManyColumns) {
        constexpr bool two = wide_waves(NB, sizeof(T) == 4) == 2;
        // sequences that have one row whatever the others have
        const int64_t more = std::max<int64_t>(1, max_rows - 1);
        const int64_t single = p.b.sequences - (p.b.rows - p.b.sequences + more - 1) / more;
        if constexpr (NB == 3 || NB == 4)
            if (p.b.sequences == 1 && !p.a.window && 3 * groups(256) >= 5 * cus && groups(256) <= 2 * cus)
                return launch_mixed<NB, 8, 1, T>(p, st);
        if (groups(128) > cus || (groups(64) * NB > 8 * cus / 5 && (!two || single * KVH >= 4 * groups(128))))
            return launch_mixed<NB, 4, 1, T>(p, st);
        if constexpr (two)
            if (groups(64) > cus) return launch_mixed<NB, 4, 2, T>(p, st);
        // (heads of 32 cannot have 1.6 CUs of these units and no more than a CU of workgroups)
        if constexpr (NB >= 2 && NB <= 4)
            if (10 * groups(64) * NB >= (NB >= 3 && p.most >= 2048 ? 11 : 16) * cus) return launch_mixed<NB, 2, 4, T>(p, st);
    }
    p.few_columns = INT32_MAX;
    const int64_t grid = few_grid(p, cols);
    if (2 * (grid - p.target - 1) >= cus) p.target = (int)std::min<int64_t>(2 * cus, kMostTarget);
    return launch_one<paged_few_kernel<NB, T>>(p, few_grid(p, cols), 64 * kFewWaves, few_lds<NB>(kFewWaves), st);
}

template <typename T>
hipError_t launch(AttnArgs& p, hipStream_t st) {
    switch (p.c.hd / 32) {
    case 1: return launch_nb<1, T>(p, st);
    case 2: return launch_nb<2, T>(p, st);
    case 3: return launch_nb<3, T>(p, st);
    case 4: return launch_nb<4, T>(p, st);
    case 5: return launch_nb<5, T>(p, st);
    case 6: return launch_nb<6, T>(p, st);
    case 7: return launch_nb<7, T>(p, st);
    default: return launch_nb<8, T>(p, st);
    }
}

}  // namespace

int64_t paged_attention_workspace(int hd) { return kMostTarget * 4 + (int64_t)kMostSlots * kFewCols * (hd + 2) * 4; }

hipError_t launch_paged_attention(bool f16_rows, const PagedAttention& a, const PagedSteps& b, const PagedKV& c,
                                  hipStream_t st) {
    AttnArgs p;
    p.a = a;
    p.b = b;
    p.c = c;
    p.G = a.heads / c.kv_heads;
    p.most = b.table_stride << (4 + c.tiles_log2);
    // a window of all positions is none; so bounded, differences of positions are 32-bit numbers
    if (a.window >= p.most) p.a.window = 0;
    p.a.sinks = std::min(a.sinks, p.most);
    p.by_group = Divisor(p.G);
    p.scale_log2 = 1.4426950408889634f / sqrtf((float)c.hd);
    p.counters = (int*)a.workspace;
    p.partials = (float*)((uint8_t*)a.workspace + kMostTarget * 4);
    p.wide_grid = 0;
    p.wide_parts = 1;
    const int size = f16_rows ? 2 : 4;
    auto whole = [&](const void* x, int64_t stride) { return !(((uintptr_t)x | (uint64_t)stride * size) & 15); };
    p.whole_q = whole(a.q, a.q_stride);
    p.whole_out = whole(a.out, a.out_stride);
    return f16_rows ? launch<f16>(p, st) : launch<float>(p, st);
}
