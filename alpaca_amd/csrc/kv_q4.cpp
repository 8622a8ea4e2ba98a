// The entry points of the 4-bit KV cache and of the per-head norm with
// rotation (alpaca_hip.h): argument checks and launches.  None allocates, copies
// or waits, so all may be captured into a HIP graph.
#include "kv_q4.h"

#include <algorithm>
#include <cmath>

#include "checks.h"

namespace {

// Head counts and dims, and the sizes that the kernels' grids and 32-bit token indexes hold.
constexpr int kMostHeads = 65535, kMostTokens = 1 << 30;

int check_shape(int kv_heads, int hd, int capacity) {
    if (kv_heads <= 0 || kv_heads > kMostHeads || capacity <= 0 || capacity > kMostTokens) return bad("cache shape");
    return check_dim(hd);
}

int check_cache(const ahip_kv_q4* c) {
    if (!c || !c->k || !c->v) return bad("null cache");
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return bad("cache buffers must be 16-byte aligned");
    return check_shape(c->kv_heads, c->head_dim, c->capacity);
}

// start .. start + tokens inside the capacity; a start on the device is checked there.
int check_range(int start, const int32_t* start_dev, int tokens, int capacity) {
    if (tokens < 0 || tokens > capacity) return bad("more tokens than the cache holds");
    if (start_dev) return (uintptr_t)start_dev & 3 ? bad("misaligned start_dev") : (int)AHIP_OK;
    if (start < 0 || start > capacity - tokens)
        return bad("positions %d to %lld exceed the capacity %d", start, (long long)start + tokens, capacity);
    return AHIP_OK;
}

Q4Cache cache_of(const ahip_kv_q4* a) {
    Q4Cache c;
    c.k = (uint8_t*)a->k;
    c.v = (uint8_t*)a->v;
    c.kv_heads = a->kv_heads;
    c.capacity = a->capacity;
    c.nb = a->head_dim / 32;
    return c;
}

}  // namespace

extern "C" int ahip_kv_q4_bytes(int kv_heads, int capacity, int head_dim, int64_t* bytes) {
    if (!bytes) return bad("null argument");
    if (int rc = check_shape(kv_heads, head_dim, capacity)) return rc;
    *bytes = (int64_t)kv_heads * q4_head_bytes(capacity, head_dim / 32);
    return AHIP_OK;
}

extern "C" int ahip_kv_q4_store(ahip_context* ctx, const ahip_kv_q4* cache, int dtype, const void* k,
                                int64_t k_stride, const void* v, int64_t v_stride, int tokens, int start,
                                const int32_t* start_dev, ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_range(start, start_dev, tokens, cache->capacity)) return rc;
    if (tokens == 0) return AHIP_OK;
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
    if (int rc = check_rows("keys", k, k_stride, width, dtype)) return rc;
    if (int rc = check_rows("values", v, v_stride, width, dtype)) return rc;
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    return launched(launch_q4_store(dtype == AHIP_F16, {k, k_stride}, {v, v_stride}, tokens, start, start_dev,
                                    cache_of(cache), st));
}

extern "C" int ahip_kv_q4_load(ahip_context* ctx, const ahip_kv_q4* cache, int dtype, int start, int tokens, void* k,
                               int64_t k_stride, void* v, int64_t v_stride, ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_range(start, nullptr, tokens, cache->capacity)) return rc;
    if (tokens == 0 || (!k && !v)) return AHIP_OK;
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
    if (k)
        if (int rc = check_rows("keys", k, k_stride, width, dtype)) return rc;
    if (v)
        if (int rc = check_rows("values", v, v_stride, width, dtype)) return rc;
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    return launched(launch_q4_load(dtype == AHIP_F16, cache_of(cache), start, tokens, k, k_stride, v, v_stride, st));
}

static int check_queries(const ahip_kv_q4* c, int tokens, int heads) {
    if (heads <= 0 || heads > kMostHeads || heads % c->kv_heads)
        return bad("query heads must be a multiple of the KV heads");
    if (tokens < 0 || tokens > c->capacity) return bad("more tokens than the cache holds");
    if ((int64_t)tokens * heads > kMostTokens) return failed(AHIP_ERR_UNSUPPORTED, "more than 2^30 queries a call");
    return AHIP_OK;
}

// By the positions that the call may see: up to its last query's, or the capacity where only
// the device knows the start.
static Q4Plan plan_of(const ahip_kv_q4* c, int dtype, int tokens, int heads, int start, bool on_device) {
    return q4_attention_plan(dtype == AHIP_F16, tokens, heads, c->kv_heads, c->head_dim,
                             on_device ? c->capacity : start + tokens);
}

static_assert(kQ4Counters * 4 == AHIP_Q4_WORKSPACE_ZERO, "the counters at the front of a workspace");

extern "C" int ahip_attention_q4_workspace(ahip_context* ctx, const ahip_kv_q4* cache, int dtype, int tokens,
                                           int heads, int start, int on_device, int64_t* bytes) {
    if (!ctx || !bytes) return bad("null argument");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_queries(cache, tokens, heads)) return rc;
    if (!on_device)
        if (int rc = check_range(start, nullptr, tokens, cache->capacity)) return rc;
    *bytes = 0;
    if (tokens == 0) return AHIP_OK;
    hipStream_t st;
    if (int rc = stream_of(ctx, nullptr, &st)) return rc;  // (the device's CU count)
    *bytes = q4_attention_workspace(tokens, heads, cache->head_dim,
                                    plan_of(cache, dtype, tokens, heads, start, on_device));
    return AHIP_OK;
}

extern "C" int ahip_attention_q4(ahip_context* ctx, const ahip_kv_q4* cache, int dtype, const void* q,
                                 int64_t q_stride, int tokens, int heads, int start, const int32_t* start_dev,
                                 void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes,
                                 ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_queries(cache, tokens, heads)) return rc;
    if (int rc = check_range(start, start_dev, tokens, cache->capacity)) return rc;
    if (tokens == 0) return AHIP_OK;
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (int rc = check_rows("queries", q, q_stride, width, dtype)) return rc;
    if (int rc = check_rows("output", out, out_stride, width, dtype)) return rc;
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    const Q4Plan plan = plan_of(cache, dtype, tokens, heads, start, start_dev);
    const int64_t need = q4_attention_workspace(tokens, heads, cache->head_dim, plan);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return bad("the attention needs %lld bytes of 16-byte aligned workspace, got %lld", (long long)need,
                   workspace ? (long long)workspace_bytes : 0);
    Q4Attention a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.tokens = tokens;
    a.heads = heads;
    a.start = start;
    a.start_dev = start_dev;
    q4_set_workspace(a, workspace);
    return launched(launch_q4_attention(dtype == AHIP_F16, a, cache_of(cache), plan, st));
}

extern "C" int ahip_qk_norm_rope(ahip_context* ctx, const ahip_norm_rope* args, ahip_stream* stream) {
    if (!ctx || !args) return bad(ctx ? "null arguments" : "null context");
    const ahip_norm_rope& n = *args;
    if (int rc = check_dtype(n.dtype)) return rc;
    if (int rc = check_dim(n.head_dim)) return rc;
    if (n.heads < 0 || n.heads > kMostHeads || n.kv_heads < 0 || n.kv_heads > kMostHeads) return bad("head counts");
    if (n.tokens < 0 || n.tokens > kMostTokens) return bad("token count");
    if ((int64_t)n.tokens * (n.heads + n.kv_heads) > kMostTokens)
        return failed(AHIP_ERR_UNSUPPORTED, "more than 2^30 heads a call");
    if ((n.q_gain || n.k_gain) && !(n.eps >= 0 && std::isfinite(n.eps))) return bad("eps must be finite and >= 0");
    if (((uintptr_t)n.q_gain | (uintptr_t)n.k_gain) & 3) return bad("misaligned gain");
    if (n.rope) {
        if ((uintptr_t)n.rope & 7) return bad("misaligned rotation table");
        if (n.rope_positions <= 0) return bad("empty rotation table");
        if (n.positions) {
            if ((uintptr_t)n.positions & 3) return bad("misaligned positions");
        } else if (n.start < 0 || n.tokens > n.rope_positions || n.start > n.rope_positions - n.tokens) {
            return bad("positions exceed the rotation table");
        }
    }
    if (n.tokens == 0 || n.heads + n.kv_heads == 0) return AHIP_OK;
    if (n.heads) {
        const int64_t width = (int64_t)n.heads * n.head_dim;
        if (int rc = check_rows("queries", n.q, n.q_stride, width, n.dtype)) return rc;
        if (int rc = check_rows("query output", n.q_out, n.q_out_stride, width, n.dtype)) return rc;
    }
    if (n.kv_heads) {
        const int64_t width = (int64_t)n.kv_heads * n.head_dim;
        if (int rc = check_rows("keys", n.k, n.k_stride, width, n.dtype)) return rc;
        if (int rc = check_rows("key output", n.k_out, n.k_out_stride, width, n.dtype)) return rc;
    }
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    return launched(launch_norm_rope(n.dtype == AHIP_F16, n, st));
}
