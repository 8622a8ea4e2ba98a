// The entry points of the 4-bit KV cache and of the per-head norm with
// rotation (alpaca_hip.h): argument checks and launches.  None allocates, copies
// or waits, so all may be captured into a HIP graph.
#include "kv_q4.h"

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/alpaca_hip.h"
#include "host.h"

namespace {

int bad(const std::string& what) { return ahip_fail(AHIP_ERR_INVALID_ARGUMENT, what); }

int launched(hipError_t e) {
    if (e == hipSuccess) return AHIP_OK;
    hipGetLastError();
    return ahip_fail(AHIP_ERR_COMMAND_FAILED, std::string("kernel launch: ") + hipGetErrorString(e));
}

// Head counts and dims, and the sizes that the kernels' grids and 32-bit token indexes hold.
constexpr int kMostHeads = 65535, kMostTokens = 1 << 30;

int check_dim(int hd) {
    if (hd <= 0 || hd % 32 || hd > 256) return bad("head dimension must be a multiple of 32 up to 256");
    return AHIP_OK;
}

int check_cache(const void* k, const void* v, int kv_heads, int hd, int capacity) {
    if (!k || !v) return bad("null cache");
    if (((uintptr_t)k | (uintptr_t)v) & 15) return bad("cache buffers must be 16-byte aligned");
    if (kv_heads <= 0 || kv_heads > kMostHeads || capacity <= 0 || capacity > kMostTokens) return bad("cache shape");
    return check_dim(hd);
}

int check_dtype(int dtype) {
    if (dtype != AHIP_F32 && dtype != AHIP_F16) return bad("rows must be f32 or f16");
    return AHIP_OK;
}

// Rows of `width` elements, `stride` elements apart.
int check_rows(const char* what, const void* p, int64_t stride, int64_t width, int dtype) {
    if (!p) return bad(std::string("null ") + what);
    if ((uintptr_t)p % (dtype == AHIP_F32 ? 4 : 2)) return bad(std::string(what) + ": misaligned");
    if (stride < width) return bad(std::string(what) + ": stride below the row's width");
    if (stride > (int64_t)1 << 32) return bad(std::string(what) + ": implausibly large stride");
    return AHIP_OK;
}

// start .. start + tokens inside the capacity; a start on the device is checked there.
int check_range(int start, const int32_t* start_dev, int tokens, int capacity) {
    if (tokens < 0 || tokens > capacity) return bad("more tokens than the cache holds");
    if (start_dev) return (uintptr_t)start_dev & 3 ? bad("misaligned start_dev") : (int)AHIP_OK;
    if (start < 0 || start > capacity - tokens)
        return bad("positions " + std::to_string(start) + " to " + std::to_string((int64_t)start + tokens) +
                   " exceed the capacity " + std::to_string(capacity));
    return AHIP_OK;
}

int stream_of(ahip_context* ctx, ahip_stream* stream, hipStream_t* out) {
    if (stream && stream->device != ctx->device) return bad("stream and context belong to different devices");
    (void)hipGetLastError();  // a launch's own failure is read back through it
    if (hipSetDevice(ctx->device) != hipSuccess) return ahip_fail(AHIP_ERR_COMMAND_FAILED, "hipSetDevice");
    *out = stream ? stream->st : ctx->stream;
    return AHIP_OK;
}

Q4Cache cache_of(void* k, void* v, int kv_heads, int hd, int capacity) {
    Q4Cache c;
    c.k = (uint8_t*)k;
    c.v = (uint8_t*)v;
    c.kv_heads = kv_heads;
    c.capacity = capacity;
    c.nb = hd / 32;
    return c;
}

}  // namespace

extern "C" int ahip_kv_q4_bytes(int kv_heads, int capacity, int head_dim, int64_t* bytes) {
    if (!bytes) return bad("null argument");
    if (kv_heads <= 0 || kv_heads > kMostHeads || capacity <= 0 || capacity > kMostTokens) return bad("cache shape");
    if (int rc = check_dim(head_dim)) return rc;
    *bytes = (int64_t)kv_heads * q4_head_bytes(capacity, head_dim / 32);
    return AHIP_OK;
}

extern "C" int ahip_kv_q4_store(ahip_context* ctx, int dtype, const void* k, int64_t k_stride, const void* v,
                                int64_t v_stride, int tokens, int start, const int32_t* start_dev, void* k_cache,
                                void* v_cache, int kv_heads, int head_dim, int capacity, ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_cache(k_cache, v_cache, kv_heads, head_dim, capacity)) return rc;
    if (int rc = check_range(start, start_dev, tokens, capacity)) return rc;
    if (tokens == 0) return AHIP_OK;
    const int64_t width = (int64_t)kv_heads * head_dim;
    if (int rc = check_rows("keys", k, k_stride, width, dtype)) return rc;
    if (int rc = check_rows("values", v, v_stride, width, dtype)) return rc;
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    return launched(launch_q4_store(dtype == AHIP_F16, {k, k_stride}, {v, v_stride}, tokens, start, start_dev,
                                    cache_of(k_cache, v_cache, kv_heads, head_dim, capacity), st));
}

extern "C" int ahip_kv_q4_load(ahip_context* ctx, int dtype, const void* k_cache, const void* v_cache, int kv_heads,
                               int head_dim, int capacity, int start, int tokens, void* k, int64_t k_stride, void* v,
                               int64_t v_stride, ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_cache(k_cache, v_cache, kv_heads, head_dim, capacity)) return rc;
    if (int rc = check_range(start, nullptr, tokens, capacity)) return rc;
    if (tokens == 0 || (!k && !v)) return AHIP_OK;
    const int64_t width = (int64_t)kv_heads * head_dim;
    if (k)
        if (int rc = check_rows("keys", k, k_stride, width, dtype)) return rc;
    if (v)
        if (int rc = check_rows("values", v, v_stride, width, dtype)) return rc;
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    return launched(launch_q4_load(dtype == AHIP_F16,
                                   cache_of((void*)k_cache, (void*)v_cache, kv_heads, head_dim, capacity), start,
                                   tokens, k, k_stride, v, v_stride, st));
}

// The keys are split by what the call can be asked for: its length, or the capacity where
// only the device knows the start.
static int attention_splits(ahip_context* ctx, int tokens, int heads, int kv_heads, int hd, int start, bool on_device,
                            int capacity, int* splits) {
    if (hipSetDevice(ctx->device) != hipSuccess) {
        hipGetLastError();
        return ahip_fail(AHIP_ERR_COMMAND_FAILED, "hipSetDevice");
    }
    *splits = q4_attention_splits(tokens, heads, kv_heads, hd, on_device ? capacity : start + tokens);
    return AHIP_OK;
}

static int check_queries(int tokens, int heads, int kv_heads, int head_dim, int capacity) {
    if (kv_heads <= 0 || kv_heads > kMostHeads || capacity <= 0 || capacity > kMostTokens) return bad("cache shape");
    if (int rc = check_dim(head_dim)) return rc;
    if (heads <= 0 || heads > kMostHeads || heads % kv_heads) return bad("query heads must be a multiple of the KV heads");
    if (tokens < 0 || tokens > capacity) return bad("more tokens than the cache holds");
    if ((int64_t)tokens * heads > kMostTokens) return ahip_fail(AHIP_ERR_UNSUPPORTED, "more than 2^30 queries a call");
    return AHIP_OK;
}

extern "C" int ahip_attention_q4_workspace(ahip_context* ctx, int tokens, int heads, int kv_heads, int head_dim,
                                           int start, int on_device, int capacity, int64_t* bytes) {
    if (!ctx || !bytes) return bad("null argument");
    if (int rc = check_queries(tokens, heads, kv_heads, head_dim, capacity)) return rc;
    if (!on_device)
        if (int rc = check_range(start, nullptr, tokens, capacity)) return rc;
    *bytes = 0;
    if (tokens == 0) return AHIP_OK;
    int splits = 1;
    if (int rc = attention_splits(ctx, tokens, heads, kv_heads, head_dim, start, on_device, capacity, &splits)) return rc;
    *bytes = q4_attention_partials(tokens, heads, head_dim, splits) * 4;
    return AHIP_OK;
}

extern "C" int ahip_attention_q4(ahip_context* ctx, int dtype, const void* q, int64_t q_stride, int tokens, int heads,
                                 int start, const int32_t* start_dev, const void* k_cache, const void* v_cache,
                                 int kv_heads, int head_dim, int capacity, void* out, int64_t out_stride,
                                 void* workspace, int64_t workspace_bytes, ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_cache(k_cache, v_cache, kv_heads, head_dim, capacity)) return rc;
    if (int rc = check_queries(tokens, heads, kv_heads, head_dim, capacity)) return rc;
    if (int rc = check_range(start, start_dev, tokens, capacity)) return rc;
    if (tokens == 0) return AHIP_OK;
    const int64_t width = (int64_t)heads * head_dim;
    if (int rc = check_rows("queries", q, q_stride, width, dtype)) return rc;
    if (int rc = check_rows("output", out, out_stride, width, dtype)) return rc;
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    int splits = 1;
    if (int rc = attention_splits(ctx, tokens, heads, kv_heads, head_dim, start, start_dev, capacity, &splits)) return rc;
    const int64_t need = q4_attention_partials(tokens, heads, head_dim, splits) * 4;
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return bad("the attention needs " + std::to_string(need) + " bytes of 16-byte aligned workspace, got " +
                   std::to_string(workspace ? workspace_bytes : 0));
    Q4Attention a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.tokens = tokens;
    a.heads = heads;
    a.start = start;
    a.start_dev = start_dev;
    a.partials = (float*)workspace;
    return launched(launch_q4_attention(dtype == AHIP_F16, a,
                                        cache_of((void*)k_cache, (void*)v_cache, kv_heads, head_dim, capacity), splits,
                                        st));
}

extern "C" int ahip_qk_norm_rope(ahip_context* ctx, int dtype, const void* q, int64_t q_stride, int heads,
                                 const float* q_gain, const void* k, int64_t k_stride, int kv_heads,
                                 const float* k_gain, int tokens, int head_dim, float eps, const float* rope,
                                 int rope_positions, int interleaved, int start, const int32_t* positions, void* q_out,
                                 int64_t q_out_stride, void* k_out, int64_t k_out_stride, ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_dim(head_dim)) return rc;
    if (heads < 0 || heads > kMostHeads || kv_heads < 0 || kv_heads > kMostHeads) return bad("head counts");
    if (tokens < 0 || tokens > kMostTokens) return bad("token count");
    if ((int64_t)tokens * (heads + kv_heads) > kMostTokens)
        return ahip_fail(AHIP_ERR_UNSUPPORTED, "more than 2^30 heads a call");
    if ((q_gain || k_gain) && !(eps >= 0 && std::isfinite(eps))) return bad("eps must be finite and >= 0");
    if (((uintptr_t)q_gain | (uintptr_t)k_gain) & 3) return bad("misaligned gain");
    if (rope) {
        if ((uintptr_t)rope & 7) return bad("misaligned rotation table");
        if (rope_positions <= 0) return bad("empty rotation table");
        if (positions) {
            if ((uintptr_t)positions & 3) return bad("misaligned positions");
        } else if (start < 0 || tokens > rope_positions || start > rope_positions - tokens) {
            return bad("positions exceed the rotation table");
        }
    }
    if (tokens == 0 || heads + kv_heads == 0) return AHIP_OK;
    if (heads) {
        const int64_t width = (int64_t)heads * head_dim;
        if (int rc = check_rows("queries", q, q_stride, width, dtype)) return rc;
        if (int rc = check_rows("query output", q_out, q_out_stride, width, dtype)) return rc;
    }
    if (kv_heads) {
        const int64_t width = (int64_t)kv_heads * head_dim;
        if (int rc = check_rows("keys", k, k_stride, width, dtype)) return rc;
        if (int rc = check_rows("key output", k_out, k_out_stride, width, dtype)) return rc;
    }
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    NormRope a;
    a.tokens = tokens;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.hd = head_dim;
    a.q = {q, q_stride};
    a.k = {k, k_stride};
    a.q_out = q_out;
    a.k_out = k_out;
    a.q_out_stride = q_out_stride;
    a.k_out_stride = k_out_stride;
    a.q_gain = q_gain;
    a.k_gain = k_gain;
    a.eps = eps;
    a.rope = (const float2*)rope;
    a.positions = rope_positions;
    a.interleaved = interleaved ? 1 : 0;
    a.start = start;
    a.position = positions;
    return launched(launch_norm_rope(dtype == AHIP_F16, a, st));
}
