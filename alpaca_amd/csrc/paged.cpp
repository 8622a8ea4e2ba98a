// The entry points of the KV cache in pages and of token log probabilities
// (alpaca_hip.h): argument checks and launches.  None allocates, copies or waits, so all
// may be captured into a HIP graph.
#include "paged.h"

#include "checks.h"
#include "logprobs.h"

namespace {

constexpr int kMostHeads = 32767;        // of either kind: both lie in one dimension of a grid
constexpr int kMostRows = 1 << 26;       // (a launch holds 2^32 threads)
constexpr int kMostPairs = 1 << 30;      // of a row and a head; positions of a table's row
constexpr int kMostLogits = 1 << 30;     // of a row
constexpr int kMostSequences = 1 << 20;

int log2_of(int x) {
    int r = 0;
    while (1 << r < x) r++;
    return r;
}

int check_layout(int kv_heads, int hd, int page_tokens, int pages) {
    if (kv_heads <= 0 || kv_heads > kMostHeads) return bad("KV head count");
    if (page_tokens < 16 || page_tokens > 1024 || page_tokens & (page_tokens - 1))
        return bad("tokens of a page must be a power of two from 16 to 1024");
    if (pages <= 0) return bad("page count");
    return check_dim(hd);
}

int check_cache(const ahip_paged_kv* c) {
    if (!c || !c->k || !c->v) return bad("null cache");
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return bad("cache buffers must be 16-byte aligned");
    return check_layout(c->kv_heads, c->head_dim, c->page_tokens, c->pages);
}

int check_batch(const ahip_paged_batch* b, const ahip_paged_kv* c) {
    if (!b) return bad("null batch");
    if (b->rows < 0 || b->rows > kMostRows || b->sequences < 0 || b->sequences > kMostSequences || b->max_rows < 0)
        return bad("batch shape");
    if (b->rows == 0 || b->sequences == 0) return AHIP_OK;  // (nothing runs)
    if (!b->row_starts || !b->lengths || !b->table) return bad("null batch array");
    if (((uintptr_t)b->row_starts | (uintptr_t)b->lengths | (uintptr_t)b->table) & 3) return bad("misaligned batch array");
    if (b->table_stride <= 0 || (int64_t)b->table_stride * c->page_tokens > kMostPairs)
        return bad("a table's row must hold 1 to 2^30 tokens");
    return AHIP_OK;
}

bool nothing(const ahip_paged_batch& b) { return b.rows == 0 || b.sequences == 0; }

PagedKV cache_of(const ahip_paged_kv& a) {
    PagedKV c;
    c.k = (uint8_t*)a.k;
    c.v = (uint8_t*)a.v;
    c.kv_heads = a.kv_heads;
    c.hd = a.head_dim;
    c.pages = a.pages;
    c.tiles_log2 = log2_of(a.page_tokens / kPagedTile);
    return c;
}

PagedSteps steps_of(const ahip_paged_batch& a) {
    PagedSteps b;
    b.row_starts = a.row_starts;
    b.lengths = a.lengths;
    b.table = a.table;
    b.sequences = a.sequences;
    b.table_stride = a.table_stride;
    b.rows = a.rows;
    return b;
}

int check_heads(const ahip_paged_batch& b, int heads) {
    if (heads > kMostHeads) return bad("query head count");
    if ((int64_t)b.rows * heads > kMostPairs) return failed(AHIP_ERR_UNSUPPORTED, "more than 2^30 queries a call");
    return AHIP_OK;
}

}  // namespace

extern "C" int ahip_paged_kv_bytes(int kv_heads, int head_dim, int page_tokens, int pages, int64_t* bytes) {
    if (!bytes) return bad("null argument");
    if (int rc = check_layout(kv_heads, head_dim, page_tokens, pages)) return rc;
    const int64_t page = (int64_t)kv_heads * page_tokens * head_dim * 2;
    if (page > INT64_MAX / pages) return bad("implausibly large cache");
    *bytes = page * pages;
    return AHIP_OK;
}

extern "C" int ahip_paged_append(ahip_context* ctx, const ahip_paged_kv* cache, const ahip_paged_batch* batch,
                                 const ahip_paged_rows* rows, ahip_stream* stream) {
    if (!ctx || !rows) return bad(ctx ? "null rows" : "null context");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(batch, cache)) return rc;
    if (int rc = check_dtype(rows->dtype)) return rc;
    if (rows->heads < 0) return bad("query head count");
    if (int rc = check_heads(*batch, rows->heads)) return rc;
    if (rows->rope) {
        if ((uintptr_t)rows->rope & 7) return bad("misaligned rotation table");
        if (rows->rope_positions <= 0) return bad("empty rotation table");
    }
    if (rows->heads == 0 && (rows->q || rows->q_out)) return bad("queries of no heads");
    if (nothing(*batch)) return AHIP_OK;
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim, q_width = (int64_t)rows->heads * cache->head_dim;
    if (int rc = check_rows("keys", rows->k, rows->k_stride, width, rows->dtype)) return rc;
    if (int rc = check_rows("values", rows->v, rows->v_stride, width, rows->dtype)) return rc;
    if (rows->heads) {
        if (int rc = check_rows("queries", rows->q, rows->q_stride, q_width, rows->dtype)) return rc;
        if (int rc = check_rows("query output", rows->q_out, rows->q_out_stride, q_width, rows->dtype)) return rc;
    }
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    PagedRows r;
    r.q = rows->q;
    r.k = rows->k;
    r.v = rows->v;
    r.q_out = rows->q_out;
    r.q_stride = rows->q_stride;
    r.k_stride = rows->k_stride;
    r.v_stride = rows->v_stride;
    r.q_out_stride = rows->q_out_stride;
    r.rope = (const float2*)rows->rope;
    r.rope_positions = rows->rope_positions;
    r.heads = rows->heads;
    r.interleaved = rows->interleaved;
    return launched(launch_paged_append(rows->dtype == AHIP_F16, r, steps_of(*batch), cache_of(*cache), st));
}

extern "C" int ahip_paged_load(ahip_context* ctx, const ahip_paged_kv* cache, const ahip_paged_batch* batch, int dtype,
                               void* k, int64_t k_stride, void* v, int64_t v_stride, ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(batch, cache)) return rc;
    if (int rc = check_dtype(dtype)) return rc;
    if (nothing(*batch) || (!k && !v)) return AHIP_OK;
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
    if (k)
        if (int rc = check_rows("keys", k, k_stride, width, dtype)) return rc;
    if (v)
        if (int rc = check_rows("values", v, v_stride, width, dtype)) return rc;
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    return launched(launch_paged_load(dtype == AHIP_F16, steps_of(*batch), cache_of(*cache), k, k_stride, v, v_stride, st));
}

static_assert(kPagedCounters * 4 == AHIP_PAGED_WORKSPACE_ZERO, "the counters at the front of a workspace");

extern "C" int ahip_paged_attention_workspace(const ahip_paged_kv* cache, int64_t* bytes) {
    if (!bytes) return bad("null argument");
    if (int rc = check_cache(cache)) return rc;
    *bytes = paged_attention_workspace(cache->head_dim);
    return AHIP_OK;
}

extern "C" int ahip_paged_attention(ahip_context* ctx, const ahip_paged_kv* cache, const ahip_paged_batch* batch,
                                    int dtype, const void* q, int64_t q_stride, int heads, int window, int sinks,
                                    void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes,
                                    ahip_stream* stream) {
    if (!ctx) return bad("null context");
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_batch(batch, cache)) return rc;
    if (int rc = check_dtype(dtype)) return rc;
    if (heads <= 0 || heads % cache->kv_heads) return bad("query heads must be a multiple of the KV heads");
    if (int rc = check_heads(*batch, heads)) return rc;
    if (window < 0 || sinks < 0) return bad("window and sinks must not be negative");
    if (nothing(*batch)) return AHIP_OK;
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (int rc = check_rows("queries", q, q_stride, width, dtype)) return rc;
    if (int rc = check_rows("output", out, out_stride, width, dtype)) return rc;
    const int64_t need = paged_attention_workspace(cache->head_dim);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))
        return bad("the attention needs %lld bytes of 16-byte aligned workspace, got %lld", (long long)need,
                   workspace ? (long long)workspace_bytes : 0);
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    PagedAttention a;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.heads = heads;
    a.window = window;
    a.sinks = sinks;
    a.max_rows = batch->max_rows;
    a.workspace = workspace;
    return launched(launch_paged_attention(dtype == AHIP_F16, a, steps_of(*batch), cache_of(*cache), st));
}

static_assert(kLogprobsMostSplitRows * 4 == AHIP_LOGPROBS_WORKSPACE_ZERO && kLogprobsMostTop == AHIP_LOGPROBS_MOST_TOP,
              "alpaca_hip.h");

extern "C" int ahip_token_logprobs_workspace(int64_t* bytes) {
    if (!bytes) return bad("null argument");
    *bytes = logprobs_workspace();
    return AHIP_OK;
}

extern "C" int ahip_token_logprobs(ahip_context* ctx, const ahip_logprobs* args, void* workspace,
                                   int64_t workspace_bytes, ahip_stream* stream) {
    if (!ctx || !args) return bad(ctx ? "null arguments" : "null context");
    const ahip_logprobs& a = *args;
    if (int rc = check_dtype(a.dtype)) return rc;
    if (a.rows < 0 || a.rows >= 1 << 24 || a.vocab <= 0 || a.vocab > kMostLogits) return bad("logits' shape");
    if (a.top < 0 || a.top > AHIP_LOGPROBS_MOST_TOP || a.top > a.vocab)
        return bad("top must be 0 to %d and at most the vocabulary", AHIP_LOGPROBS_MOST_TOP);
    if (a.rows == 0 || (!a.logprobs && !a.entropy && !a.top)) return AHIP_OK;
    if (int rc = check_rows("logits", a.logits, a.stride, a.vocab, a.dtype)) return rc;
    if (a.logprobs && !a.tokens) return bad("null tokens");
    if (a.top && (!a.top_tokens || !a.top_logprobs)) return bad("null top outputs");
    if (((uintptr_t)a.tokens | (uintptr_t)a.logprobs | (uintptr_t)a.entropy) & 3) return bad("misaligned array");
    if (a.top && ((uintptr_t)a.top_tokens | (uintptr_t)a.top_logprobs) & 3) return bad("misaligned array");
    if (workspace && (workspace_bytes < logprobs_workspace() || ((uintptr_t)workspace & 15)))
        return bad("a workspace must have %lld bytes, 16-byte aligned, got %lld", (long long)logprobs_workspace(),
                   (long long)workspace_bytes);
    hipStream_t st;
    if (int rc = stream_of(ctx, stream, &st)) return rc;
    LogprobsArgs p;
    p.logits = a.logits;
    p.stride = a.stride;
    p.rows = a.rows;
    p.vocab = a.vocab;
    p.top = a.top;
    p.tokens = a.tokens;
    p.logprobs = a.logprobs;
    p.entropy = a.entropy;
    p.top_tokens = a.top_tokens;
    p.top_logprobs = a.top_logprobs;
    return launched(launch_logprobs(a.dtype == AHIP_F16, p, workspace, st));
}
