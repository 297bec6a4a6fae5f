// C ABI of the attention operators (see include/rbmoe.h): attention of whole sequences both ways, the paged cache, decode rows
// over it.  Checks of arguments and launches only; every call is enqueued on the context's stream, allocates nothing and waits for
// nothing, so it can be captured into a graph.
#include <cmath>
#include <new>
#include <string>

#include "attention_kernels.h"
#include "kv_cache_kernels.h"
#include "rbmoe_context.h"

using namespace rbmoe;

struct rbmoe_attention {
    rbmoe_ctx* ctx = nullptr;
    int heads = 0, kv_heads = 0, head_dim = 0, dtype = 0, backward_rows = 0;
    void* workspace = nullptr;  // references and deltas of rows, then sums of shares
    size_t bytes = 0, parts_at = 0;
    int part_rows = 0;
};

struct rbmoe_kv_cache {
    rbmoe_ctx* ctx = nullptr;
    CachePool pool{};
    int dtype = 0;
    size_t bytes = 0;
};

struct rbmoe_decode {
    rbmoe_ctx* ctx = nullptr;
    int heads = 0, kv_heads = 0, head_dim = 0, dtype = 0, max_sequences = 0;
    size_t partials = 0, bytes = 0;
    void* workspace = nullptr;
};

namespace {

constexpr int kMostHeads = 1024, kMostSequences = 65535, kMostRows = 1 << 30, kMostCacheRows = 1 << 28;

bool off_element(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == RBMOE_BF16 ? 2 : 4) != 0; }

// What every operator asks of its heads.
int heads_problem(rbmoe_ctx* ctx, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype) {
    if (heads <= 0 || kv_heads <= 0 || head_dim <= 0) return fail(ctx, RBMOE_INVALID_CONFIG, "heads, kv_heads and head_dim must be positive");
    if (heads % kv_heads)
        return fail(ctx, RBMOE_INVALID_CONFIG, "n_heads (" + std::to_string(heads) + ") must be a multiple of n_kv_heads (" + std::to_string(kv_heads) + ")");
    if (heads > kMostHeads) return fail(ctx, RBMOE_UNSUPPORTED, "more than 1024 heads");
    if (head_dim % 8 || head_dim > kMostHeadDim) return fail(ctx, RBMOE_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128");
    if (dtype != RBMOE_F32 && dtype != RBMOE_BF16) return fail(ctx, RBMOE_INVALID_CONFIG, "rows must be f32 or bf16");
    return RBMOE_OK;
}

// `stride` of rows of `width` elements, 0: without gaps
int stride_problem(rbmoe_ctx* ctx, int32_t stride, int width, long long& out) {
    if (stride != 0 && stride < width) return fail(ctx, RBMOE_INVALID_INPUT, "a row stride is smaller than the row");
    out = stride ? stride : width;
    return RBMOE_OK;
}

int scale_problem(rbmoe_ctx* ctx, float scale) {
    if (!std::isfinite(scale) || !(scale > 0.0f)) return fail(ctx, RBMOE_INVALID_INPUT, "scale must be finite and positive");
    return RBMOE_OK;
}

// What both directions ask of the sequences; fills the common part of a call.  `nothing`: no workgroup would have anything to do.
int sequences_problem(rbmoe_attention* at, int32_t sequences, int32_t longest_queries, int32_t longest_keys, const int32_t* query_begin,
                      const int32_t* query_count, const int32_t* key_begin, const int32_t* key_count, int32_t query_rows, int32_t key_rows,
                      int32_t q_stride, int32_t k_stride, int32_t v_stride, float scale, AttentionCall& a) {
    rbmoe_ctx* ctx = at->ctx;
    if (sequences < 0 || longest_queries < 0 || longest_keys < 0 || query_rows < 0 || key_rows < 0)
        return fail(ctx, RBMOE_INVALID_INPUT, "counts must not be negative");
    if (sequences > kMostSequences || query_rows > kMostRows || key_rows > kMostRows)
        return fail(ctx, RBMOE_UNSUPPORTED, "more than 65535 sequences or 2^30 rows");
    if (const int rc = scale_problem(ctx, scale)) return rc;
    if ((key_begin != nullptr) != (key_count != nullptr)) return fail(ctx, RBMOE_NULL_POINTER, "key_begin and key_count come together");
    if (sequences > 0 && (!query_begin || !query_count)) return fail(ctx, RBMOE_NULL_POINTER, "query_begin or query_count is NULL");
    for (const void* p : {query_begin, query_count, key_begin, key_count})
        if (off_element(p, RBMOE_F32)) return fail(ctx, RBMOE_INVALID_INPUT, "begins and counts must start at an element");
    if (const int rc = stride_problem(ctx, q_stride, at->heads * at->head_dim, a.q_stride)) return rc;
    if (const int rc = stride_problem(ctx, k_stride, at->kv_heads * at->head_dim, a.k_stride)) return rc;
    if (const int rc = stride_problem(ctx, v_stride, at->kv_heads * at->head_dim, a.v_stride)) return rc;
    a.query_begin = query_begin;
    a.query_count = query_count;
    a.key_begin = key_begin ? key_begin : query_begin;
    a.key_count = key_count ? key_count : query_count;
    a.sequences = sequences;
    a.query_rows = query_rows;
    a.key_rows = key_rows;
    a.longest_queries = longest_queries;
    a.longest_keys = longest_keys;
    a.most_queries = longest_queries < query_rows ? longest_queries : query_rows;
    a.most_keys = longest_keys < key_rows ? longest_keys : key_rows;
    a.heads = at->heads;
    a.kv_heads = at->kv_heads;
    a.head_dim = at->head_dim;
    a.scale = scale;
    const long long tiles = ((long long)a.most_queries + 127) / 128, key_tiles = ((long long)a.most_keys + 127) / 128;
    if (tiles * at->heads * sequences > (1 << 23) || key_tiles * at->kv_heads * sequences > (1 << 23))
        return fail(ctx, RBMOE_UNSUPPORTED, "sequences * heads * longest is more than a launch has workgroups for");
    return RBMOE_OK;
}

}  // namespace

extern "C" {

int rbmoe_attention_create(rbmoe_ctx* ctx, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t backward_rows,
                           rbmoe_attention** out) {
    if (!ctx || !out) return fail(ctx, RBMOE_NULL_POINTER, "ctx or out is NULL");
    *out = nullptr;
    if (const int rc = heads_problem(ctx, heads, kv_heads, head_dim, dtype)) return rc;
    if (backward_rows < 0) return fail(ctx, RBMOE_INVALID_CONFIG, "backward_rows must not be negative");
    if (backward_rows > kMostRows) return fail(ctx, RBMOE_UNSUPPORTED, "more than 2^30 rows");
    rbmoe_attention* a = new (std::nothrow) rbmoe_attention();
    if (!a) return fail(ctx, RBMOE_OUT_OF_MEMORY, "no host memory for the attention");
    a->ctx = ctx;
    a->heads = heads;
    a->kv_heads = kv_heads;
    a->head_dim = head_dim;
    a->dtype = dtype;
    a->backward_rows = backward_rows;
    a->part_rows = attention_part_rows(backward_rows, kv_heads, heads / kv_heads);
    a->parts_at = ((size_t)backward_rows * heads * 8 + 15) / 16 * 16;
    a->bytes = a->parts_at + (size_t)a->part_rows * (heads / kv_heads) * 2 * head_dim * 4;
    if (a->bytes)
        if (const int rc = ctx_alloc(ctx, a->bytes, "the backward pass's sums", &a->workspace)) {
            delete a;
            return rc;
        }
    ++ctx->refs;
    *out = a;
    return RBMOE_OK;
}

void rbmoe_attention_destroy(rbmoe_attention* a) {
    if (!a) return;
    (void)hipStreamSynchronize(a->ctx->stream);
    ctx_free(a->ctx, a->workspace, a->bytes);
    ctx_release(a->ctx);
    delete a;
}

int rbmoe_attention_forward(rbmoe_attention* at, int32_t sequences, int32_t longest_queries, int32_t longest_keys, const int32_t* query_begin,
                            const int32_t* query_count, const int32_t* key_begin, const int32_t* key_count, int32_t query_rows,
                            int32_t key_rows, const void* q, int32_t q_stride, const void* k, int32_t k_stride, const void* v,
                            int32_t v_stride, int32_t causal, float scale, void* out, float* lse) {
    if (!at) return fail(nullptr, RBMOE_NULL_POINTER, "attention is NULL");
    rbmoe_ctx* ctx = at->ctx;
    AttentionCall a{};
    if (const int rc = sequences_problem(at, sequences, longest_queries, longest_keys, query_begin, query_count, key_begin, key_count, query_rows,
                                         key_rows, q_stride, k_stride, v_stride, scale, a))
        return rc;
    if (sequences == 0 || a.most_queries == 0) return RBMOE_OK;
    if (!q || !out || (a.most_keys > 0 && (!k || !v))) return fail(ctx, RBMOE_NULL_POINTER, "q, k, v or out is NULL");
    for (const void* p : {q, k, v, (const void*)out})
        if (off_element(p, at->dtype)) return fail(ctx, RBMOE_INVALID_INPUT, "rows must start at an element");
    if (off_element(lse, RBMOE_F32)) return fail(ctx, RBMOE_INVALID_INPUT, "lse must start at an element");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.lse = lse;
    a.causal = causal != 0;
    HIP_TRY(ctx, launch_attention_forward(a, at->dtype == RBMOE_BF16, ctx->stream));
    return RBMOE_OK;
}

int rbmoe_attention_backward(rbmoe_attention* at, int32_t sequences, int32_t longest_queries, int32_t longest_keys, const int32_t* query_begin,
                             const int32_t* query_count, const int32_t* key_begin, const int32_t* key_count, int32_t query_rows,
                             int32_t key_rows, const void* q, int32_t q_stride, const void* k, int32_t k_stride, const void* v,
                             int32_t v_stride, int32_t causal, float scale, const void* out, const float* lse, const void* grad_out,
                              void* grad_q, void* grad_k, void* grad_v) {
    if (!at) return fail(nullptr, RBMOE_NULL_POINTER, "attention is NULL");
    rbmoe_ctx* ctx = at->ctx;
    AttentionCall a{};
    if (const int rc = sequences_problem(at, sequences, longest_queries, longest_keys, query_begin, query_count, key_begin, key_count, query_rows,
                                         key_rows, q_stride, k_stride, v_stride, scale, a))
        return rc;
    if (query_rows > at->backward_rows)
        return fail(ctx, RBMOE_INVALID_INPUT, "this attention was created for the backward pass of " + std::to_string(at->backward_rows) + " rows, got " +
                                                  std::to_string(query_rows));
    if (sequences == 0 || (a.most_queries == 0 && a.most_keys == 0)) return RBMOE_OK;
    if (a.most_queries > 0) {
        if (!q || !out || !lse || !grad_out || !grad_q) return fail(ctx, RBMOE_NULL_POINTER, "q, out, lse, grad_out or grad_q is NULL");
    }
    if (a.most_keys > 0 && (!k || !v || !grad_k || !grad_v)) return fail(ctx, RBMOE_NULL_POINTER, "k, v, grad_k or grad_v is NULL");
    if (grad_q && (grad_q == grad_k || grad_q == grad_v)) return fail(ctx, RBMOE_INVALID_INPUT, "gradients must be three arrays");
    if (grad_k && grad_k == grad_v) return fail(ctx, RBMOE_INVALID_INPUT, "gradients must be three arrays");
    for (const void* p : {q, k, v, out, grad_out, (const void*)grad_q, (const void*)grad_k, (const void*)grad_v})
        if (off_element(p, at->dtype)) return fail(ctx, RBMOE_INVALID_INPUT, "rows must start at an element");
    if (off_element(lse, RBMOE_F32)) return fail(ctx, RBMOE_INVALID_INPUT, "lse must start at an element");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = const_cast<void*>(out);
    a.lse = const_cast<float*>(lse);
    a.causal = causal != 0;
    a.grad_out = grad_out;
    a.grad_q = grad_q;
    a.grad_k = grad_k;
    a.grad_v = grad_v;
    a.delta = static_cast<float*>(at->workspace);
    a.parts = reinterpret_cast<float*>(static_cast<char*>(at->workspace) + at->parts_at);
    a.part_rows = at->part_rows;
    HIP_TRY(ctx, launch_attention_backward(a, at->dtype == RBMOE_BF16, ctx->stream));
    return RBMOE_OK;
}

int rbmoe_kv_cache_create(rbmoe_ctx* ctx, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t cache_dtype, int32_t page_rows,
                          int32_t pages, rbmoe_kv_cache** out) {
    if (!ctx || !out) return fail(ctx, RBMOE_NULL_POINTER, "ctx or out is NULL");
    *out = nullptr;
    if (const int rc = heads_problem(ctx, kv_heads, kv_heads, head_dim, dtype)) return rc;
    if (cache_dtype != dtype && cache_dtype != RBMOE_I8) return fail(ctx, RBMOE_INVALID_CONFIG, "a cache is of its rows' type or int8");
    if (pages <= 0) return fail(ctx, RBMOE_INVALID_CONFIG, "the number of pages must be positive");
    if (page_rows < 16 || page_rows > 4096 || (page_rows & (page_rows - 1)))
        return fail(ctx, RBMOE_INVALID_CONFIG, "a page has a power of two of rows between 16 and 4096");
    rbmoe_kv_cache* c = new (std::nothrow) rbmoe_kv_cache();
    if (!c) return fail(ctx, RBMOE_OUT_OF_MEMORY, "no host memory for the cache");
    c->ctx = ctx;
    c->dtype = dtype;
    int shift = 4;
    while ((1 << shift) < page_rows) ++shift;
    c->pool = CachePool{nullptr, pages, shift, kv_heads, head_dim, cache_dtype};
    c->bytes = cache_bytes(c->pool);
    void* p = nullptr;
    if (const int rc = ctx_alloc(ctx, c->bytes, "the cache's pages", &p)) {
        delete c;
        return rc;
    }
    c->pool.base = static_cast<unsigned char*>(p);
    hipError_t e = hipMemsetAsync(p, 0, c->bytes, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) {
        ctx_free(ctx, p, c->bytes);
        delete c;
        return hip_fail(ctx, e, "clearing the cache's pages");
    }
    ++ctx->refs;
    *out = c;
    return RBMOE_OK;
}

void rbmoe_kv_cache_destroy(rbmoe_kv_cache* c) {
    if (!c) return;
    (void)hipStreamSynchronize(c->ctx->stream);
    ctx_free(c->ctx, c->pool.base, c->bytes);
    ctx_release(c->ctx);
    delete c;
}

static int cache_rows_call(rbmoe_kv_cache* c, int32_t rows, const void* k, int32_t k_stride, const void* v, int32_t v_stride,
                           const int64_t* slots, bool write) {
    if (!c) return fail(nullptr, RBMOE_NULL_POINTER, "cache is NULL");
    rbmoe_ctx* ctx = c->ctx;
    if (rows < 0) return fail(ctx, RBMOE_INVALID_INPUT, "the row count must not be negative");
    if (rows > kMostCacheRows) return fail(ctx, RBMOE_UNSUPPORTED, "more than 2^28 rows");  // (a launch's 2^32 threads)
    CacheRows a{};
    if (const int rc = stride_problem(ctx, k_stride, c->pool.kv_heads * c->pool.head_dim, a.k_stride)) return rc;
    if (const int rc = stride_problem(ctx, v_stride, c->pool.kv_heads * c->pool.head_dim, a.v_stride)) return rc;
    if (rows == 0) return RBMOE_OK;
    if (!k || !v || !slots) return fail(ctx, RBMOE_NULL_POINTER, "k, v or slots is NULL");
    if (off_element(k, c->dtype) || off_element(v, c->dtype)) return fail(ctx, RBMOE_INVALID_INPUT, "rows must start at an element");
    if (reinterpret_cast<uintptr_t>(slots) % 8) return fail(ctx, RBMOE_INVALID_INPUT, "slots must start at an element");
    if (!write && k == v) return fail(ctx, RBMOE_INVALID_INPUT, "keys and values must be two arrays");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    a.pool = c->pool;
    a.k = const_cast<void*>(k);
    a.v = const_cast<void*>(v);
    a.slots = slots;
    a.rows = rows;
    HIP_TRY(ctx, write ? launch_cache_write(a, c->dtype == RBMOE_BF16, ctx->stream) : launch_cache_read(a, c->dtype == RBMOE_BF16, ctx->stream));
    return RBMOE_OK;
}

int rbmoe_kv_cache_write(rbmoe_kv_cache* c, int32_t rows, const void* k, int32_t k_stride, const void* v, int32_t v_stride, const int64_t* slots) {
    return cache_rows_call(c, rows, k, k_stride, v, v_stride, slots, true);
}

int rbmoe_kv_cache_read(rbmoe_kv_cache* c, int32_t rows, void* k, int32_t k_stride, void* v, int32_t v_stride, const int64_t* slots) {
    return cache_rows_call(c, rows, k, k_stride, v, v_stride, slots, false);
}

int rbmoe_decode_create(rbmoe_ctx* ctx, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t max_sequences,
                        rbmoe_decode** out) {
    if (!ctx || !out) return fail(ctx, RBMOE_NULL_POINTER, "ctx or out is NULL");
    *out = nullptr;
    if (const int rc = heads_problem(ctx, heads, kv_heads, head_dim, dtype)) return rc;
    if (max_sequences <= 0) return fail(ctx, RBMOE_INVALID_CONFIG, "max_sequences must be positive");
    if (max_sequences > kMostSequences) return fail(ctx, RBMOE_UNSUPPORTED, "more than 65535 sequences");
    rbmoe_decode* d = new (std::nothrow) rbmoe_decode();
    if (!d) return fail(ctx, RBMOE_OUT_OF_MEMORY, "no host memory for the decode attention");
    d->ctx = ctx;
    d->heads = heads;
    d->kv_heads = kv_heads;
    d->head_dim = head_dim;
    d->dtype = dtype;
    d->max_sequences = max_sequences;
    d->partials = decode_partials(max_sequences, kv_heads, heads / kv_heads);
    d->bytes = d->partials * ((head_dim <= 64 ? 64 : 128) + 2) * 4;
    if (const int rc = ctx_alloc(ctx, d->bytes, "the parts of long caches", &d->workspace)) {
        delete d;
        return rc;
    }
    ++ctx->refs;
    *out = d;
    return RBMOE_OK;
}

void rbmoe_decode_destroy(rbmoe_decode* d) {
    if (!d) return;
    (void)hipStreamSynchronize(d->ctx->stream);
    ctx_free(d->ctx, d->workspace, d->bytes);
    ctx_release(d->ctx);
    delete d;
}

int rbmoe_decode_attention(rbmoe_decode* d, rbmoe_kv_cache* c, int32_t sequences, const void* q, int32_t q_stride, const int32_t* tables,
                           int32_t table_pages, const int32_t* lengths, int32_t longest, float scale, void* out) {
    if (!d) return fail(nullptr, RBMOE_NULL_POINTER, "decode is NULL");
    rbmoe_ctx* ctx = d->ctx;
    if (!c) return fail(ctx, RBMOE_NULL_POINTER, "cache is NULL");
    if (c->ctx != ctx) return fail(ctx, RBMOE_INVALID_INPUT, "the cache belongs to another context");
    if (c->pool.kv_heads != d->kv_heads || c->pool.head_dim != d->head_dim || c->dtype != d->dtype)
        return fail(ctx, RBMOE_INVALID_INPUT, "the cache has other heads or rows of another type");
    if (sequences < 0 || table_pages < 0 || longest < 0) return fail(ctx, RBMOE_INVALID_INPUT, "counts must not be negative");
    if (sequences > d->max_sequences)
        return fail(ctx, RBMOE_INVALID_INPUT, "this decode attention was created for " + std::to_string(d->max_sequences) + " sequences, got " +
                                                  std::to_string(sequences));
    if (longest > kMostRows) return fail(ctx, RBMOE_UNSUPPORTED, "caches of more than 2^30 rows a sequence");
    if (const int rc = scale_problem(ctx, scale)) return rc;
    DecodeCall a{};
    if (const int rc = stride_problem(ctx, q_stride, d->heads * d->head_dim, a.q_stride)) return rc;
    if (sequences == 0) return RBMOE_OK;
    if (!q || !out || !lengths || (table_pages > 0 && !tables)) return fail(ctx, RBMOE_NULL_POINTER, "q, tables, lengths or out is NULL");
    if (off_element(q, d->dtype) || off_element(out, d->dtype)) return fail(ctx, RBMOE_INVALID_INPUT, "rows must start at an element");
    if (off_element(tables, RBMOE_F32) || off_element(lengths, RBMOE_F32))
        return fail(ctx, RBMOE_INVALID_INPUT, "tables and lengths must start at an element");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    a.pool = c->pool;
    a.q = q;
    a.out = out;
    a.tables = tables;
    a.lengths = lengths;
    a.sequences = sequences;
    a.heads = d->heads;
    a.table_pages = table_pages;
    a.longest = longest;
    const DecodePlan plan = decode_plan(sequences, d->kv_heads, d->heads / d->kv_heads, longest);
    a.ranges = plan.ranges;
    a.many = plan.many;
    a.scale = scale;
    a.partial = static_cast<float*>(d->workspace);
    a.statistics = a.partial + d->partials * (d->head_dim <= 64 ? 64 : 128);
    HIP_TRY(ctx, launch_decode_attention(a, d->dtype == RBMOE_BF16, ctx->stream));
    return RBMOE_OK;
}

// Which rows of a sequence a call finds: q0, nq, k0, nk, ahead; for tests (no GPU needed).
void rbmoe_internal_attention_sequence(int32_t query_begin, int32_t query_count, int32_t key_begin, int32_t key_count, int32_t query_rows,
                                       int32_t key_rows, int32_t longest_queries, int32_t longest_keys, int32_t* out) {
    const Sequence s = cut_sequence(query_begin, query_count, key_begin, key_count, query_rows, key_rows, longest_queries, longest_keys);
    out[0] = s.q0;
    out[1] = s.nq;
    out[2] = s.k0;
    out[3] = s.nk;
    out[4] = s.ahead;
}

// Into how many ranges a call cuts its sequences: for tests (no GPU needed).
int rbmoe_internal_decode_ranges(int32_t sequences, int32_t kv_heads, int32_t group, int32_t longest) {
    return decode_plan(sequences, kv_heads, group, longest).ranges;
}
// And for how many parts of heads the workspace of a handle for so many sequences has room.
int64_t rbmoe_internal_decode_parts(int32_t max_sequences, int32_t kv_heads, int32_t group) {
    return (int64_t)decode_partials(max_sequences, kv_heads, group);
}

}  // extern "C"
