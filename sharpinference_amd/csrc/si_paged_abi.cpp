// C ABI of the paged cache (si_paged.hip, si_paged_attention.hip): argument
// checks, then the launches on the context stream.
#include "si_context.hpp"
#include "si_internal.hpp"
#include "si_paged.hpp"

#include <cmath>

using namespace si_abi;

namespace {

constexpr int MAX_ROWS = 1 << 20, MAX_KV_HEADS = 256;
constexpr int64_t MAX_POSITIONS = 1ll << 30;       // of a sequence: max_pages * page_size

int check_ptr(si_hip_context* ctx, const char* op, const void* p, const char* name, uintptr_t align)
{
    if (!p || !aligned(p, align))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %s must be a non-null %u-byte aligned device pointer", op, name,
                    static_cast<unsigned>(align));
    return SI_HIP_OK;
}

struct Span {
    const void* p;
    uint64_t n;
};

int check_apart(si_hip_context* ctx, const char* op, std::initializer_list<Span> writes,
                std::initializer_list<Span> reads)
{
    for (auto w = writes.begin(); w != writes.end(); ++w) {
        for (const auto& r : reads)
            if (overlaps(w->p, w->n, r.p, r.n))
                return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: an output overlaps an input", op);
        for (auto v = w + 1; v != writes.end(); ++v)
            if (overlaps(w->p, w->n, v->p, v->n))
                return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: outputs overlap", op);
    }
    return SI_HIP_OK;
}

// Shape of one page of one KV head; 0 or a status.
int check_page(si_hip_context* ctx, const char* op, int fmt, int page_size, int head_size)
{
    if (fmt != SI_HIP_F16 && fmt != SI_HIP_Q4_0)
        return fail(ctx, SI_HIP_ERR_UNSUPPORTED, "%s: pages of %s (%d) are not F16 or Q4_0", op, fmt_name(fmt), fmt);
    if (head_size != 64 && head_size != 128)
        return fail(ctx, SI_HIP_ERR_UNSUPPORTED, "%s: head size %d (64 and 128 are built)", op, head_size);
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: page size %d is not a power of two in 16..256", op, page_size);
    return SI_HIP_OK;
}

struct Paged {
    si::PagedBatch batch;
    si::PagedCache cache;
    uint64_t table_bytes, starts_bytes, lengths_bytes, pool_bytes;
};

// Checks a batch and the cache that it goes with.
int take(si_hip_context* ctx, const char* op, const si_hip_paged_batch* b, const si_hip_paged_cache* c, Paged* out)
{
    if (!b || !c)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: null batch or cache", op);
    if (const int rc = check_page(ctx, op, c->cache_format, c->page_size, c->head_size))
        return rc;
    if (c->kv_heads < 1 || c->kv_heads > MAX_KV_HEADS)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d KV heads outside 1..%d", op, c->kv_heads, MAX_KV_HEADS);
    if (c->pages < 1 || c->pages > INT32_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %lld pages outside 1..%d", op, static_cast<long long>(c->pages),
                    INT32_MAX);
    if (b->sequences < 1 || b->sequences > si::PAGED_SEQUENCES_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d sequences outside 1..%d", op, b->sequences,
                    si::PAGED_SEQUENCES_MAX);
    if (b->max_pages < 1 || static_cast<int64_t>(b->max_pages) * c->page_size > MAX_POSITIONS)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d pages of %d positions for a sequence outside 1..%lld positions", op,
                    b->max_pages, c->page_size, static_cast<long long>(MAX_POSITIONS));
    if (b->rows < 1 || b->rows > MAX_ROWS)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d rows outside 1..%d", op, b->rows, MAX_ROWS);
    if (b->max_rows < 1 || b->max_rows > b->rows)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: %d rows of a sequence outside 1..%d", op, b->max_rows, b->rows);
    if (check_ptr(ctx, op, b->page_table, "page table", 4) || check_ptr(ctx, op, b->row_starts, "row starts", 4) ||
        check_ptr(ctx, op, b->lengths, "lengths", 4) || check_ptr(ctx, op, c->key_pages, "key pages", 16) ||
        check_ptr(ctx, op, c->value_pages, "value pages", 16))
        return SI_HIP_ERR_ARGUMENT;
    out->batch = {b->page_table, b->row_starts, b->lengths, b->sequences, b->max_pages, b->rows, b->max_rows};
    const bool q4 = c->cache_format == SI_HIP_Q4_0;
    out->cache = {static_cast<char*>(c->key_pages), static_cast<char*>(c->value_pages), c->pages, c->page_size,
                  __builtin_ctz(static_cast<unsigned>(c->page_size)), c->kv_heads, c->head_size, q4};
    out->table_bytes = static_cast<uint64_t>(b->sequences) * b->max_pages * 4;
    out->starts_bytes = (static_cast<uint64_t>(b->sequences) + 1) * 4;
    out->lengths_bytes = static_cast<uint64_t>(b->sequences) * 4;
    out->pool_bytes = static_cast<uint64_t>(c->pages) * c->kv_heads * si::paged_head_bytes(q4, c->page_size, c->head_size);
    return SI_HIP_OK;
}

int check_heads(si_hip_context* ctx, const char* op, int heads, int kv_heads)
{
    if (heads < 1 || heads % kv_heads != 0 || heads / kv_heads > si::PAGED_GROUP_MAX)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: query heads %d must be 1..%d times KV heads %d", op, heads,
                    si::PAGED_GROUP_MAX, kv_heads);
    return SI_HIP_OK;
}

int launched(si_hip_context* ctx, hipError_t e, const char* op)
{
    return e == hipSuccess ? SI_HIP_OK : hip_fail(ctx, e, op);
}

}  // namespace

extern "C" {

int si_hip_paged_page_bytes(int cache_format, int page_size, int head_size, uint64_t* bytes)
{
    if (!bytes)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "paged_page_bytes: null output");
    if (const int rc = check_page(nullptr, "paged_page_bytes", cache_format, page_size, head_size))
        return rc;
    *bytes = static_cast<uint64_t>(si::paged_head_bytes(cache_format == SI_HIP_Q4_0, page_size, head_size));
    return SI_HIP_OK;
}

int si_hip_paged_kv_append(si_hip_context* ctx, const si_hip_paged_append_args* args)
{
    const char* op = "paged_kv_append";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (!args)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: null arguments", op);
    Paged p;
    if (const int rc = take(ctx, op, &args->batch, &args->cache, &p))
        return rc;
    const int d = p.cache.head;
    if (check_heads(ctx, op, args->query_heads, p.cache.kv_heads))
        return SI_HIP_ERR_ARGUMENT;
    if (args->rotary_size < 0 || args->rotary_size > d || args->rotary_size % 2 != 0)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: rotary size %d is not even in 0..%d", op, args->rotary_size, d);
    if (!std::isfinite(args->rope_scale))
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: the rotary scale must be finite", op);
    if (check_ptr(ctx, op, args->qkv, "qkv", 4) || check_ptr(ctx, op, args->query, "query", 4) ||
        (args->rotary_size && check_ptr(ctx, op, args->frequencies, "frequencies", 4)))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t rows = static_cast<uint64_t>(p.batch.rows);
    const uint64_t q_b = rows * args->query_heads * d * 4, qkv_b = q_b + rows * 2 * p.cache.kv_heads * d * 4;
    if (check_apart(ctx, op,
                    {{args->query, q_b}, {p.cache.keys, p.pool_bytes}, {p.cache.values, p.pool_bytes}},
                    {{args->qkv, qkv_b},
                     {args->frequencies, static_cast<uint64_t>(args->rotary_size) * 2},
                     {p.batch.table, p.table_bytes},
                     {p.batch.starts, p.starts_bytes},
                     {p.batch.lengths, p.lengths_bytes}}))
        return SI_HIP_ERR_ARGUMENT;
    const si::PagedAppendArgs a{p.batch, p.cache, args->qkv, args->frequencies, args->query, args->query_heads,
                                args->rotary_size, args->rope_scale};
    return launched(ctx, si::launch_paged_append(a, ctx->stream), op);
}

int si_hip_paged_kv_read(si_hip_context* ctx, const si_hip_paged_batch* batch, const si_hip_paged_cache* cache,
                         float* keys, float* values)
{
    const char* op = "paged_kv_read";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    Paged p;
    if (const int rc = take(ctx, op, batch, cache, &p))
        return rc;
    if (check_ptr(ctx, op, keys, "keys", 4) || check_ptr(ctx, op, values, "values", 4))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t out_b = static_cast<uint64_t>(p.batch.rows) * p.cache.kv_heads * p.cache.head * 4;
    if (check_apart(ctx, op, {{keys, out_b}, {values, out_b}},
                    {{p.cache.keys, p.pool_bytes},
                     {p.cache.values, p.pool_bytes},
                     {p.batch.table, p.table_bytes},
                     {p.batch.starts, p.starts_bytes},
                     {p.batch.lengths, p.lengths_bytes}}))
        return SI_HIP_ERR_ARGUMENT;
    return launched(ctx, si::launch_paged_read(p.batch, p.cache, keys, values, ctx->stream), op);
}

int si_hip_paged_attention_workspace_bytes(int query_heads, int kv_heads, int head_size, uint64_t* bytes)
{
    const char* op = "paged_attention_workspace_bytes";
    if (!bytes)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null output", op);
    if (head_size != 64 && head_size != 128)
        return fail(nullptr, SI_HIP_ERR_UNSUPPORTED, "%s: head size %d (64 and 128 are built)", op, head_size);
    if (kv_heads < 1 || kv_heads > MAX_KV_HEADS)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: %d KV heads outside 1..%d", op, kv_heads, MAX_KV_HEADS);
    if (check_heads(nullptr, op, query_heads, kv_heads))
        return SI_HIP_ERR_ARGUMENT;
    *bytes = static_cast<uint64_t>(si::paged_attention_workspace_floats(query_heads, kv_heads, head_size)) * 4;
    return SI_HIP_OK;
}

int si_hip_paged_attention(si_hip_context* ctx, const si_hip_paged_attention_args* args)
{
    const char* op = "paged_attention";
    if (!ctx)
        return fail(nullptr, SI_HIP_ERR_ARGUMENT, "%s: null context", op);
    Enter g(ctx);
    if (g.err != hipSuccess)
        return hip_fail(ctx, g.err, "hipSetDevice");
    if (!args)
        return fail(ctx, SI_HIP_ERR_ARGUMENT, "%s: null arguments", op);
    Paged p;
    if (const int rc = take(ctx, op, &args->batch, &args->cache, &p))
        return rc;
    const int d = p.cache.head;
    if (check_heads(ctx, op, args->query_heads, p.cache.kv_heads))
        return SI_HIP_ERR_ARGUMENT;
    if (args->output_format != SI_HIP_F32 && args->output_format != SI_HIP_F16 && args->output_format != SI_HIP_BF16)
        return fail(ctx, SI_HIP_ERR_UNSUPPORTED, "%s: output of %s (%d) is not F32, F16 or BF16", op,
                    fmt_name(args->output_format), args->output_format);
    if (check_ptr(ctx, op, args->query, "query", 16) || check_ptr(ctx, op, args->output, "output", 16) ||
        check_ptr(ctx, op, args->workspace, "workspace", 16))
        return SI_HIP_ERR_ARGUMENT;
    const uint64_t count = static_cast<uint64_t>(p.batch.rows) * args->query_heads * d;
    const uint64_t ws_b =
        static_cast<uint64_t>(si::paged_attention_workspace_floats(args->query_heads, p.cache.kv_heads, d)) * 4;
    if (check_apart(ctx, op, {{args->output, count * (args->output_format == SI_HIP_F32 ? 4 : 2)}, {args->workspace, ws_b}},
                    {{args->query, count * 4},
                     {p.cache.keys, p.pool_bytes},
                     {p.cache.values, p.pool_bytes},
                     {p.batch.table, p.table_bytes},
                     {p.batch.starts, p.starts_bytes},
                     {p.batch.lengths, p.lengths_bytes}}))
        return SI_HIP_ERR_ARGUMENT;
    const si::PagedAttentionArgs a{p.batch, p.cache, args->query, args->output, static_cast<float*>(args->workspace),
                                   args->query_heads,
                                   args->output_format == SI_HIP_F32   ? si::PAGED_OUT_F32
                                   : args->output_format == SI_HIP_F16 ? si::PAGED_OUT_F16
                                                                       : si::PAGED_OUT_BF16,
                                   0};
    return launched(ctx, si::launch_paged_attention(a, ctx->stream), op);
}

}  // extern "C"
