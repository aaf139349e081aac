// C ABI of attention over a window or a paged cache and of the cache's pages (see include/pimdl.h): checks and launches.
#include "serve_common.h"

using namespace pimdl;

namespace {

uint32_t dtype_bytes(uint32_t t) { return t == PIMDL_F32 ? 4 : 2; }

// Device memory of the context's own device, aligned to `align` bytes.
int check_device(Ctx* ctx, const char* fn, const char* name, const void* p, uintptr_t align)
{
    if (!p) return set_error(ctx, PIMDL_ERR_INVALID, "%s: %s is null", fn, name);
    if (reinterpret_cast<uintptr_t>(p) % align)
        return set_error(ctx, PIMDL_ERR_INVALID, "%s: %s must be aligned to %u bytes", fn, name, (unsigned)align);
    hipPointerAttribute_t attr = {};
    if (hipPointerGetAttributes(&attr, p) != hipSuccess) {
        (void)hipGetLastError();  // ordinary host memory
        return set_error(ctx, PIMDL_ERR_INVALID, "%s: %s must be a device pointer", fn, name);
    }
    if (attr.type != hipMemoryTypeDevice && attr.type != hipMemoryTypeManaged)
        return set_error(ctx, PIMDL_ERR_INVALID, "%s: %s must be a device pointer", fn, name);
    if (attr.type == hipMemoryTypeDevice && attr.device != ctx->device)
        return set_error(ctx, PIMDL_ERR_INVALID, "%s: %s is on device %d, the context on device %d", fn, name, attr.device, ctx->device);
    return PIMDL_OK;
}

int check_batch(Ctx* ctx, const char* fn, const int32_t* starts, uint32_t batch, uint32_t tokens)
{
    if (batch >= 1u << 24 || tokens >= 1u << 30) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: batch must be below 2^24 and tokens below 2^30", fn);
    return check_device(ctx, fn, "starts", starts, 4);
}

// What every attention call shares: heads, row sizes and the scale.
int check_heads(Ctx* ctx, const char* fn, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t q_stride, uint32_t out_stride, float scale)
{
    if (head_dim == 0 || heads == 0 || kv_heads == 0) return set_error(ctx, PIMDL_ERR_INVALID, "%s: zero-sized heads", fn);
    if (head_dim > 256) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: head_dim=%u (up to 256)", fn, head_dim);
    if (heads % kv_heads) return set_error(ctx, PIMDL_ERR_INVALID, "%s: heads=%u is not a multiple of kv_heads=%u", fn, heads, kv_heads);
    if (heads > 65535) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: heads must be below 65536", fn);
    if ((uint64_t)heads * head_dim > q_stride || (uint64_t)heads * head_dim > out_stride)
        return set_error(ctx, PIMDL_ERR_INVALID, "%s: q_stride and out_stride must hold heads * head_dim elements", fn);
    if (!(scale >= -0x1p96f && scale <= 0x1p96f)) return set_error(ctx, PIMDL_ERR_INVALID, "%s: scale must be finite, of a magnitude up to 2^96", fn);
    return PIMDL_OK;
}

int check_cache(Ctx* ctx, const char* fn, const pimdl_paged_cache* c, uint32_t dtype)
{
    if (!c) return set_error(ctx, PIMDL_ERR_INVALID, "%s: cache is null", fn);
    if (c->dtype > PIMDL_BF16 || dtype > PIMDL_BF16) return set_error(ctx, PIMDL_ERR_INVALID, "%s: unknown dtype", fn);
    if (dtype != PIMDL_F32 && dtype != c->dtype)
        return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: 16-bit tensors need a cache of their own type", fn);
    if (c->page_tokens < 16 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1)))
        return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: page_tokens=%u (a power of two, 16 .. 1024)", fn, c->page_tokens);
    if (c->kv_heads == 0 || c->head_dim == 0 || c->pages == 0 || c->seqs == 0 || c->table_width == 0)
        return set_error(ctx, PIMDL_ERR_INVALID, "%s: zero-sized cache", fn);
    if (c->head_dim > 256 || c->kv_heads > 65535) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: head_dim up to 256, kv_heads below 65536", fn);
    if (c->pages > 0x7fffffffu || (uint64_t)c->table_width * c->page_tokens > 0x7fffffffu - 4096)
        return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: pages and table_width * page_tokens must be below 2^31 - 4096", fn);
    return PIMDL_OK;
}

int check_cache_memory(Ctx* ctx, const char* fn, const pimdl_paged_cache* c)
{
    int rc = check_device(ctx, fn, "cache k", c->k, 16);
    if (!rc) rc = check_device(ctx, fn, "cache v", c->v, 16);
    if (!rc) rc = check_device(ctx, fn, "cache tables", c->tables, 4);
    if (!rc) rc = check_device(ctx, fn, "cache lengths", c->lengths, 4);
    if (!rc && c->lacking) rc = check_device(ctx, fn, "cache lacking", c->lacking, 4);
    return rc;
}

uint32_t shift_of(uint32_t page_tokens) { return (uint32_t)__builtin_ctz(page_tokens); }

// tables: whether the call needs them (and with them lengths, refs and lacking)
int check_book(Ctx* ctx, const char* fn, const pimdl_page_book* b, bool tables, bool pools)
{
    if (!b) return set_error(ctx, PIMDL_ERR_INVALID, "%s: book is null", fn);
    if (b->pages == 0 || b->pages > 1u << 24) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: pages=%u (1 .. 2^24)", fn, b->pages);
    int rc = PIMDL_OK;
    if (tables) {
        if (b->page_tokens == 0) return set_error(ctx, PIMDL_ERR_INVALID, "%s: page_tokens is zero", fn);
        if (b->seqs == 0 || b->seqs > 16384) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: seqs=%u (1 .. 16384)", fn, b->seqs);
        if (b->table_width == 0 || (uint64_t)b->table_width * b->page_tokens > 0x7fffffffu - 4096)
            return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: table_width * page_tokens must be 1 .. 2^31 - 4096", fn);
        rc = check_device(ctx, fn, "tables", b->tables, 4);
        if (!rc) rc = check_device(ctx, fn, "lengths", b->lengths, 4);
        if (!rc) rc = check_device(ctx, fn, "refs", b->refs, 4);
        if (!rc) rc = check_device(ctx, fn, "lacking", b->lacking, 4);
    }
    if (!rc && pools) {
        if (b->pool_count && !b->pools) return set_error(ctx, PIMDL_ERR_INVALID, "%s: pools is null", fn);
        if (b->pool_count > 64) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: pool_count=%u (up to 64)", fn, b->pool_count);
        if (b->layers > 65536) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: layers=%u (up to 65536)", fn, b->layers);
        if (b->pool_count && (b->page_bytes == 0 || b->page_bytes % 16 || b->page_bytes > 1u << 30))
            return set_error(ctx, PIMDL_ERR_INVALID, "%s: page_bytes must be a multiple of 16, up to 2^30", fn);
        for (uint32_t i = 0; i < b->pool_count && !rc; ++i) rc = check_device(ctx, fn, "pools[i]", b->pools[i], 16);
    }
    return rc;
}

int check_list(Ctx* ctx, const char* fn, const char* name, const int32_t* list, uint32_t n)
{
    if (n > 16384) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "%s: a list of %u (up to 16384)", fn, n);
    return check_device(ctx, fn, name, list, 4);
}

}  // namespace

extern "C" {

int pimdl_attention_window(pimdl_ctx* ctx, const pimdl_attention_window_desc* d)
{
    static const char fn[] = "pimdl_attention_window";
    if (!ctx) return PIMDL_ERR_INVALID;
    if (!d) return set_error(ctx, PIMDL_ERR_INVALID, "%s: null argument", fn);
    if (d->dtype > PIMDL_BF16) return set_error(ctx, PIMDL_ERR_INVALID, "%s: unknown dtype", fn);
    int rc = check_heads(ctx, fn, d->heads, d->kv_heads, d->head_dim, d->q_stride, d->out_stride, d->scale);
    if (rc) return rc;
    if ((uint64_t)d->kv_heads * d->head_dim > d->kv_stride)
        return set_error(ctx, PIMDL_ERR_INVALID, "%s: kv_stride must hold kv_heads * head_dim elements", fn);
    if (d->tokens == 0 || d->batch == 0) return PIMDL_OK;
    const uint32_t e = dtype_bytes(d->dtype);
    if ((rc = check_batch(ctx, fn, d->starts, d->batch, d->tokens)) || (rc = check_device(ctx, fn, "q", d->q, e)) ||
        (rc = check_device(ctx, fn, "k", d->k, e)) || (rc = check_device(ctx, fn, "v", d->v, e)) || (rc = check_device(ctx, fn, "out", d->out, e)))
        return rc;
    if ((rc = activate(ctx))) return rc;
    AttnArgs a = {};
    a.q = d->q, a.k = d->k, a.v = d->v, a.out = d->out, a.starts = d->starts;
    a.batch = d->batch, a.tokens = d->tokens, a.heads = d->heads, a.kv_heads = d->kv_heads, a.head_dim = d->head_dim, a.group = d->heads / d->kv_heads;
    a.q_stride = d->q_stride, a.kv_stride = d->kv_stride, a.out_stride = d->out_stride;
    a.left = d->left, a.right = d->right, a.sinks = d->sinks;
    a.dtype = a.cache_dtype = d->dtype, a.scale = d->scale;
    return launch_attention(ctx, a);
}

int pimdl_attention_paged(pimdl_ctx* ctx, const pimdl_paged_cache* cache, const int32_t* seqs, const int32_t* starts, uint32_t batch,
                          uint32_t tokens, const void* q, void* out, uint32_t heads, uint32_t q_stride, uint32_t out_stride, uint32_t dtype,
                          uint32_t left, uint32_t sinks, float scale)
{
    static const char fn[] = "pimdl_attention_paged";
    if (!ctx) return PIMDL_ERR_INVALID;
    int rc = check_cache(ctx, fn, cache, dtype);
    if (rc || (rc = check_heads(ctx, fn, heads, cache->kv_heads, cache->head_dim, q_stride, out_stride, scale))) return rc;
    if (!seqs && batch > cache->seqs) return set_error(ctx, PIMDL_ERR_INVALID, "%s: batch=%u exceeds the cache's %u sequences", fn, batch, cache->seqs);
    if (tokens == 0 || batch == 0) return PIMDL_OK;
    const uint32_t e = dtype_bytes(dtype);
    if ((rc = check_cache_memory(ctx, fn, cache)) || (rc = check_batch(ctx, fn, starts, batch, tokens)) || (seqs && (rc = check_device(ctx, fn, "seqs", seqs, 4))) ||
        (rc = check_device(ctx, fn, "q", q, e)) || (rc = check_device(ctx, fn, "out", out, e)))
        return rc;
    if ((rc = activate(ctx))) return rc;
    AttnArgs a = {};
    a.q = q, a.k = cache->k, a.v = cache->v, a.out = out, a.starts = starts, a.seqs = seqs, a.tables = cache->tables, a.lengths = cache->lengths;
    a.batch = batch, a.tokens = tokens, a.heads = heads, a.kv_heads = cache->kv_heads, a.head_dim = cache->head_dim, a.group = heads / cache->kv_heads;
    a.q_stride = q_stride, a.out_stride = out_stride;
    a.left = left, a.right = 0, a.sinks = sinks;
    a.pages = cache->pages, a.page_shift = shift_of(cache->page_tokens), a.table_width = cache->table_width, a.seq_count = cache->seqs;
    a.dtype = dtype, a.cache_dtype = cache->dtype, a.paged = 1, a.scale = scale;
    return launch_attention(ctx, a);
}

int pimdl_attention_last_plan(const pimdl_ctx* ctx, pimdl_attention_plan* out)
{
    if (!ctx || !out) return PIMDL_ERR_INVALID;
    *out = ctx->attn_plan;
    return PIMDL_OK;
}

int pimdl_cache_append(pimdl_ctx* ctx, const pimdl_paged_cache* cache, const int32_t* seqs, const int32_t* starts, uint32_t batch,
                       uint32_t tokens, const void* k, const void* v, uint32_t kv_stride, uint32_t dtype)
{
    static const char fn[] = "pimdl_cache_append";
    if (!ctx) return PIMDL_ERR_INVALID;
    int rc = check_cache(ctx, fn, cache, dtype);
    if (rc) return rc;
    if ((uint64_t)cache->kv_heads * cache->head_dim > kv_stride)
        return set_error(ctx, PIMDL_ERR_INVALID, "%s: kv_stride must hold kv_heads * head_dim elements", fn);
    if (!seqs && batch > cache->seqs) return set_error(ctx, PIMDL_ERR_INVALID, "%s: batch=%u exceeds the cache's %u sequences", fn, batch, cache->seqs);
    if (tokens == 0 || batch == 0) return PIMDL_OK;
    const uint32_t e = dtype_bytes(dtype);
    if ((rc = check_cache_memory(ctx, fn, cache)) || (rc = check_batch(ctx, fn, starts, batch, tokens)) || (seqs && (rc = check_device(ctx, fn, "seqs", seqs, 4))) ||
        (rc = check_device(ctx, fn, "k", k, e)) || (rc = check_device(ctx, fn, "v", v, e)))
        return rc;
    if ((rc = activate(ctx))) return rc;
    return launch_cache_append(ctx, *cache, seqs, starts, batch, tokens, k, v, kv_stride, dtype);
}

int pimdl_pages_reserve(pimdl_ctx* ctx, const pimdl_page_book* book, const int32_t* seqs, const int32_t* counts, uint32_t n)
{
    static const char fn[] = "pimdl_pages_reserve";
    if (!ctx) return PIMDL_ERR_INVALID;
    int rc = check_book(ctx, fn, book, true, false);
    if (!rc && n) rc = check_list(ctx, fn, "seqs", seqs, n);
    if (!rc && n) rc = check_list(ctx, fn, "counts", counts, n);
    if (rc || (rc = activate(ctx))) return rc;
    return launch_pages_reserve(ctx, *book, seqs, counts, n);
}

int pimdl_pages_fork(pimdl_ctx* ctx, const pimdl_page_book* book, const int32_t* parents, const int32_t* children, uint32_t n)
{
    static const char fn[] = "pimdl_pages_fork";
    if (!ctx) return PIMDL_ERR_INVALID;
    int rc = check_book(ctx, fn, book, true, true);
    if (!rc && n) rc = check_list(ctx, fn, "parents", parents, n);
    if (!rc && n) rc = check_list(ctx, fn, "children", children, n);
    if (rc || (rc = activate(ctx))) return rc;
    return launch_pages_fork(ctx, *book, parents, children, n);
}

int pimdl_pages_free(pimdl_ctx* ctx, const pimdl_page_book* book, const int32_t* seqs, uint32_t n)
{
    static const char fn[] = "pimdl_pages_free";
    if (!ctx) return PIMDL_ERR_INVALID;
    int rc = check_book(ctx, fn, book, true, false);
    if (!rc && n) rc = check_list(ctx, fn, "seqs", seqs, n);
    if (rc || n == 0 || (rc = activate(ctx))) return rc;
    return launch_pages_free(ctx, *book, seqs, n);
}

int pimdl_pages_compact(pimdl_ctx* ctx, const pimdl_page_book* book)
{
    static const char fn[] = "pimdl_pages_compact";
    if (!ctx) return PIMDL_ERR_INVALID;
    int rc = check_book(ctx, fn, book, true, true);
    if (rc || (rc = activate(ctx))) return rc;
    return launch_pages_compact(ctx, *book);
}

int pimdl_pages_copy(pimdl_ctx* ctx, const pimdl_page_book* book, const int32_t* src, const int32_t* dst, uint32_t n)
{
    static const char fn[] = "pimdl_pages_copy";
    if (!ctx) return PIMDL_ERR_INVALID;
    int rc = check_book(ctx, fn, book, false, true);
    if (rc || n == 0) return rc;
    if (n > book->pages) return set_error(ctx, PIMDL_ERR_INVALID, "%s: more pairs than pages", fn);
    if ((rc = check_device(ctx, fn, "src", src, 4)) || (rc = check_device(ctx, fn, "dst", dst, 4)) || (rc = activate(ctx))) return rc;
    return launch_pages_copy(ctx, *book, src, dst, n);
}

}  // extern "C"
