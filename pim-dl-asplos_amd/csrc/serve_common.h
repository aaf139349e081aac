// What the kernels of attention over a window or a paged cache and of the cache's pages share (gfx950).
#pragma once
#include "pimdl_internal.h"

namespace pimdl {

// One call of pimdl_attention_window or pimdl_attention_paged, checked by the caller.
struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t *starts, *seqs, *tables, *lengths;  // seqs may be null
    uint32_t batch, tokens, heads, kv_heads, head_dim, group;  // group: query heads per key head
    uint32_t q_stride, kv_stride, out_stride;
    uint32_t left, right, sinks;
    uint32_t pages, page_shift, table_width, seq_count;  // paged only
    uint32_t dtype, cache_dtype, paged;
    float scale;
    // of a tree of drafted tokens (masks null: there is none): see pimdl_tree
    const uint32_t* masks;
    const int32_t* depths;
    uint32_t words;
};

// One call of pimdl_rotate or pimdl_cache_append_rotary, checked by the caller.
struct RotaryArgs {
    const double* freqs;
    uint32_t dims, pairs;
    const int32_t *starts, *depths;  // depths may be null
    uint32_t batch, tokens, heads, kv_heads, head_dim;
    const void *q, *k, *v;
    void *q_out, *k_out;             // k_out: not paged
    uint32_t q_stride, k_stride, q_out_stride, k_out_stride;  // k_stride: of v too
    uint32_t dtype;
    // paged only
    const int32_t* seqs;             // may be null
    pimdl_paged_cache cache;
    uint32_t page_shift;
};

// A launch has fewer than 2^32 threads along x, so workgroups beyond GRID_X lie in rows of that many (a multiple of the XCDs that they are dealt out to).
constexpr uint32_t GRID_X = 1u << 20;
inline bool fits_launch(uint64_t blocks, uint32_t threads) { return blocks * threads < 1ull << 32; }
inline dim3 grid_of(uint64_t blocks) { return blocks <= GRID_X ? dim3((uint32_t)blocks) : dim3(GRID_X, (uint32_t)((blocks + GRID_X - 1) / GRID_X)); }

int launch_attention(Ctx* ctx, const AttnArgs& a);
int launch_cache_append(Ctx* ctx, const pimdl_paged_cache& c, const int32_t* seqs, const int32_t* starts, uint32_t batch, uint32_t tokens,
                        const void* k, const void* v, uint32_t kv_stride, uint32_t dtype);
int launch_rotary(Ctx* ctx, const RotaryArgs& a, bool paged);
int launch_tree_build(Ctx* ctx, const int32_t* parents, const int32_t* starts, uint32_t batch, uint32_t tokens, uint32_t words, uint32_t* masks,
                      int32_t* depths);
int launch_pages_accept(Ctx* ctx, const pimdl_page_book& b, const int32_t* seqs, const int32_t* starts, uint32_t batch, uint32_t tokens,
                        const pimdl_tree& tree, const int32_t* last, uint32_t row_bytes, int32_t* kept);
int launch_pages_reserve(Ctx* ctx, const pimdl_page_book& b, const int32_t* seqs, const int32_t* counts, uint32_t n);
int launch_pages_fork(Ctx* ctx, const pimdl_page_book& b, const int32_t* parents, const int32_t* children, uint32_t n);
int launch_pages_free(Ctx* ctx, const pimdl_page_book& b, const int32_t* seqs, uint32_t n);
int launch_pages_compact(Ctx* ctx, const pimdl_page_book& b);
int launch_pages_copy(Ctx* ctx, const pimdl_page_book& b, const int32_t* src, const int32_t* dst, uint32_t n);

#ifdef __HIPCC__

// Row b of a packed batch: its rows of the token buffers and, paged, its sequence's table and length.  Everything comes from
// device memory that the library cannot check beforehand, so every number is brought into range here.
struct Row {
    uint32_t first, n;     // rows of the token buffers
    int32_t length, pos0;  // keys there are; position of the first row (negative where there are more rows than keys)
    const int32_t* table;
};

__device__ __forceinline__ uint32_t clamped_start(const int32_t* starts, uint32_t b, uint32_t tokens)
{
    const int32_t s = starts[b];
    return s < 0 ? 0u : (uint32_t)s < tokens ? (uint32_t)s : tokens;
}

// index of the last row whose start is not behind token t (a row without tokens shares its start with the next one)
__device__ __forceinline__ uint32_t row_of_token(const int32_t* starts, uint32_t batch, uint32_t tokens, uint32_t t)
{
    uint32_t lo = 0, hi = batch;  // starts[lo] <= t (or lo == 0)
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (clamped_start(starts, mid, tokens) <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ Row load_row(const int32_t* starts, const int32_t* seqs, const int32_t* tables, const int32_t* lengths,
                                        uint32_t tokens, uint32_t seq_count, uint32_t table_width, uint32_t page_shift, bool paged, uint32_t b)
{
    Row r;
    const uint32_t end = clamped_start(starts, b + 1, tokens);
    r.first = clamped_start(starts, b, tokens);
    r.n = end > r.first ? end - r.first : 0;
    r.table = nullptr;
    if (!paged) {
        r.length = (int32_t)r.n;
        r.pos0 = 0;
        return r;
    }
    const int32_t s = seqs ? seqs[b] : (int32_t)b;
    r.length = 0;
    if (s >= 0 && (uint32_t)s < seq_count) {
        const int32_t most = (int32_t)(table_width << page_shift);
        const int32_t len = lengths[s];
        r.length = len < 0 ? 0 : len < most ? len : most;
        r.table = tables + (size_t)s * table_width;
    }
    r.pos0 = r.length - (int32_t)r.n;
    return r;
}

template <typename T>
__device__ __forceinline__ float to_float(T x) { return (float)x; }

#endif

}  // namespace pimdl
