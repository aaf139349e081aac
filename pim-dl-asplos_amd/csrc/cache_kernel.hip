// The paged cache for gfx950 (MI355X): writing new keys and values, and the bookkeeping and moving of pages (pimdl_cache_append,
// pimdl_pages_*).  The book -- tables, lengths and reference counts -- stays in device memory; what decides (which pages are free, in what
// order they are given out) is a scan by one workgroup, what touches many entries or moves pages is a launch over the whole device that follows
// lists which the scan left in the context's scratch.
#include "serve_common.h"

namespace pimdl {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------------------------------
// append: token t's columns, N at a time, rounded to nearest even and stored where its position lies.  One pass, bound by HBM: 8 prompts of up to 4000 tokens, 16 heads
// of 128, fp32 to bf16, 91 us, 5.4 TB/s; 64 single tokens 3.6 us, the launch.  us by 8 elements / by one: 16 heads of 128 91, of 31, an eighth of whose
// lanes' bytes each load takes, 92 for a quarter as much.
// ------------------------------------------------------------------------------------------------------------
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T x[N];
};

template <typename TI, typename TC, int N>
__global__ __launch_bounds__(256) void cache_append_kernel(const TI* __restrict__ k, const TI* __restrict__ v, pimdl_paged_cache c,
                                                           const int32_t* __restrict__ seqs, const int32_t* __restrict__ starts, uint32_t batch,
                                                           uint32_t tokens, uint32_t kv_stride, uint32_t page_shift)
{
    const uint32_t row = c.kv_heads * c.head_dim / N;  // packs of a token's row
    const uint64_t item = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
    const uint32_t t = (uint32_t)(item / row), part = (uint32_t)(item % row);
    if (t >= tokens || (c.lacking && *c.lacking != 0)) return;
    const Row r = load_row(starts, seqs, c.tables, c.lengths, tokens, c.seqs, c.table_width, page_shift, true, row_of_token(starts, batch, tokens, t));
    if (t < r.first || t - r.first >= r.n) return;
    const int32_t pos = r.pos0 + (int32_t)(t - r.first);
    if (pos < 0) return;
    const int32_t page = r.table[pos >> page_shift];
    if (page < 0 || (uint32_t)page >= c.pages) return;
    const uint32_t col = part * N, h = col / c.head_dim, d = col % c.head_dim;
    const size_t to = (((((size_t)page * c.kv_heads + h) << page_shift) + (pos & ((1u << page_shift) - 1))) * c.head_dim + d);
    const Pack<TI, N> ki = *reinterpret_cast<const Pack<TI, N>*>(k + (size_t)t * kv_stride + col);
    const Pack<TI, N> vi = *reinterpret_cast<const Pack<TI, N>*>(v + (size_t)t * kv_stride + col);
    Pack<TC, N> ko, vo;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        ko.x[i] = (TC)to_float(ki.x[i]);
        vo.x[i] = (TC)to_float(vi.x[i]);
    }
    *reinterpret_cast<Pack<TC, N>*>(static_cast<TC*>(c.k) + to) = ko;
    *reinterpret_cast<Pack<TC, N>*>(static_cast<TC*>(c.v) + to) = vo;
}

template <typename TI, typename TC>
int launch_append(Ctx* ctx, const pimdl_paged_cache& c, const int32_t* seqs, const int32_t* starts, uint32_t batch, uint32_t tokens, const void* k,
                  const void* v, uint32_t kv_stride)
{
    const bool packs = c.head_dim % 8 == 0 && kv_stride * sizeof(TI) % 16 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0;
    const uint64_t items = (uint64_t)tokens * c.kv_heads * c.head_dim / (packs ? 8 : 1);
    if (items > 65535ull * GRID_X * 256) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "pimdl_cache_append: too many elements for one launch");
    const dim3 grid = grid_of((items + 255) / 256);
    const uint32_t shift = (uint32_t)__builtin_ctz(c.page_tokens);
    const TI *ki = static_cast<const TI*>(k), *vi = static_cast<const TI*>(v);
    if (packs) hipLaunchKernelGGL((cache_append_kernel<TI, TC, 8>), grid, dim3(256), 0, ctx->stream, ki, vi, c, seqs, starts, batch, tokens, kv_stride, shift);
    else hipLaunchKernelGGL((cache_append_kernel<TI, TC, 1>), grid, dim3(256), 0, ctx->stream, ki, vi, c, seqs, starts, batch, tokens, kv_stride, shift);
    return hip_check(ctx, hipGetLastError(), "cache_append_kernel launch");
}

// ------------------------------------------------------------------------------------------------------------
// The book
// ------------------------------------------------------------------------------------------------------------
struct Book {
    int32_t *tables, *lengths, *refs, *lacking;
    uint32_t seqs, width, pages, page_tokens;
};
struct Pools {
    char* at[64];
    uint32_t count, layers;
    uint64_t layer_bytes, page_bytes;
};

Book book_of(const pimdl_page_book& b) { return {b.tables, b.lengths, b.refs, b.lacking, b.seqs, b.table_width, b.pages, b.page_tokens}; }
Pools pools_of(const pimdl_page_book& b)
{
    Pools p = {};
    p.count = b.pool_count, p.layers = b.layers, p.page_bytes = b.page_bytes, p.layer_bytes = b.page_bytes * b.pages;
    for (uint32_t i = 0; i < b.pool_count; ++i) p.at[i] = static_cast<char*>(b.pools[i]);
    return p;
}

constexpr int SCAN = 1024;  // threads of the workgroup that decides

// exclusive sum over the workgroup's threads; *total: all of it.  `tmp`: SCAN / 64 + 1 words
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* tmp, T* total)
{
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T y = __shfl_up(x, o);
        if (lane >= (uint32_t)o) x += y;
    }
    __syncthreads();  // (tmp may still be read from the call before)
    if (lane == 63) tmp[wave] = x;
    __syncthreads();
    if (wave == 0) {
        const uint32_t waves = blockDim.x >> 6;
        T w = lane < waves ? tmp[lane] : 0, s = w;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const T y = __shfl_up(s, o);
            if (lane >= (uint32_t)o) s += y;
        }
        if (lane < waves) tmp[lane] = s - w;
        if (lane == waves - 1) tmp[waves] = s;
    }
    __syncthreads();
    *total = tmp[blockDim.x >> 6];
    return tmp[wave] + x - v;
}

// Which of a thread's pages in the SCAN_EACH * SCAN from p0 on are free.  Asked for before anything that it does not wait for.
constexpr uint32_t SCAN_EACH = 8;
__device__ __forceinline__ uint32_t free_mask(const int32_t* refs, uint32_t pages, uint32_t p0)
{
    const uint32_t p = p0 + threadIdx.x * SCAN_EACH;
    uint32_t mask = 0;
#pragma unroll
    for (uint32_t i = 0; i < SCAN_EACH; ++i)
        if (p + i < pages && refs[p + i] == 0) mask |= 1u << i;
    return mask;
}
// The `want` lowest free pages into fresh[0 ..] (device memory or LDS); returns how many of them there are.  `mask`: free_mask of page 0.
__device__ __forceinline__ uint32_t lowest_free(const int32_t* refs, uint32_t pages, uint32_t want, uint32_t mask, int32_t* fresh, uint32_t* tmp)
{
    uint32_t found = 0;
    for (uint32_t p0 = 0; p0 < pages && found < want; p0 += SCAN * SCAN_EACH) {
        if (p0) mask = free_mask(refs, pages, p0);
        uint32_t total, at = found + block_scan<uint32_t>(__popc(mask), tmp, &total);
#pragma unroll
        for (uint32_t i = 0; i < SCAN_EACH; ++i)
            if (mask >> i & 1) {
                if (at < want) fresh[at] = (int32_t)(p0 + threadIdx.x * SCAN_EACH + i);
                ++at;
            }
        found += total;
    }
    __syncthreads();
    return found < want ? found : want;
}

// mark[s] = first place of sequence s in the list
__device__ __forceinline__ void first_places(const int32_t* list, uint32_t n, int32_t* mark, uint32_t seqs)
{
    for (uint32_t s = threadIdx.x; s < seqs; s += blockDim.x) mark[s] = 0x7fffffff;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const int32_t s = list[i];
        if (s >= 0 && (uint32_t)s < seqs) atomicMin(&mark[s], (int32_t)i);
    }
    __syncthreads();
}

__device__ __forceinline__ uint32_t pages_for(int64_t length, uint32_t page_tokens) { return (uint32_t)((length + page_tokens - 1) / page_tokens); }
__device__ __forceinline__ int32_t held_length(const Book& b, int32_t s)
{
    const int64_t len = b.lengths[s], most = (int64_t)b.width * b.page_tokens;
    return (int32_t)(len < 0 ? 0 : len < most ? len : most);
}
__device__ __forceinline__ int32_t short_of(uint64_t want, uint32_t found)
{
    const uint64_t d = want - found;
    return d > 0x7fffffffull ? 0x7fffffff : (int32_t)d;
}

__global__ __launch_bounds__(SCAN) void pages_reserve_kernel(Book b, const int32_t* __restrict__ seqs, const int32_t* __restrict__ counts, uint32_t n,
                                                             int32_t* fresh)
{
    extern __shared__ int32_t lds[];  // mark[seqs], base[n]
    __shared__ uint64_t tmp64[SCAN / 64 + 1];
    __shared__ uint32_t tmp32[SCAN / 64 + 1], too_long;
    __shared__ int32_t few[SCAN];  // the new pages, where they fit
    int32_t *mark = lds, *base = lds + b.seqs;
    const uint32_t mask = free_mask(b.refs, b.pages, 0);
    if (threadIdx.x == 0) too_long = 0;
    first_places(seqs, n, mark, b.seqs);
    auto grown = [&](uint32_t i, int32_t* s, int32_t* have) -> int64_t {  // the new length of entry i's sequence, or -1
        *s = seqs[i];
        if (*s < 0 || (uint32_t)*s >= b.seqs || mark[*s] != (int32_t)i) return -1;
        *have = held_length(b, *s);
        return (int64_t)*have + (counts[i] > 0 ? counts[i] : 0);
    };
    uint64_t want = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += SCAN) {
        const uint32_t i = i0 + threadIdx.x;
        uint64_t need = 0, total;
        int32_t s, have;
        if (i < n) {
            const int64_t len = grown(i, &s, &have);
            if (len > (int64_t)b.width * b.page_tokens) too_long = 1;
            else if (len >= 0) need = pages_for(len, b.page_tokens) - pages_for(have, b.page_tokens);
        }
        const uint64_t at = want + block_scan<uint64_t>(need, tmp64, &total);
        if (i < n) base[i] = (int32_t)(at < 0x7fffffffull ? at : 0x7fffffffull);
        want += total;
    }
    __syncthreads();
    if (too_long) {
        if (threadIdx.x == 0) *b.lacking = -1;
        return;
    }
    const uint32_t asked = (uint32_t)(want < b.pages ? want : b.pages);
    if (asked <= SCAN) fresh = few;
    const uint32_t found = lowest_free(b.refs, b.pages, asked, mask, fresh, tmp32);
    if (found < want) {
        if (threadIdx.x == 0) *b.lacking = short_of(want, found);
        return;
    }
    for (uint32_t t = threadIdx.x; t < found; t += SCAN) {
        uint32_t lo = 0, hi = n;  // the last entry that begins at or before page t
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if ((uint32_t)base[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int32_t s = seqs[lo], page = fresh[t];
        b.tables[(size_t)s * b.width + pages_for(held_length(b, s), b.page_tokens) + (t - (uint32_t)base[lo])] = page;
        b.refs[page] = 1;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += SCAN) {
        int32_t s, have;
        const int64_t len = grown(i, &s, &have);
        if (len >= 0) b.lengths[s] = (int32_t)len;
    }
    if (threadIdx.x == 0) *b.lacking = 0;
}

// ---- copies of pages: `count` pairs, a workgroup 16 KiB of one pair in one layer of one buffer at a time: its loads all asked for before the first store
constexpr uint32_t COPY_BYTES = 16384;

__device__ __forceinline__ void copy_pages(const Pools& pl, const int32_t* src, const int32_t* dst, uint32_t count, uint32_t pages, uint32_t block,
                                           uint32_t blocks)
{
    const uint32_t pieces = (uint32_t)((pl.page_bytes + COPY_BYTES - 1) / COPY_BYTES);
    const uint64_t per_pair = (uint64_t)pieces * pl.count * pl.layers, items = per_pair * count;
    for (uint64_t it = block; it < items; it += blocks) {
        const uint32_t pair = (uint32_t)(it / per_pair), rest = (uint32_t)(it % per_pair);
        const uint32_t piece = rest % pieces, slot = rest / pieces;
        const int32_t s = src[pair], d = dst[pair];
        if (s < 0 || d < 0 || (uint32_t)s >= pages || (uint32_t)d >= pages || s == d) continue;
        char* pool = pl.at[slot / pl.layers] + (size_t)(slot % pl.layers) * pl.layer_bytes;
        const uint64_t at = (uint64_t)piece * COPY_BYTES;
        const u32x4* from = reinterpret_cast<const u32x4*>(pool + (size_t)s * pl.page_bytes + at);
        u32x4* to = reinterpret_cast<u32x4*>(pool + (size_t)d * pl.page_bytes + at);
        const uint32_t vecs = (uint32_t)((pl.page_bytes - at < COPY_BYTES ? pl.page_bytes - at : COPY_BYTES) / 16);
        u32x4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (threadIdx.x + 256 * i < vecs) x[i] = from[threadIdx.x + 256 * i];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (threadIdx.x + 256 * i < vecs) to[threadIdx.x + 256 * i] = x[i];
    }
}

__global__ __launch_bounds__(256) void pages_copy_kernel(Pools pl, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, uint32_t n, uint32_t pages)
{
    copy_pages(pl, src, dst, n, pages, blockIdx.x, gridDim.x);
}

// ---- fork: one workgroup decides (6.5 us for 32 entries, a chain of loads: the list, the parent's length, its last page, the counts), the device copies (7.6 us for
// 19 MB in 12 layers); each waits for the launch before more than for memory.
// take[i]: the page that entry i's partly filled last page is copied to, -1 where there is none, -2 where the entry is left out; length[i]: of
// its parent before the call (which may be another entry's child: then 0)
struct ForkLists {
    int32_t *fresh, *take, *length, *src, *dst, *count;
};

__global__ __launch_bounds__(SCAN) void pages_fork_kernel(Book b, const int32_t* __restrict__ parents, const int32_t* __restrict__ children, uint32_t n,
                                                          ForkLists f)
{
    extern __shared__ int32_t lds[];  // mark[seqs]
    __shared__ uint32_t tmp[SCAN / 64 + 1];
    __shared__ int32_t few[SCAN];  // the new pages, where they fit
    int32_t* mark = lds;
    const uint32_t mask = free_mask(b.refs, b.pages, 0);
    first_places(children, n, mark, b.seqs);
    // the last page of entry i's parent if partly filled, -1: none, -2: the entry is left out
    auto last_page = [&](uint32_t i, int32_t* len) -> int32_t {
        const int32_t p = parents[i], c = children[i];
        *len = 0;
        if (p < 0 || (uint32_t)p >= b.seqs || c < 0 || (uint32_t)c >= b.seqs || mark[c] != (int32_t)i || b.lengths[c] != 0) return -2;
        *len = held_length(b, p);
        if (*len % b.page_tokens == 0) return -1;
        const int32_t page = b.tables[(size_t)p * b.width + *len / b.page_tokens];
        return page >= 0 && (uint32_t)page < b.pages ? page : -1;
    };
    uint32_t want = 0, at = 0, total;
    int32_t page = -2, len = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += SCAN) {
        const uint32_t i = i0 + threadIdx.x;
        page = i < n ? last_page(i, &len) : -2;
        at = want + block_scan<uint32_t>(page >= 0, tmp, &total);
        if (n > SCAN && i < n) {  // (else they stay in registers)
            if (page >= 0) f.src[at] = page;
            f.take[i] = page >= 0 ? (int32_t)at : page;
            f.length[i] = len;
        }
        want += total;
    }
    const uint32_t asked = want < b.pages ? want : b.pages;
    int32_t* const fresh = asked <= SCAN ? few : f.fresh;
    const uint32_t found = lowest_free(b.refs, b.pages, asked, mask, fresh, tmp);
    const bool done = found == want;
    if (n <= SCAN) {
        if (threadIdx.x < n) {
            const int32_t take = !done ? -2 : page >= 0 ? fresh[at] : page;
            f.take[threadIdx.x] = take;
            f.length[threadIdx.x] = len;
            if (take >= 0) {
                f.src[at] = page;
                f.dst[at] = take;
                b.refs[take] = 1;
            }
        }
    } else {
        for (uint32_t i = threadIdx.x; i < n; i += SCAN) {
            if (!done) f.take[i] = -2;
            else if (f.take[i] >= 0) f.take[i] = fresh[f.take[i]];
        }
        if (done)
            for (uint32_t t = threadIdx.x; t < want; t += SCAN) {
                f.dst[t] = fresh[t];
                b.refs[fresh[t]] = 1;
            }
    }
    if (threadIdx.x == 0) {
        *f.count = done ? (int32_t)want : 0;
        *b.lacking = short_of(want, found);
    }
}

// blocks 0 .. n * row_blocks - 1: the children's rows, 1024 entries each; the others: the copies
__global__ __launch_bounds__(256) void pages_fork_apply_kernel(Book b, Pools pl, const int32_t* __restrict__ parents, const int32_t* __restrict__ children,
                                                               uint32_t n, uint32_t row_blocks, ForkLists f)
{
    if (blockIdx.x >= n * row_blocks) {
        copy_pages(pl, f.src, f.dst, (uint32_t)*f.count, b.pages, blockIdx.x - n * row_blocks, gridDim.x - n * row_blocks);
        return;
    }
    const uint32_t i = blockIdx.x / row_blocks, j0 = blockIdx.x % row_blocks * 1024;
    const int32_t take = f.take[i];
    if (take == -2) return;
    const int32_t p = parents[i], c = children[i], len = f.length[i];
    const uint32_t whole = (uint32_t)len / b.page_tokens;
    const int32_t* from = b.tables + (size_t)p * b.width;
    int32_t* to = b.tables + (size_t)c * b.width;
    for (uint32_t j = j0 + threadIdx.x; j < j0 + 1024 && j < whole; j += 256) {
        const int32_t page = from[j];
        to[j] = page;
        if (page >= 0 && (uint32_t)page < b.pages) atomicAdd(&b.refs[page], 1);
    }
    if (j0 == 0 && threadIdx.x == 0) {
        if (take >= 0) to[whole] = take;
        b.lengths[c] = len;
    }
}

// A sequence that is listed twice gives its pages back once: whoever takes an entry out of the row lowers the count.
__global__ __launch_bounds__(256) void pages_free_kernel(Book b, const int32_t* __restrict__ seqs)
{
    const int32_t s = seqs[blockIdx.y];
    if (s < 0 || (uint32_t)s >= b.seqs) return;
    int32_t* row = b.tables + (size_t)s * b.width;
    for (uint32_t j = blockIdx.x * 1024 + threadIdx.x; j < blockIdx.x * 1024 + 1024 && j < b.width; j += 256) {
        if (row[j] == -1) continue;
        const int32_t page = atomicExch(&row[j], -1);
        if (page >= 0 && (uint32_t)page < b.pages) atomicSub(&b.refs[page], 1);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) b.lengths[s] = 0;
}

// ---- compaction.  rank(p): pages in use before p; L: pages in use.  The page at p >= L is the (rank(p) - rank(L))-th to move, the free
// place p < L the (p - rank(p))-th to be filled.  Ranks take two launches of 4.5 us; moving a third of 4096 pages in 12 layers 288 us, read and
// written at 5.0 TB/s.
constexpr uint32_t COMPACT_PAGES = 1024;  // that a workgroup looks at
struct CompactLists {
    int32_t *counts, *holes, *mover, *rank, *meta;  // in use per workgroup; places by order; pages by rank; rank by page; L and rank(L)
};

__global__ __launch_bounds__(256) void pages_count_kernel(Book b, int32_t* __restrict__ counts)
{
    __shared__ uint32_t tmp[5];
    uint32_t live = 0, total;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t p = blockIdx.x * COMPACT_PAGES + i * 256 + threadIdx.x;
        live += p < b.pages && b.refs[p] != 0;
    }
    block_scan<uint32_t>(live, tmp, &total);
    if (threadIdx.x == 0) counts[blockIdx.x] = (int32_t)total;
}

__global__ __launch_bounds__(256) void pages_rank_kernel(Book b, CompactLists c)
{
    __shared__ uint32_t tmp[5];
    uint32_t mine = 0, before = 0, all, at;
    for (uint32_t i = threadIdx.x; i < gridDim.x; i += 256) {
        mine += (uint32_t)c.counts[i];
        if (i < blockIdx.x) before += (uint32_t)c.counts[i];
    }
    block_scan<uint32_t>(mine, tmp, &all);
    block_scan<uint32_t>(before, tmp, &at);
    uint32_t mask = 0, total;
    const uint32_t p0 = blockIdx.x * COMPACT_PAGES + threadIdx.x * 4;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (p0 + i < b.pages && b.refs[p0 + i] != 0) mask |= 1u << i;
    uint32_t rank = at + block_scan<uint32_t>(__popc(mask), tmp, &total);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t p = p0 + i;
        const bool live = mask >> i & 1;
        if (p < b.pages) {
            if (p == all) c.meta[1] = (int32_t)rank;
            if (p < all && !live) c.holes[p - rank] = (int32_t)p;
            if (p >= all) {
                c.rank[p] = live ? (int32_t)rank : -1;
                if (live) c.mover[rank] = (int32_t)p;
            }
        }
        rank += live;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        c.meta[0] = (int32_t)all;
        if (all == b.pages) c.meta[1] = (int32_t)all;
    }
}

__global__ __launch_bounds__(256) void pages_compact_kernel(Book b, Pools pl, CompactLists c)
{
    const uint32_t live = (uint32_t)c.meta[0], first = (uint32_t)c.meta[1], moves = live - first;
    copy_pages(pl, c.mover + first, c.holes, moves, b.pages, blockIdx.x, gridDim.x);
    const uint64_t entries = (uint64_t)b.seqs * b.width;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (uint64_t)gridDim.x * 256) {
        const int32_t page = b.tables[i];
        if (page < (int32_t)live || (uint32_t)page >= b.pages) continue;
        const int32_t rank = c.rank[page];
        if (rank >= 0) b.tables[i] = c.holes[(uint32_t)rank - first];
    }
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < moves; i += gridDim.x * 256) {
        const int32_t from = c.mover[first + i], to = c.holes[i];
        b.refs[to] = b.refs[from];
        b.refs[from] = 0;
    }
}

// workgroups of a copy of up to `pairs` pages: enough to fill the device, no more than there is work
uint32_t copy_blocks(const Ctx* ctx, const Pools& p, uint64_t pairs)
{
    const uint64_t items = pairs * p.count * p.layers * ((p.page_bytes + COPY_BYTES - 1) / COPY_BYTES), most = (uint64_t)ctx->prop.multiProcessorCount * 8;
    return (uint32_t)(items < most ? items : most);
}

int book_scratch(Ctx* ctx, size_t ints, int32_t** out)
{
    int rc = ensure_scratch(ctx, &ctx->d_book, &ctx->book_bytes, ints * 4, "page lists");
    *out = reinterpret_cast<int32_t*>(ctx->d_book);
    return rc;
}

}  // namespace

int launch_cache_append(Ctx* ctx, const pimdl_paged_cache& c, const int32_t* seqs, const int32_t* starts, uint32_t batch, uint32_t tokens,
                        const void* k, const void* v, uint32_t kv_stride, uint32_t dtype)
{
    if (dtype == PIMDL_BF16) return launch_append<__bf16, __bf16>(ctx, c, seqs, starts, batch, tokens, k, v, kv_stride);
    if (dtype == PIMDL_F16) return launch_append<_Float16, _Float16>(ctx, c, seqs, starts, batch, tokens, k, v, kv_stride);
    if (c.dtype == PIMDL_BF16) return launch_append<float, __bf16>(ctx, c, seqs, starts, batch, tokens, k, v, kv_stride);
    if (c.dtype == PIMDL_F16) return launch_append<float, _Float16>(ctx, c, seqs, starts, batch, tokens, k, v, kv_stride);
    return launch_append<float, float>(ctx, c, seqs, starts, batch, tokens, k, v, kv_stride);
}

int launch_pages_reserve(Ctx* ctx, const pimdl_page_book& b, const int32_t* seqs, const int32_t* counts, uint32_t n)
{
    int32_t* fresh;
    int rc = book_scratch(ctx, b.pages, &fresh);
    if (!rc) rc = allow_dynamic_lds(ctx, reinterpret_cast<const void*>(pages_reserve_kernel), 2 * 16384 * 4, "pages_reserve_kernel LDS");
    if (rc) return rc;
    hipLaunchKernelGGL(pages_reserve_kernel, dim3(1), dim3(SCAN), (b.seqs + n) * 4, ctx->stream, book_of(b), seqs, counts, n, fresh);
    return hip_check(ctx, hipGetLastError(), "pages_reserve_kernel launch");
}

int launch_pages_fork(Ctx* ctx, const pimdl_page_book& b, const int32_t* parents, const int32_t* children, uint32_t n)
{
    int32_t* s;
    int rc = book_scratch(ctx, 5 * (size_t)n + 1, &s);
    if (!rc) rc = allow_dynamic_lds(ctx, reinterpret_cast<const void*>(pages_fork_kernel), 16384 * 4, "pages_fork_kernel LDS");
    if (rc) return rc;
    const ForkLists f = {s + 1, s + 1 + n, s + 1 + 2 * (size_t)n, s + 1 + 3 * (size_t)n, s + 1 + 4 * (size_t)n, s};
    const Book book = book_of(b);
    const Pools p = pools_of(b);
    const uint32_t row_blocks = (b.table_width + 1023) / 1024;
    const uint64_t blocks = (uint64_t)n * row_blocks + copy_blocks(ctx, p, n);
    if (!fits_launch(blocks, 256)) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "pimdl_pages_fork: rows of %u pages, %u of them", b.table_width, n);
    hipLaunchKernelGGL(pages_fork_kernel, dim3(1), dim3(SCAN), b.seqs * 4, ctx->stream, book, parents, children, n, f);
    if ((rc = hip_check(ctx, hipGetLastError(), "pages_fork_kernel launch")) || n == 0) return rc;
    hipLaunchKernelGGL(pages_fork_apply_kernel, dim3((uint32_t)blocks), dim3(256), 0, ctx->stream, book, p, parents, children, n, row_blocks, f);
    return hip_check(ctx, hipGetLastError(), "pages_fork_apply_kernel launch");
}

int launch_pages_free(Ctx* ctx, const pimdl_page_book& b, const int32_t* seqs, uint32_t n)
{
    hipLaunchKernelGGL(pages_free_kernel, dim3((b.table_width + 1023) / 1024, n), dim3(256), 0, ctx->stream, book_of(b), seqs);
    return hip_check(ctx, hipGetLastError(), "pages_free_kernel launch");
}

int launch_pages_compact(Ctx* ctx, const pimdl_page_book& b)
{
    const uint32_t blocks = (b.pages + COMPACT_PAGES - 1) / COMPACT_PAGES;
    int32_t* s;
    int rc = book_scratch(ctx, 2 + blocks + 3 * (size_t)b.pages, &s);
    if (rc) return rc;
    const CompactLists c = {s + 2, s + 2 + blocks, s + 2 + blocks + (size_t)b.pages, s + 2 + blocks + 2 * (size_t)b.pages, s};
    const Book book = book_of(b);
    const Pools p = pools_of(b);
    hipLaunchKernelGGL(pages_count_kernel, dim3(blocks), dim3(256), 0, ctx->stream, book, c.counts);
    if ((rc = hip_check(ctx, hipGetLastError(), "pages_count_kernel launch"))) return rc;
    hipLaunchKernelGGL(pages_rank_kernel, dim3(blocks), dim3(256), 0, ctx->stream, book, c);
    if ((rc = hip_check(ctx, hipGetLastError(), "pages_rank_kernel launch"))) return rc;
    const uint64_t entries = ((uint64_t)b.seqs * b.table_width + 255) / 256;
    const uint32_t most = (uint32_t)ctx->prop.multiProcessorCount * 8, work = copy_blocks(ctx, p, b.pages / 2 + 1);
    const uint32_t grid = work > entries ? work : (uint32_t)(entries < most ? entries : most);
    hipLaunchKernelGGL(pages_compact_kernel, dim3(grid), dim3(256), 0, ctx->stream, book, p, c);
    return hip_check(ctx, hipGetLastError(), "pages_compact_kernel launch");
}

int launch_pages_copy(Ctx* ctx, const pimdl_page_book& b, const int32_t* src, const int32_t* dst, uint32_t n)
{
    const Pools p = pools_of(b);
    const uint32_t blocks = copy_blocks(ctx, p, n);
    if (blocks == 0) return PIMDL_OK;
    hipLaunchKernelGGL(pages_copy_kernel, dim3(blocks), dim3(256), 0, ctx->stream, p, src, dst, n, b.pages);
    return hip_check(ctx, hipGetLastError(), "pages_copy_kernel launch");
}

}  // namespace pimdl
