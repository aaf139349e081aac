// Trees of drafted tokens for gfx950 (MI355X): who is whose ancestor (pimdl_tree_build), and the end of a sequence behind the chosen branch (pimdl_pages_accept).
#include "serve_common.h"

namespace pimdl {

namespace {

// ------------------------------------------------------------------------------------------------------------
// Ancestors by doubling: mask(i), which holds i and its next d ancestors, and the ancestor j after those give mask(i) | mask(j), for 2 d, in as many rounds as the
// longest branch has bits.  A workgroup takes a row of the batch, a thread a node, whose mask is in registers for itself and in LDS for its descendants.
// ------------------------------------------------------------------------------------------------------------
template <int WORDS>
__global__ __launch_bounds__(WORDS < 2 ? 64 : WORDS * 32) void tree_build_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ starts, uint32_t tokens,
                                                                                 uint32_t words, uint32_t* __restrict__ masks, int32_t* __restrict__ depths)
{
    constexpr uint32_t NODES = WORDS * 32, PITCH = WORDS | 1;  // (rows of even pitch would meet in few banks)
    __shared__ uint32_t seen[NODES * PITCH];
    __shared__ int32_t next[NODES];
    const uint32_t first = clamped_start(starts, blockIdx.x, tokens), end = clamped_start(starts, blockIdx.x + 1, tokens);
    const uint32_t n = end > first ? end - first : 0, i = threadIdx.x;
    if (n > 32 * words) {
        for (uint64_t at = i; at < (uint64_t)n * words; at += blockDim.x) masks[(uint64_t)first * words + at] = 0;
        for (uint32_t t = i; t < n; t += blockDim.x) depths[first + t] = 0;
        return;
    }
    uint32_t mine[WORDS];
    int32_t to = -1;
    if (i < n) {
        to = parents[first + i];
        if (to < 0 || to >= (int32_t)i) to = -1;
    }
#pragma unroll
    for (int w = 0; w < WORDS; ++w) mine[w] = i < n && i / 32 == (uint32_t)w ? 1u << (i & 31) : 0u;
    if (i < NODES) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w) seen[i * PITCH + w] = mine[w];
        next[i] = to;
    }
    while (__syncthreads_or(to >= 0)) {
        if (to >= 0) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) mine[w] |= seen[to * PITCH + w];
            to = next[to];
        }
        __syncthreads();
        if (i < n) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) seen[i * PITCH + w] = mine[w];
            next[i] = to;
        }
    }
    if (i < n) {
        int32_t depth = -1;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) depth += __popc(mine[w]);
        depths[first + i] = depth;
    }
    // out of LDS in the order of memory: a word of each lane's own mask would be 64 lines a store (64 trees of 512 nodes 10.4 us, this way 7.3)
    uint32_t* const out = masks + (uint64_t)first * words;
    for (uint32_t at = i; at < n * words; at += blockDim.x) {
        const uint32_t node = words == WORDS ? at / WORDS : at / words;
        out[at] = seen[node * PITCH + at - node * words];
    }
}

template <int WORDS>
int launch_build(Ctx* ctx, const int32_t* parents, const int32_t* starts, uint32_t batch, uint32_t tokens, uint32_t words, uint32_t* masks, int32_t* depths)
{
    hipLaunchKernelGGL((tree_build_kernel<WORDS>), dim3(batch), dim3(WORDS < 2 ? 64 : WORDS * 32), 0, ctx->stream, parents, starts, tokens, words, masks, depths);
    return hip_check(ctx, hipGetLastError(), "tree_build_kernel launch");
}

// ------------------------------------------------------------------------------------------------------------
// Accepting a branch, in two launches: rows move, then the book follows, since every workgroup of the first reads tables and counts that the second changes.
// The branch is the set bits of its last node's mask, in order; its j-th node moves to place j, which is never behind its own.  A thread of the first launch owns a
// part of a row (of one head, layer and pool) and moves that of every node in order, ACCEPT_AHEAD of them asked for before the first is stored: none of them is a place
// that has been written, as later nodes lie behind all places up to their own.
// Memory bounds it, and the longest branch: those of 64 trees in 12 layers, 8 heads of 128, bf16, up to 82 rows that move, 158 MB, take 41 us (3.9 TB/s; a plain copy reaches 4.8), 16
// rows ahead 40; in workgroups of 256 threads, half as many CUs to a branch, 48, of 64, each of which finds out the same, 44; the book 4 us.  One branch alone waits for memory five
// times in a row: 6.4 us.
// ------------------------------------------------------------------------------------------------------------
struct AcceptArgs {
    const int32_t *seqs, *starts, *last, *lengths, *refs, *lacking, *tables;
    const uint32_t* masks;
    int32_t* kept;
    uint32_t batch, tokens, words, seq_count, width, pages, page_tokens;
};
struct AcceptPools {
    char* at[64];
    uint32_t count, layers, runs, row_bytes;  // runs: of page_tokens rows in a page
    uint64_t page_bytes, layer_bytes;
};
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));  // (an array of HIP's own uint4 would be in scratch)
constexpr uint32_t ACCEPT_NODES = 1024, ACCEPT_AHEAD = 8, ACCEPT_THREADS = 128;

template <typename T>
__global__ __launch_bounds__(ACCEPT_THREADS) void pages_accept_kernel(AcceptArgs a, AcceptPools pl)
{
    __shared__ uint64_t from[ACCEPT_NODES], to[ACCEPT_NODES];  // of the rows that move: first byte in a layer's buffer, of a page's first run
    __shared__ int32_t path[ACCEPT_NODES];
    __shared__ uint32_t before[33], unmoved, wrong, others;  // others: have a page that this would change (a flag of its own: `wrong` may still be read then)
    const uint32_t tid = threadIdx.x, b = blockIdx.y;
    const int32_t s = a.seqs ? a.seqs[b] : (int32_t)b, last = a.last[b];
    const uint32_t first = clamped_start(a.starts, b, a.tokens), end = clamped_start(a.starts, b + 1, a.tokens), n = end > first ? end - first : 0;
    if (tid == 0) unmoved = 0, wrong = 0, others = 0;
    __syncthreads();
    const bool there = s >= 0 && (uint32_t)s < a.seq_count;
    int64_t length = 0;
    if (there) {
        const int64_t most = (int64_t)a.width * a.page_tokens;
        length = a.lengths[s];
        length = length < 0 ? 0 : length < most ? length : most;
    }
    const int64_t base = length - n;
    if (tid == 0 && (*a.lacking != 0 || !there || base < 0 || n > 32 * a.words || last < -1 || last >= (int32_t)n)) wrong = 1;
    if (a.seqs)
        for (uint32_t i = tid; i < b; i += ACCEPT_THREADS)
            if (a.seqs[i] == s) wrong = 1;  // (who comes first)
    __syncthreads();
    if (wrong) {
        if (blockIdx.x == 0 && tid == 0) a.kept[b] = -1;
        return;
    }
    const uint32_t* const mask = a.masks + (uint64_t)(first + (last < 0 ? 0 : last)) * a.words;
    auto word_of = [&](uint32_t w) {  // nodes up to the last one
        const int32_t top = last - 32 * (int32_t)w;
        return top < 0 ? 0u : mask[w] & (top >= 31 ? ~0u : (2u << top) - 1);
    };
    if (tid < 64) {
        uint32_t x = tid < a.words ? __popc(word_of(tid)) : 0;
        const uint32_t own = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up(x, o);
            if (tid >= (uint32_t)o) x += y;
        }
        if (tid < 32) before[tid] = x - own;
        if (tid == 31) before[32] = x;
    }
    __syncthreads();
    const uint32_t count = before[32];
    if (last >= 0)
        for (uint32_t i = tid; i <= (uint32_t)last; i += ACCEPT_THREADS) {
            const uint32_t word = word_of(i / 32), bit = 1u << (i & 31);
            if (word & bit) path[before[i / 32] + __popc(word & (bit - 1))] = (int32_t)i;
        }
    __syncthreads();
    if (tid == 0 && last >= 0 && (count == 0 || path[count - 1] != last)) wrong = 1;  // its own bit is not there
    for (uint32_t j = tid; j < count; j += ACCEPT_THREADS)
        if (path[j] == (int32_t)j) atomicAdd(&unmoved, 1u);  // (the first ones: a node behind one that moves lies behind its place)
    __syncthreads();
    if (wrong) {
        if (blockIdx.x == 0 && tid == 0) a.kept[b] = -1;
        return;
    }
    const int32_t* const table = a.tables + (size_t)s * a.width;
    if (n) {
        const uint32_t p0 = (uint32_t)((base + unmoved) / a.page_tokens), p1 = (uint32_t)((base + count + a.page_tokens - 1) / a.page_tokens);
        for (uint32_t p = p0 + tid; p < p1; p += ACCEPT_THREADS) {
            const int32_t page = table[p];
            if (page >= 0 && (uint32_t)page < a.pages && a.refs[page] > 1) others = 1;
        }
    }
    auto byte_of = [&](int64_t place) -> int64_t {
        const int32_t page = table[place / a.page_tokens];
        return page < 0 || (uint32_t)page >= a.pages ? -1 : (int64_t)(page * pl.page_bytes + place % a.page_tokens * pl.row_bytes);
    };
    for (uint32_t j = unmoved + tid; j < count; j += ACCEPT_THREADS) {
        const int64_t f = byte_of(base + path[j]), t = byte_of(base + j);
        // (a row on no page is not there: what would move from it or to it stays)
        from[j - unmoved] = f < 0 || t < 0 ? 0 : (uint64_t)f;
        to[j - unmoved] = f < 0 || t < 0 ? ~0ull : (uint64_t)t;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) a.kept[b] = others ? -1 : (int32_t)count;
    if (others) return;
    const uint32_t rows = count - unmoved, parts = pl.row_bytes / (uint32_t)sizeof(T);
    const uint64_t columns = (uint64_t)parts * pl.runs * pl.layers * pl.count, run_bytes = (uint64_t)a.page_tokens * pl.row_bytes;
    if (rows == 0) return;
    for (uint64_t c = (uint64_t)blockIdx.x * ACCEPT_THREADS + tid; c < columns; c += (uint64_t)gridDim.x * ACCEPT_THREADS) {
        const uint32_t part = (uint32_t)(c % parts), rest = (uint32_t)(c / parts), run = rest % pl.runs, slot = rest / pl.runs;
        char* const at = pl.at[slot / pl.layers] + (size_t)(slot % pl.layers) * pl.layer_bytes + run * run_bytes + (size_t)part * sizeof(T);
        for (uint32_t j0 = 0; j0 < rows; j0 += ACCEPT_AHEAD) {
            typename std::conditional<sizeof(T) < 4, uint32_t, T>::type x[ACCEPT_AHEAD];
#pragma unroll
            for (uint32_t j = 0; j < ACCEPT_AHEAD; ++j) x[j] = *reinterpret_cast<const T*>(at + from[j0 + j < rows ? j0 + j : rows - 1]);
#pragma unroll
            for (uint32_t j = 0; j < ACCEPT_AHEAD; ++j) {
                const uint64_t place = to[j0 + j < rows ? j0 + j : rows - 1];
                asm("" : "+v"(x[j]));  // (or the compiler asks for it in the branch, behind all others)
                if (j0 + j < rows && place != ~0ull) *reinterpret_cast<T*>(at + place) = (T)x[j];
            }
        }
    }
}

__global__ __launch_bounds__(64) void pages_accept_book_kernel(AcceptArgs a, int32_t* tables, int32_t* lengths, int32_t* refs)
{
    const uint32_t b = blockIdx.x;
    const int32_t kept = a.kept[b];
    if (kept < 0) return;
    const int32_t s = a.seqs ? a.seqs[b] : (int32_t)b;
    const uint32_t first = clamped_start(a.starts, b, a.tokens), end = clamped_start(a.starts, b + 1, a.tokens), n = end > first ? end - first : 0;
    if (n == 0) return;
    const int64_t most = (int64_t)a.width * a.page_tokens, held = lengths[s], old = held < 0 ? 0 : held < most ? held : most, length = old - n + kept;
    const uint32_t p0 = (uint32_t)((length + a.page_tokens - 1) / a.page_tokens), p1 = (uint32_t)((old + a.page_tokens - 1) / a.page_tokens);
    int32_t* const row = tables + (size_t)s * a.width;
    for (uint32_t p = p0 + threadIdx.x; p < p1; p += 64) {
        const int32_t page = row[p];
        row[p] = -1;
        if (page >= 0 && (uint32_t)page < a.pages) atomicSub(&refs[page], 1);
    }
    if (threadIdx.x == 0) lengths[s] = (int32_t)length;
}

template <typename T>
int launch_accept(Ctx* ctx, const AcceptArgs& a, const AcceptPools& pl)
{
    // workgroups enough for the device, no more than there are columns
    const uint64_t columns = (uint64_t)(pl.row_bytes / sizeof(T)) * pl.runs * pl.layers * pl.count, blocks = (columns + ACCEPT_THREADS - 1) / ACCEPT_THREADS;
    if (columns > 0xffffffffu) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "pimdl_pages_accept: more parts of rows than 2^32");
    const uint64_t most = ((uint64_t)ctx->prop.multiProcessorCount * 16 + a.batch - 1) / a.batch;
    const uint32_t grid = (uint32_t)(blocks == 0 ? 1 : blocks < most ? blocks : most);
    hipLaunchKernelGGL((pages_accept_kernel<T>), dim3(grid, a.batch), dim3(ACCEPT_THREADS), 0, ctx->stream, a, pl);
    return hip_check(ctx, hipGetLastError(), "pages_accept_kernel launch");
}

}  // namespace

int launch_tree_build(Ctx* ctx, const int32_t* parents, const int32_t* starts, uint32_t batch, uint32_t tokens, uint32_t words, uint32_t* masks,
                      int32_t* depths)
{
    if (words <= 1) return launch_build<1>(ctx, parents, starts, batch, tokens, words, masks, depths);
    if (words <= 2) return launch_build<2>(ctx, parents, starts, batch, tokens, words, masks, depths);
    if (words <= 4) return launch_build<4>(ctx, parents, starts, batch, tokens, words, masks, depths);
    if (words <= 8) return launch_build<8>(ctx, parents, starts, batch, tokens, words, masks, depths);
    if (words <= 16) return launch_build<16>(ctx, parents, starts, batch, tokens, words, masks, depths);
    return launch_build<32>(ctx, parents, starts, batch, tokens, words, masks, depths);
}

int launch_pages_accept(Ctx* ctx, const pimdl_page_book& b, const int32_t* seqs, const int32_t* starts, uint32_t batch, uint32_t tokens,
                        const pimdl_tree& tree, const int32_t* last, uint32_t row_bytes, int32_t* kept)
{
    const AcceptArgs a = {seqs, starts, last, b.lengths, b.refs, b.lacking, b.tables, tree.masks, kept, batch, tokens, tree.words, b.seqs, b.table_width, b.pages, b.page_tokens};
    AcceptPools pl = {};
    pl.count = b.pool_count, pl.layers = b.layers, pl.row_bytes = row_bytes;
    pl.runs = (uint32_t)(b.pool_count ? b.page_bytes / ((uint64_t)b.page_tokens * row_bytes) : 0);
    pl.page_bytes = b.page_bytes, pl.layer_bytes = b.page_bytes * b.pages;
    for (uint32_t i = 0; i < b.pool_count; ++i) pl.at[i] = static_cast<char*>(b.pools[i]);
    int rc;
    if (row_bytes % 16 == 0) rc = launch_accept<u32x4>(ctx, a, pl);
    else if (row_bytes % 4 == 0) rc = launch_accept<uint32_t>(ctx, a, pl);
    else if (row_bytes % 2 == 0) rc = launch_accept<uint16_t>(ctx, a, pl);
    else rc = launch_accept<uint8_t>(ctx, a, pl);
    if (rc) return rc;
    hipLaunchKernelGGL(pages_accept_book_kernel, dim3(batch), dim3(64), 0, ctx->stream, a, b.tables, b.lengths, b.refs);
    return hip_check(ctx, hipGetLastError(), "pages_accept_book_kernel launch");
}

}  // namespace pimdl
