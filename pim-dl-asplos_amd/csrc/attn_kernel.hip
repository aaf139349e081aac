// Attention of a ragged batch over a window or a paged cache for gfx950 (MI355X): see pimdl_attention_window and
// pimdl_attention_paged.
#include <algorithm>

#include "attn_body.h"

namespace pimdl {

namespace {

using attn::LOG2E;

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// ---------------------------------------------------------------------------------------------
// Any head size up to 256, any stride and alignment: a workgroup takes one query of one head, its four waves blocks of 64 keys in turn, each with the
// running maximum m and sum l of a streaming softmax: a block with maximum m' gives o = o 2^(c (m - m')) + sum p v, l = l 2^(c (m - m')) + sum p,
// p = 2^(c (s - m')), s being raw products (times the scale's sign) and c = |scale| log2(e).  Eight lanes share a key and read its row N elements each, 8 keys at once, so that a load takes whole lines; lane (key j, eighth e) has columns
// (8 c + e) N + i of q, and of the sums over its keys, which are added up over lanes and waves at the end.  Bound by the loads' latency, so eight of them are asked
// for before the first is used: 32 sequences of up to 4000, 16 heads over 4, bf16, of 256 dims 141 us (210 where the compiler waits for each; 327 MB of keys and values, 4 times from
// L2), of 72 73 us, 48 37 us, 70 (elements of 2 bytes) 170 us; a window of 257 of 4 x 750 tokens, 12 heads of 72, fp32, 611 us, where matrix instructions
// take 68 for 80.
// ---------------------------------------------------------------------------------------------
template <typename TQ, typename TK, bool PAGED, int N, int DIMS>
__global__ __launch_bounds__(256, DIMS == 256 ? 2 : 3) void attention_plain_kernel(AttnArgs a)
{
    constexpr int CHUNKS = DIMS / (8 * N), BATCH = CHUNKS < 8 ? CHUNKS : 8, AHEAD = 8 / BATCH;  // loads of a row, and rows, under way together
    // a load, taken as bits: what is not there is cleared by a mask, for which the compiler does not take the load apart or put it behind a branch
    typedef typename std::conditional<N * sizeof(TK) == 16, attn::u32x4, typename std::conditional<sizeof(TK) == 4, uint32_t, uint16_t>::type>::type Bits;
    struct Pack {
        TK x[N];
    };
    static_assert(sizeof(Bits) == sizeof(Pack), "a load holds N elements");
    __shared__ float sums[4][DIMS];
    __shared__ float mls[4][2];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e8 = lane & 7, j8 = lane >> 3;
    // heads that share a key head on one XCD (workgroups are dealt out to 8 in turn)
    const uint32_t block = blockIdx.y * gridDim.x + blockIdx.x, item = block / (8 * a.group) * 8 + block % 8;
    const uint32_t t = item / a.kv_heads, kh = item % a.kv_heads, h = kh * a.group + block / 8 % a.group;
    if (t >= a.tokens) return;
    const uint32_t b = row_of_token(a.starts, a.batch, a.tokens, t);
    const Row r = load_row(a.starts, a.seqs, a.tables, a.lengths, a.tokens, a.seq_count, a.table_width, a.page_shift, PAGED, b);
    if (t < r.first || t - r.first >= r.n) return;  // a row of no sequence
    const uint32_t hd = a.head_dim;
    const TQ* q = static_cast<const TQ*>(a.q) + (size_t)t * a.q_stride + (size_t)h * hd;
    float qs[CHUNKS][N], o[CHUNKS][N];
    auto offset = [&](int c) { return (8 * c + e8) * N < hd ? (8 * c + e8) * N : 0; };  // of the lane's columns, 0 behind the last
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const uint32_t col = (8 * c + e8) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            qs[c][i] = col < hd ? to_float(q[col + i]) : 0.0f;
            o[c][i] = 0.0f;
        }
    }

    const int64_t pos = r.pos0 + (int64_t)(t - r.first);
    const int64_t hi64 = pos + (int64_t)a.right + 1;
    const int32_t hi = (int32_t)(hi64 < 0 ? 0 : hi64 < r.length ? hi64 : r.length);
    const int64_t lo64 = pos - (int64_t)a.left;
    const int32_t lo = (int32_t)(lo64 < 0 ? 0 : lo64 < hi ? lo64 : hi);
    const int32_t sinks = a.sinks < (uint32_t)lo ? (int32_t)a.sinks : lo;
    // element offset of key j's row of this head, or -1 where its page does not exist
    auto row_at = [&](int32_t j) -> int64_t {
        if constexpr (PAGED) {
            const int32_t page = r.table[j >> a.page_shift];
            if (page < 0 || (uint32_t)page >= a.pages) return -1;
            return ((((int64_t)page * a.kv_heads + kh) << a.page_shift) + (j & ((1 << a.page_shift) - 1))) * hd;
        } else {
            return (int64_t)(r.first + j) * a.kv_stride + (int64_t)kh * hd;
        }
    };
    const TK* k = static_cast<const TK*>(a.k);
    const TK* v = static_cast<const TK*>(a.v);
    const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f, scale = (a.scale == 0.0f ? 1.0f : fabsf(a.scale)) * LOG2E;
    float m = -__builtin_inff(), l = 0.0f;
    auto keys = [&](int32_t from, int32_t to) {
        for (int32_t j0 = from + 64 * (int32_t)wave; j0 < to; j0 += 256) {
            const int32_t j = j0 + (int32_t)(8 * e8 + j8);  // the lane's own key, whose place, score and p it holds
            int64_t at = j < to ? row_at(j) : -1;
            auto row = [&](int g) { return (int64_t)__shfl((int)(at >> 32), (int)(8 * j8) + g) << 32 | (uint32_t)__shfl((int)at, (int)(8 * j8) + g); };
            // chunks c0 .. c0 + BATCH - 1 of rows g0 .. g0 + AHEAD - 1, all asked for before the first is needed
            Bits x[AHEAD][BATCH];
            bool there[AHEAD];
            auto fetch = [&](const TK* src, int g0, int c0) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int64_t from = row(g0 + u);
                    there[u] = from >= 0;
                    const TK* const start = src + (from < 0 ? 0 : from);
#pragma unroll
                    for (int c = 0; c < BATCH; ++c) x[u][c] = *reinterpret_cast<const Bits*>(start + offset(c0 + c));
                }
                __builtin_amdgcn_sched_barrier(0);
            };
            float s = -__builtin_inff();
#pragma unroll 1
            for (int g0 = 0; g0 < 8; g0 += AHEAD) {
                float dot[AHEAD] = {};
#pragma unroll
                for (int c0 = 0; c0 < CHUNKS; c0 += BATCH) {
                    fetch(k, g0, c0);
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                        for (int c = 0; c < BATCH; ++c) {
                            // (an infinite element must not meet the 0 behind q's last)
                            const Pack y = __builtin_bit_cast(Pack, (Bits)(x[u][c] & ((8 * (c0 + c) + e8) * N < hd ? ~0u : 0u)));
#pragma unroll
                            for (int i = 0; i < N; ++i) dot[u] = fmaf(qs[c0 + c][i], to_float(y.x[i]), dot[u]);
                        }
                }
#pragma unroll
                for (int w = 1; w < 8; w <<= 1)
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u) dot[u] += __shfl_xor(dot[u], w);
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
                    if (e8 == (uint32_t)(g0 + u) && at >= 0) s = dot[u] * sign;
            }
            const float mx = fmaxf(m, wave_max(s));
            const float base = mx == -__builtin_inff() ? 0.0f : mx;  // (nothing yet but scores of -infinity)
            const float p = exp2f((s - base) * scale), alpha = exp2f((m - base) * scale);
            m = mx;
            l = l * alpha + wave_sum(p);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int i = 0; i < N; ++i) o[c][i] *= alpha;
#pragma unroll 1
            for (int g0 = 0; g0 < 8; g0 += AHEAD) {
                float pj[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) pj[u] = __shfl(p, (int)(8 * j8) + g0 + u);
#pragma unroll
                for (int c0 = 0; c0 < CHUNKS; c0 += BATCH) {
                    fetch(v, g0, c0);
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                        for (int c = 0; c < BATCH; ++c) {
                            const Pack y = __builtin_bit_cast(Pack, (Bits)(x[u][c] & (there[u] ? ~0u : 0u)));
#pragma unroll
                            for (int i = 0; i < N; ++i) o[c0 + c][i] = fmaf(pj[u], to_float(y.x[i]), o[c0 + c][i]);
                        }
                }
            }
        }
    };
    keys(0, sinks);
    keys(lo, hi);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int w = 8; w < 64; w <<= 1) o[c][i] += __shfl_xor(o[c][i], w);
            if (j8 == 0) sums[wave][(8 * c + e8) * N + i] = o[c][i];
        }
    if (lane == 0) {
        mls[wave][0] = m;
        mls[wave][1] = l;
    }
    __syncthreads();
    const float top = fmaxf(fmaxf(mls[0][0], mls[1][0]), fmaxf(mls[2][0], mls[3][0])), base = top == -__builtin_inff() ? 0.0f : top;
    float f[4];
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = exp2f((mls[w][0] - base) * scale);
        l += mls[w][1] * f[w];
    }
    if (threadIdx.x < hd) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum += sums[w][threadIdx.x] * f[w];
        static_cast<TQ*>(a.out)[(size_t)t * a.out_stride + (size_t)h * hd + threadIdx.x] = (TQ)(l == 0.0f ? 0.0f : sum * (1.0f / l));
    }
}

template <typename TQ, typename TK, bool PAGED, int N>
int launch_plain_of(Ctx* ctx, const AttnArgs& a)
{
    const uint64_t items = ((uint64_t)a.tokens * a.kv_heads + 7) / 8 * 8 * a.group;
    if (items > 1u << 30) return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "attention: too many rows for one launch");
    const dim3 grid = grid_of(items);
    if (a.head_dim <= 64) hipLaunchKernelGGL((attention_plain_kernel<TQ, TK, PAGED, N, 64>), grid, dim3(256), 0, ctx->stream, a);
    else if (a.head_dim <= 128) hipLaunchKernelGGL((attention_plain_kernel<TQ, TK, PAGED, N, 128>), grid, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((attention_plain_kernel<TQ, TK, PAGED, N, 256>), grid, dim3(256), 0, ctx->stream, a);
    return hip_check(ctx, hipGetLastError(), "attention_plain_kernel launch");
}

template <typename TQ, typename TK>
int launch_plain(Ctx* ctx, const AttnArgs& a)
{
    constexpr int N = 16 / sizeof(TK);
    const bool packs = a.head_dim % N == 0 && ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15) == 0 && (a.paged || a.kv_stride % N == 0);
    if (a.paged) return packs ? launch_plain_of<TQ, TK, true, N>(ctx, a) : launch_plain_of<TQ, TK, true, 1>(ctx, a);
    return packs ? launch_plain_of<TQ, TK, false, N>(ctx, a) : launch_plain_of<TQ, TK, false, 1>(ctx, a);
}

// ---------------------------------------------------------------------------------------------
// Joins what the splits of a row have: out = sum_s o_s 2^(c (m_s - m)) / sum_s l_s 2^(c (m_s - m)).  A workgroup takes `rows` rows of up to 16 of a
// sequence and key head (blocks of 16 are numbered as first_slot does, or, by_row, the first of each row of the batch: where only those of few rows are
// split, the others would be 20 us of workgroups with nothing to do in a batch of 2300 tokens, 32 heads); of a row's threads head_dim / 4 take four columns each, and `groups` sets of
// them every groups-th split.
// ---------------------------------------------------------------------------------------------
constexpr uint32_t JOIN_ROWS = 16;

template <typename TQ>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnArgs a, attn::Partial part, uint32_t by_row, uint32_t parts, uint32_t rows, uint32_t groups,
                                                             uint32_t wide_splits, uint32_t narrow_splits, uint32_t narrow_rows)
{
    __shared__ float sums[256][4];
    __shared__ float mls[256][2];
    const uint32_t tid = threadIdx.x, lanes = a.head_dim / 4;
    const uint32_t kh = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads, slot = rest / parts;
    const uint32_t b = by_row ? slot : attn::row_of_slot(a, slot, JOIN_ROWS);
    const uint32_t first = clamped_start(a.starts, b, a.tokens), end = clamped_start(a.starts, b + 1, a.tokens), before = by_row ? slot : attn::first_slot(a, b, first, JOIN_ROWS);
    if (slot < before || end <= first) return;
    const uint32_t count = (end - first) * a.group, row0 = (slot - before) * JOIN_ROWS, stop = row0 + JOIN_ROWS < count ? row0 + JOIN_ROWS : count;
    const uint32_t splits = count <= narrow_rows ? narrow_splits : wide_splits;
    if (row0 >= count || splits == 1) return;
    const uint32_t set = tid / lanes, mine = set / groups, g = set % groups, col = tid % lanes * 4;
    for (uint32_t from = row0 + rest % parts * rows; from < stop; from += parts * rows) {
        const uint32_t row = from + mine;
        const bool works = mine < rows && row < stop;
        const uint32_t t = first + row / a.group, head = kh * a.group + row % a.group;
        const uint64_t at = (uint64_t)t * a.heads + head;
        float top = -__builtin_inff(), l = 0.0f;
        const float c = works ? part.c[at] : 1.0f;
        attn::f32x4 y = {0.f, 0.f, 0.f, 0.f};
        auto take = [&](auto count) __attribute__((always_inline)) {
            constexpr uint32_t AHEAD = decltype(count)::value;  // splits whose results are asked for together
            for (uint32_t s0 = g; s0 < splits; s0 += AHEAD * groups) {
                float m[AHEAD], lm[AHEAD];
                attn::f32x4 x[AHEAD];
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    const uint32_t s = s0 + i * groups < splits ? s0 + i * groups : splits - 1;
                    const uint64_t where = s * part.rows + at;
                    m[i] = part.ml[2 * where];
                    lm[i] = s0 + i * groups < splits ? part.ml[2 * where + 1] : 0.0f;
                    x[i] = *reinterpret_cast<const attn::f32x4*>(part.o + where * a.head_dim + col);  // (anything where l is 0)
                }
                float up = top;
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) up = fmaxf(up, m[i]);
                const float base = up == -__builtin_inff() ? 0.0f : up, alpha = __builtin_amdgcn_exp2f((top - base) * c);
                top = up;
                l *= alpha;
                y *= alpha;
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    const float f = __builtin_amdgcn_exp2f((m[i] - base) * c);
                    l += lm[i] == 0.0f ? 0.0f : lm[i] * f;  // (NaN is not)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] += lm[i] == 0.0f ? 0.0f : x[i][e] * f;
                }
            }
        };
        if (works) {
            if (splits <= 2 * groups) take(std::integral_constant<uint32_t, 2>{});
            else if (splits <= 4 * groups) take(std::integral_constant<uint32_t, 4>{});
            else take(std::integral_constant<uint32_t, 8>{});
        }
        *reinterpret_cast<attn::f32x4*>(sums[tid]) = y;
        mls[tid][0] = top;
        mls[tid][1] = l;
        __syncthreads();
        if (works && g == 0) {
            for (uint32_t i = 1; i < groups; ++i) top = fmaxf(top, mls[tid + i * lanes][0]);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            l = 0.0f;
            y = (attn::f32x4){0.f, 0.f, 0.f, 0.f};
            for (uint32_t i = 0; i < groups; ++i) {
                const float lm = mls[tid + i * lanes][1];
                if (lm == 0.0f) continue;
                const float f = __builtin_amdgcn_exp2f((mls[tid + i * lanes][0] - base) * c);
                l += lm * f;
                y += *reinterpret_cast<const attn::f32x4*>(sums[tid + i * lanes]) * f;
            }
            attn::store4(static_cast<TQ*>(a.out) + (size_t)t * a.out_stride + (size_t)head * a.head_dim + col, l == 0.0f ? (attn::f32x4){0.f, 0.f, 0.f, 0.f} : y * (1.0f / l));
        }
        __syncthreads();
    }
}

// Whether only rows of the batch with up to NARROW_ROWS rows are split.
bool joins_by_row(const attn::Plan& p) { return p.wide && p.wide_splits == 1; }

template <typename TQ>
int launch_join(Ctx* ctx, const AttnArgs& a, const attn::Plan& p)
{
    const uint32_t lanes = a.head_dim / 4, splits = std::max(p.wide_splits, p.narrow_splits);
    uint32_t groups = 1;
    while (groups < 16 && groups * 4 < splits && 2 * groups * lanes <= 256) groups *= 2;
    const uint32_t rows = std::min(JOIN_ROWS, 256 / (lanes * groups));
    const bool by_row = joins_by_row(p);
    ctx->attn_plan.join = by_row ? 2 : 1;
    static_assert(attn::NARROW_ROWS <= JOIN_ROWS, "a block holds all rows of a sequence of few");
    const uint64_t slots = (by_row ? 0 : (uint64_t)a.tokens * a.group / JOIN_ROWS) + a.batch;
    // workgroups that share a block, where there are few blocks
    const uint32_t parts = slots * a.kv_heads >= 4 * (uint64_t)ctx->prop.multiProcessorCount ? 1 : (JOIN_ROWS + rows - 1) / rows;
    const uint64_t grid = slots * parts * a.kv_heads;
    hipLaunchKernelGGL((attention_join_kernel<TQ>), dim3((uint32_t)grid), dim3(256), 0, ctx->stream, a, p.part, (uint32_t)by_row, parts, rows, groups, p.wide ? p.wide_splits : 1,
                       p.narrow ? p.narrow_splits : 1, p.narrow ? p.narrow_rows : 0);
    return hip_check(ctx, hipGetLastError(), "attention_join_kernel launch");
}

// Whether the matrix-core kernels take the call: head sizes that they are built for, rows of whole 16 bytes.
bool matrix_form(const AttnArgs& a)
{
    if (a.head_dim != 32 && a.head_dim != 64 && a.head_dim != 80 && a.head_dim != 96 && a.head_dim != 128) return false;
    const uint64_t qe = a.dtype == PIMDL_F32 ? 4 : 2, ke = a.cache_dtype == PIMDL_F32 ? 4 : 2;
    uint64_t all = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
    all |= a.q_stride * qe | a.out_stride * qe | (a.paged ? 0 : a.kv_stride * ke);
    // (offsets within a page, or within a tile of rows, are 32-bit numbers)
    if (a.paged && ((uint64_t)a.kv_heads << a.page_shift) * a.head_dim * ke >= 1ull << 32) return false;
    return all % 16 == 0 && (uint64_t)a.tokens * a.group < 1u << 30 && a.kv_stride < 1u << 22;
}

// Which kernels run, and over how many workgroups the keys of a row are split.
int make_plan(Ctx* ctx, const AttnArgs& a, attn::Plan* p)
{
    *p = {};
    const uint64_t rows = (uint64_t)a.tokens * a.group, cus = (uint64_t)ctx->prop.multiProcessorCount;
    // keys that a row may see at most
    uint64_t keys = a.paged ? (uint64_t)a.table_width << a.page_shift : a.tokens;
    keys = std::min<uint64_t>(keys, (uint64_t)a.left + a.right + 1 + a.sinks + attn::WIDE_ROWS);
    const uint64_t wide_items = (rows + attn::WIDE_ROWS - 1) / attn::WIDE_ROWS * a.kv_heads;
    // So few blocks of 128 rows that most of the device would idle take blocks of 16, unless there are so many keys that every one of those fills
    // its CU anyway: 2^15 scores a CU.  us in blocks of 16 / 128: windows over 128 to 512 tokens, 12 heads, fp32 (12 / 24 / 36 / 48 blocks of 128)
    // 6.6 / 12.2, 7.6 / 18.3, 15.9 / 25.1, 19.2 / 31.8, over 1024 (96) 44.4 / 38.4; 32 heads over 8, bf16, 256 and 512 tokens (64, 128) 12.4 / 13.4,
    // 26.9 / 21.1.  New tokens of a paged cache, 32 heads over 8, at 2^13 scores a CU: 15.6 / 30.0 (16 over 4000 keys); 2^14: 17.9 / 31.5 (32),
    // 14.3 / 29.1 (8 x 16 over 1000); 2^15: 22.8 / 34.1 (64), 34.6 / 40.3 (8 x 8); 2^16: 51.4 / 36.6 (128), 58.5 / 46.3 (8 x 16), 34.8 / 48.5 (32 over
    // 16000); 2^17: 56.5 / 54.0 (64 over 16000), 95.5 / 56.0 (8 x 32).  Keys are counted by what a row of the table can hold, not by what it does: the
    // lengths are on the device.
    const bool few = 16 * wide_items <= 3 * cus && (uint64_t)a.tokens * a.heads * keys <= cus << 15;
    p->narrow = a.paged || few;
    p->wide = !few && !(a.paged && a.tokens <= a.batch);
    p->by_slot = few && a.tokens > a.batch;
    p->narrow_rows = p->wide ? attn::NARROW_ROWS : 0xffffffffu;
    p->wide_splits = p->narrow_splits = 1;
    p->slots = (uint32_t)(rows / attn::WIDE_ROWS) + a.batch;
    if (p->narrow) {
        const uint64_t items = (p->by_slot ? (rows + attn::NARROW_ROWS - 1) / attn::NARROW_ROWS : a.batch) * a.kv_heads;
        // Up to 1024 keys: no split, whose join costs more than it saves (32 heads over 8, bf16, one sequence of 777: 8.8 us, in three 11.3; of 1500
        // 12.3 and 11.3, of 2000 14.7 and 11.2).  Fewer items than half the CUs: every CU one workgroup, of at least 256 keys.  More: shares of at least 1024 keys, so that long sequences are dealt
        // out too.  us with shares of 512 / 1024 / 2048 keys for more items: 64 sequences of up to 8191 231 / 203 / 203, 32 of up to 4000, 12 heads,
        // fp32 116 / 96 / 118; for fewer: two of 100 000 67 / 55 / 50 (one workgroup per CU), 32 of up to 16000 with one key head 52 / 44 / 41.
        p->narrow_splits = (uint32_t)std::max<uint64_t>(1, keys <= 1024 ? 1 : 2 * items <= cus ? std::min<uint64_t>({(cus + items - 1) / items, keys / 256, 256})
                                                                        : std::min<uint64_t>((8 * cus + items - 1) / items, keys / 1024));
    }
    // About two workgroups a CU, rounded up: registers leave room for two, or for one in fp32 above 80 dims and fp32 over 16 bits above 96, which the rule
    // does not look at.  us at 1 / 2 / 3 / 4: 10 chunks of 200 to 400 tokens over up to 4000 keys, 16 heads over 8, bf16, 189 / 180 / 165 / 165, of 300 to
    // 600 235 / 235 / 231 / 231; one of 256 over 16000, 32 heads over 8, 171 / 137 / 158 / 143; two of 500 to 700 over 5000, 12 heads, fp32 over fp16,
    // 70 / 70 / 66 / 70; 64 sequences with 1 to 40 new tokens over up to 5000 179 / 191 / 214 / 221; 16 with chunks of up to 512 or a token over up to 6000
    // 214 / 224 / 225 / 236; three of 300 to 512 over up to 3000, 16 heads of 80, fp32, 144 / 118 / 125 / 124.
    if (p->wide) p->wide_splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({(2 * cus + wide_items - 1) / wide_items, keys / 512, 16}));
    // what the splits hand over is kept below 128 MiB
    const uint64_t row_bytes = (uint64_t)(a.head_dim + 2) * 4 * a.tokens * a.heads, most = std::max<uint64_t>(1, (128ull << 20) / row_bytes);
    p->narrow_splits = (uint32_t)std::min<uint64_t>(p->narrow_splits, most);
    p->wide_splits = (uint32_t)std::min<uint64_t>(p->wide_splits, most);
    const uint32_t splits = std::max(p->narrow_splits, p->wide_splits);
    const uint64_t batch_rows = (uint64_t)a.batch * a.kv_heads, blocks16 = rows / attn::NARROW_ROWS * a.kv_heads + batch_rows;
    const bool fits = p->wide ? fits_launch((uint64_t)p->slots * a.kv_heads * p->wide_splits + (p->narrow ? batch_rows * p->narrow_splits : 0), 256)
                              : fits_launch((p->by_slot ? blocks16 : batch_rows) * p->narrow_splits, 512);
    const bool join_fits = splits == 1 || fits_launch(joins_by_row(*p) ? batch_rows : blocks16, 256);
    if ((uint64_t)a.tokens * a.heads > 1u << 30 || !fits || !join_fits)
        return set_error(ctx, PIMDL_ERR_UNSUPPORTED, "attention: too many rows for one launch");
    if (splits > 1) {
        int rc = ensure_scratch(ctx, &ctx->d_attn, &ctx->attn_bytes, row_bytes * splits + (uint64_t)a.tokens * a.heads * 4, "attention's partial results");
        if (rc) return rc;
        p->part.rows = (uint64_t)a.tokens * a.heads;
        p->part.o = reinterpret_cast<float*>(ctx->d_attn);
        p->part.ml = p->part.o + p->part.rows * splits * a.head_dim;
        p->part.c = p->part.ml + p->part.rows * splits * 2;
    }
    return PIMDL_OK;
}

}  // namespace

int launch_attention(Ctx* ctx, const AttnArgs& a)
{
    ctx->attn_plan = {};
    if (a.tokens == 0 || a.batch == 0) return PIMDL_OK;
    if (!matrix_form(a)) {
        ctx->attn_plan.plain = 1;
        if (a.dtype == PIMDL_BF16) return launch_plain<__bf16, __bf16>(ctx, a);
        if (a.dtype == PIMDL_F16) return launch_plain<_Float16, _Float16>(ctx, a);
        if (a.cache_dtype == PIMDL_BF16) return launch_plain<float, __bf16>(ctx, a);
        if (a.cache_dtype == PIMDL_F16) return launch_plain<float, _Float16>(ctx, a);
        return launch_plain<float, float>(ctx, a);
    }
    attn::Plan p;
    int rc = make_plan(ctx, a, &p);
    if (rc) return rc;
    ctx->attn_plan = {0, p.wide, p.narrow, p.wide ? p.wide_splits : 0, p.narrow ? p.narrow_splits : 0, p.by_slot, 0};
    if (a.dtype == PIMDL_BF16) rc = attn::launch_bf16(ctx, a, p);
    else if (a.dtype == PIMDL_F16) rc = attn::launch_f16(ctx, a, p);
    else if (a.cache_dtype == PIMDL_BF16) rc = attn::launch_f32_bf16(ctx, a, p);
    else if (a.cache_dtype == PIMDL_F16) rc = attn::launch_f32_f16(ctx, a, p);
    else rc = attn::launch_f32(ctx, a, p);
    if (rc || (p.wide_splits == 1 && p.narrow_splits == 1)) return rc;
    if (a.dtype == PIMDL_BF16) return launch_join<__bf16>(ctx, a, p);
    if (a.dtype == PIMDL_F16) return launch_join<_Float16>(ctx, a, p);
    return launch_join<float>(ctx, a, p);
}

}  // namespace pimdl
