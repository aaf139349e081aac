// Queries and keys turned by their positions, in place or on the way into the paged cache (pimdl_rotate, pimdl_cache_append_rotary), for gfx950 (MI355X).
//
// At position p the pair (a, b) of frequency f becomes (a cos pf - b sin pf, a sin pf + b cos pf): a token's angles are the same for all of its heads, so a
// workgroup works out those of its tokens once, in LDS, while the heads' columns are on their way.
//
// HBM bounds it: 6 prompts of up to 4096 tokens, 32 heads over 8 of 128 dims, bf16, 343 MB, 68 to 70 us (5.0 TB/s; a copy of 4 GiB reaches 4.8); 12 on their way into the cache, values
// too, 696 MB, 129 to 135.  A few tokens wait for memory three times over (starts; lengths and pages; frequencies), 5.2 and 6.4 us, and for the host, 9 us a call.
#include <algorithm>
#include <type_traits>

#include "serve_common.h"

namespace pimdl {

namespace {

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T x[N];
};

// Sine and cosine of a finite angle.  The angle less the nearest multiple k of a quarter turn, pi / 2 being taken as the sum of two doubles (Cody and Waite), is
// within pi / 4 and exact to 2^-53 of the angle; there Taylor's series to the 9th and 10th power is within 2e-9.
__device__ __forceinline__ void sine_cosine(double angle, float* s, float* c)
{
    const double k = __builtin_rint(angle * 0.63661977236758134308);
    double rest = fma(-k, 1.57079632679489655800, angle);
    rest = fma(-k, 6.12323399573676603587e-17, rest);
    const int quarter = (int)(k - 4.0 * __builtin_floor(k * 0.25));
    const float r = (float)rest, r2 = r * r;
    const float sine = fmaf(r * r2, fmaf(r2, fmaf(r2, fmaf(r2, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), r);
    const float cosine = fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const float x = quarter & 1 ? cosine : sine, y = quarter & 1 ? sine : cosine;
    *s = quarter & 2 ? -x : x;
    *c = (quarter + 1) & 2 ? -y : y;
}

// x / d for x and d of the sizes that launch_rotary says: m = ceil(2^32 / d)
struct Divide {
    uint32_t d, m;
    __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return d == 1 ? x : __umulhi(x, m); }
};
Divide divide_by(uint32_t d) { return {d, (uint32_t)(((1ull << 32) + d - 1) / d)}; }

constexpr uint32_t STARTS = 1024;   // of the batch, at most, in LDS
constexpr uint32_t MOST_TOKENS = 64, MOST_ANGLES = 2048, AHEAD = 4;

// Shared memory of a workgroup with `group` tokens: their cosines and sines [group][dims], starts or every step-th of them, and a token's place
struct Places {
    int64_t position[MOST_TOKENS];
    int64_t slot[MOST_TOKENS];   // row of the cache (page, then row of the page) or -1
    uint32_t of_batch[MOST_TOKENS];
};

// A unit is 2 N columns of one head of one token: N pairs, or 2 N columns that are carried over as they are.  A token's units: those of its query
// heads, its key heads and (paged) its value heads.
template <typename TI, typename TC, bool PAGED, bool HALVES, int N>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, uint32_t group, Divide units, Divide per_head)
{
    extern __shared__ __attribute__((aligned(16))) float turns[];
    __shared__ int32_t some_starts[STARTS];
    __shared__ Places places;
    const uint32_t tid = threadIdx.x, half = a.dims / 2, hd = a.head_dim;
    const uint64_t block = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x;
    const uint64_t first64 = block * group;
    if (first64 >= a.tokens) return;
    const uint32_t first = (uint32_t)first64, count = a.tokens - first < group ? a.tokens - first : group, items = count * units.d;
    const bool writes = !PAGED || !a.cache.lacking || *a.cache.lacking == 0;

    struct Unit {
        uint32_t token, head, col0, col1;  // head: of queries, then keys, then values; columns of the two packs
        bool turned;
    };
    auto unit_of = [&](uint32_t item) {
        Unit u;
        u.token = group == 1 ? 0 : units(item);
        const uint32_t rest = item - u.token * units.d;
        u.head = per_head(rest);
        const uint32_t i = rest - u.head * per_head.d;
        u.turned = i < half / N && u.head < a.heads + a.kv_heads;
        if (HALVES && u.turned) u.col0 = i * N, u.col1 = i * N + half;
        else if (HALVES && u.head < a.heads + a.kv_heads) u.col0 = a.dims + (i - half / N) * 2 * N, u.col1 = u.col0 + N;
        else u.col0 = i * 2 * N, u.col1 = u.col0 + N;
        return u;
    };
    Pack<TI, N> x[AHEAD][2];
    auto fetch = [&](uint32_t from) {
#pragma unroll
        for (uint32_t n = 0; n < AHEAD; ++n) {
            const uint32_t item = from + n * 256 + tid;
            if (item >= items) continue;
            const Unit u = unit_of(item);
            const size_t t = first + u.token;
            const TI* row = u.head < a.heads                ? static_cast<const TI*>(a.q) + t * a.q_stride + (size_t)u.head * hd
                            : u.head < a.heads + a.kv_heads ? static_cast<const TI*>(a.k) + t * a.k_stride + (size_t)(u.head - a.heads) * hd
                                                            : static_cast<const TI*>(a.v) + t * a.k_stride + (size_t)(u.head - a.heads - a.kv_heads) * hd;
            x[n][0] = *reinterpret_cast<const Pack<TI, N>*>(row + u.col0);
            if (u.col1 < hd) x[n][1] = *reinterpret_cast<const Pack<TI, N>*>(row + u.col1);  // (one column may be left over)
        }
    };
    fetch(0);

    // each token's row of the batch: among every step-th start in LDS, then among those between
    const uint32_t step = a.batch / STARTS + 1;
    for (uint32_t i = tid; i * step <= a.batch; i += 256) some_starts[i] = a.starts[i * step];
    __syncthreads();
    if (tid < count) {
        const uint32_t t = first + tid;
        auto clamped = [&](int32_t s) { return s < 0 ? 0u : (uint32_t)s < a.tokens ? (uint32_t)s : a.tokens; };
        uint32_t lo = 0, up = a.batch / step + 1;  // some_starts[lo] is not behind t (or lo == 0)
        while (up - lo > 1) {
            const uint32_t mid = (lo + up) / 2;
            if (clamped(some_starts[mid]) <= t) lo = mid;
            else up = mid;
        }
        lo *= step;
        up = lo + step < a.batch ? lo + step : a.batch;
        lo = lo < a.batch ? lo : a.batch - 1;
        while (up > lo + 1) {
            const uint32_t mid = (lo + up) / 2;
            if (clamped_start(a.starts, mid, a.tokens) <= t) lo = mid;
            else up = mid;
        }
        const Row r = load_row(a.starts, a.seqs, a.cache.tables, a.cache.lengths, a.tokens, a.cache.seqs, a.cache.table_width, a.page_shift, PAGED, lo);
        const bool mine = t >= r.first && t - r.first < r.n;
        int64_t slot = -1;
        if (PAGED && mine && writes) {
            const int32_t pos = r.pos0 + (int32_t)(t - r.first);
            if (pos >= 0) {
                const int32_t page = r.table[pos >> a.page_shift];
                if (page >= 0 && (uint32_t)page < a.cache.pages) slot = (int64_t)page << a.page_shift | (pos & ((1 << a.page_shift) - 1));
            }
        }
        places.position[tid] = (int64_t)r.pos0 + (mine && a.depths ? (int64_t)a.depths[t] : (int64_t)t - r.first);
        places.slot[tid] = slot;
        places.of_batch[tid] = mine;
    }
    __syncthreads();
    for (uint32_t i = tid; i < count * half; i += 256) {
        const uint32_t token = i / half, pair = i % half;
        float s, c;
        sine_cosine((double)places.position[token] * a.freqs[pair], &s, &c);
        turns[token * a.dims + pair] = c;
        turns[token * a.dims + half + pair] = s;
    }
    __syncthreads();

    for (uint32_t from = 0; from < items; from += AHEAD * 256) {
        if (from) fetch(from);
#pragma unroll
        for (uint32_t n = 0; n < AHEAD; ++n) {
            const uint32_t item = from + n * 256 + tid;
            if (item >= items) continue;
            const Unit u = unit_of(item);
            if (!places.of_batch[u.token]) continue;  // a row of no sequence
            const size_t t = first + u.token;
            float y[2][N];
#pragma unroll
            for (int i = 0; i < N; ++i) y[0][i] = to_float(x[n][0].x[i]), y[1][i] = to_float(x[n][1].x[i]);
            if (u.turned) {
                const float *cs, *sn;
                if constexpr (HALVES) cs = turns + u.token * a.dims + u.col0, sn = cs + half;
                else cs = turns + u.token * a.dims + u.col0 / 2, sn = cs + half;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    float &p = HALVES ? y[0][i] : y[2 * i / N][2 * i % N], &q = HALVES ? y[1][i] : y[(2 * i + 1) / N][(2 * i + 1) % N];
                    const float c = cs[i], s = sn[i], old = p;
                    p = fmaf(old, c, -(q * s));
                    q = fmaf(old, s, q * c);
                }
            }
            auto store = [&](auto* row) {
                typedef typename std::remove_reference<decltype(*row)>::type TO;
                Pack<TO, N> o[2];
#pragma unroll
                for (int i = 0; i < N; ++i) o[0].x[i] = (TO)y[0][i], o[1].x[i] = (TO)y[1][i];
                *reinterpret_cast<Pack<TO, N>*>(row + u.col0) = o[0];
                if (u.col1 < hd) *reinterpret_cast<Pack<TO, N>*>(row + u.col1) = o[1];
            };
            if (u.head < a.heads) {
                store(static_cast<TI*>(a.q_out) + t * a.q_out_stride + (size_t)u.head * hd);
            } else if constexpr (PAGED) {
                const int64_t slot = places.slot[u.token];
                const bool value = u.head >= a.heads + a.kv_heads;
                const uint32_t h = u.head - a.heads - (value ? a.kv_heads : 0);
                const uint64_t in_page = (uint64_t)slot & ((1u << a.page_shift) - 1), page = (uint64_t)slot >> a.page_shift;
                if (slot >= 0) store(static_cast<TC*>(value ? a.cache.v : a.cache.k) + ((((page * a.kv_heads + h) << a.page_shift) + in_page) * hd));
            } else {
                store(static_cast<TI*>(a.k_out) + t * a.k_out_stride + (size_t)(u.head - a.heads) * hd);
            }
        }
    }
}

template <typename TI, typename TC, bool PAGED, bool HALVES, int N>
int launch_of(Ctx* ctx, const RotaryArgs& a)
{
    // A head's units; where N is 1 an odd head's last column is half a one.  Divisions: by it of up to 2^25 units of a token (an error below d in m is below 1 in the quotient up to
    // 2^32 / d), by a token's units of up to AHEAD * 256 of several.
    const uint32_t per_head = (a.head_dim + 2 * N - 1) / (2 * N);
    const uint64_t units = (uint64_t)(a.heads + (PAGED ? 2 : 1) * a.kv_heads) * per_head;
    const uint32_t group = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({AHEAD * 256 / units, MOST_TOKENS, MOST_ANGLES / (a.dims / 2)}));
    const uint64_t blocks = ((uint64_t)a.tokens + group - 1) / group;
    const size_t lds = (size_t)group * a.dims * 4;
    hipLaunchKernelGGL((rotary_kernel<TI, TC, PAGED, HALVES, N>), grid_of(blocks), dim3(256), lds, ctx->stream, a, group, divide_by((uint32_t)units), divide_by(per_head));
    return hip_check(ctx, hipGetLastError(), "rotary_kernel launch");
}

// Columns to a pack: 16 bytes, 8, or one, by what a head's columns and the rows' addresses are multiples of.
template <typename TI, typename TC, bool PAGED>
int launch_types(Ctx* ctx, const RotaryArgs& a)
{
    uint64_t all = 0;
    if (a.heads) all |= reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) | (a.q_stride | a.q_out_stride) * (uint64_t)sizeof(TI);
    if (a.kv_heads) all |= reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | a.k_stride * (uint64_t)sizeof(TI);
    if (!PAGED && a.kv_heads) all |= reinterpret_cast<uintptr_t>(a.k_out) | a.k_out_stride * (uint64_t)sizeof(TI);
    auto packs = [&](uint32_t n) { return a.dims % (2 * n) == 0 && a.head_dim % (2 * n) == 0 && all % (n * sizeof(TI)) == 0; };
    const bool halves = a.pairs == PIMDL_PAIRS_HALVES;
    if constexpr (sizeof(TI) == 2)
        if (packs(8)) return halves ? launch_of<TI, TC, PAGED, true, 8>(ctx, a) : launch_of<TI, TC, PAGED, false, 8>(ctx, a);
    if (packs(4)) return halves ? launch_of<TI, TC, PAGED, true, 4>(ctx, a) : launch_of<TI, TC, PAGED, false, 4>(ctx, a);
    return halves ? launch_of<TI, TC, PAGED, true, 1>(ctx, a) : launch_of<TI, TC, PAGED, false, 1>(ctx, a);
}

}  // namespace

int launch_rotary(Ctx* ctx, const RotaryArgs& a, bool paged)
{
    if (!paged) {
        if (a.dtype == PIMDL_BF16) return launch_types<__bf16, __bf16, false>(ctx, a);
        if (a.dtype == PIMDL_F16) return launch_types<_Float16, _Float16, false>(ctx, a);
        return launch_types<float, float, false>(ctx, a);
    }
    if (a.dtype == PIMDL_BF16) return launch_types<__bf16, __bf16, true>(ctx, a);
    if (a.dtype == PIMDL_F16) return launch_types<_Float16, _Float16, true>(ctx, a);
    if (a.cache.dtype == PIMDL_BF16) return launch_types<float, __bf16, true>(ctx, a);
    if (a.cache.dtype == PIMDL_F16) return launch_types<float, _Float16, true>(ctx, a);
    return launch_types<float, float, true>(ctx, a);
}

}  // namespace pimdl
