// Attention of drafted trees of many rows, dealt out evenly (gfx950); part of attn_body.h.
//
// A batch of drafts has few rows over contexts of any length: a key head's keys are read for 64 to 500 rows at a time, and a workgroup per block of rows, or per
// equal split of it, leaves most of the device waiting for the longest sequence.  So a workgroup takes up to 256 rows (eight waves of 32), which reads most drafts' keys
// once, a CU has one, and all blocks' tiles of keys are one row of units of time -- sequences in turn, their key heads, the heads' blocks, a block's tiles, each as many units as its
// block's rows take -- that is cut into equal shares, a workgroup each.  Lengths are in device memory, so each workgroup works out the deal by itself, from every
// sequence's number of units and a sum over them.  A block that one share holds whole is written at once; of others every share leaves its sums, which
// attention_deal_join_kernel joins.
//
// 32 sequences of 16 to 64 nodes over up to 8191 keys, 32 heads over 8 of 128 dims, bf16: 210 us once the clock has settled, after some hundred launches on end, 259 in the median of the first 40;
// 574 MB alone would be 121 us, the matrix instructions, a third of them for the second piece of p, 142.  These are at work in 39 % of the SIMDs' cycles, others in 44 %, and mostly not at once: a product leaves the vector unit
// to others for a part of its time only, 57 cycles for a product of 32 and its share of 9 others.  Shares end within 5 % of each other; a block's own 10 us come twice in most.
#pragma once
#include "attn_deal_units.h"

namespace pimdl {
namespace attn {

// What the shares of one call leave: share w's sums of a block that began in an earlier share in slot 2 w, of one that goes on in a later share in slot 2 w + 1.
struct DealPart {
    float* o;        // [2 shares][rows of a block][head_dim]
    f32x4* mlc;      // [2 shares][rows of a block]: m, l and c of a row
    u32x4* joins;    // [shares][2]: of the block that begins in a share and goes on: shares that have some of it (0: there is none), rows; first token, row and key head
};

template <typename C>
struct Deal {
    static constexpr uint32_t WAVES = PER_CU<C> == 2 ? 8 : 4, THREADS = WAVES * 64, ROWS = WAVES * 32;
    static constexpr int TILE = C::NK == 1 || (WAVES == 8 && C::HD <= 64) ? 64 : 32;  // (five tiles in LDS)
    // A tile's rows in LDS are an odd number of 32 bytes apart: reads of 8 rows at a part, and transposing ones of 8 rows at 4 parts, meet every bank as often, and a
    // step's place is a constant in its reads.
    static constexpr int PITCH = C::LB / 32 % 2 ? C::LB : C::LB + 32, PIECE = TILE * PITCH, BYTES = PIECE * C::NK + (C::HD % 32 ? 64 : 0);
    typedef Stage<C, TILE, THREADS> S;
    static __device__ __forceinline__ void store(const S& x, char* lds, uint32_t tid)
    {
#pragma unroll
        for (int u = 0; u < S::LOADS; ++u) {
            const uint32_t flat = u * THREADS + tid, row = flat / C::PARTS, part = flat % C::PARTS;
            if (S::TOTAL % THREADS && row >= TILE) continue;
            if constexpr (C::NK == 1) {
                *reinterpret_cast<u32x4*>(lds + row * PITCH + part * 16) = x.x[u];
            } else {
                char* to = lds + row * PITCH + part * 8;
                uint32_t lo[3], hi[3];
                pieces<false, 3>(number(x.x[u][0]), number(x.x[u][1]), lo);
                pieces<false, 3>(number(x.x[u][2]), number(x.x[u][3]), hi);
#pragma unroll
                for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2*>(to + n * PIECE) = (u32x2){lo[n], hi[n]};
            }
        }
    }
    static constexpr size_t SUMS = WAVES / 2 * Rows<C, 32>::DT * 16 * 64 * 4;  // of half of the waves
    struct Tiles {
        alignas(16) char k[3][BYTES];
        alignas(16) char v[2][BYTES];
    };
    struct Shared {
        union {
            Tiles tile;
            struct {
                float sums[SUMS / 4];
                float ml[WAVES / 2][2][64];
            };
        };
        uint8_t marks[2][TILE * C::PARTS];  // values that are not finite, of a tile that some rows see and others do not
        uint32_t bad[4];                    // whether there is one, by tile
        // of the rows of the batch: first unit, first token, keys
        uint32_t unit[DEAL_BATCH + 1], token[DEAL_BATCH + 1];
        int32_t length[DEAL_BATCH];
        uint32_t tmp[WAVES];
    };
};
// the same by numbers
inline uint32_t deal_rows(bool alone) { return alone ? 128 : 256; }
inline int32_t deal_tile(bool fp32_keys, uint32_t head_dim) { return fp32_keys && head_dim > 64 ? 32 : 64; }

template <typename C>
__device__ __forceinline__ DealRow deal_row(const AttnArgs& a, const Row& r)
{
    typedef Deal<C> D;
    if (r.n == 0) return {0, D::ROWS, 1, 1, 1};
    const uint32_t rows = r.n * a.group;
    return deal_row_of<D::TILE>(rows, D::ROWS, span_of<true>(a, r, 0, rows - 1, D::TILE).total);
}

// Looks at every row of the batch (up to DEAL_BATCH, a thread each); returns all units.
template <typename C>
__device__ __forceinline__ uint32_t deal_units(const AttnArgs& a, typename Deal<C>::Shared& sh)
{
    typedef Deal<C> D;
    constexpr uint32_t EACH = (DEAL_BATCH + D::THREADS - 1) / D::THREADS;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint32_t mine[EACH], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t b = tid * EACH + i;
        mine[i] = 0;
        if (b < a.batch) {
            const Row r = load_row(a.starts, a.seqs, a.tables, a.lengths, a.tokens, a.seq_count, a.table_width, a.page_shift, true, b);
            sh.token[b] = r.first;
            if (b == a.batch - 1) sh.token[a.batch] = r.first + r.n;
            sh.length[b] = r.length;
            mine[i] = deal_row<C>(a, r).units() * a.kv_heads;
        }
        sum = add_units(sum, mine[i]);
    }
    uint32_t x = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o);
        if (lane >= (uint32_t)o) x = add_units(x, y);
    }
    if (lane == 63) sh.tmp[wave] = x;
    __syncthreads();
    uint32_t before = __shfl_up(x, 1), total = 0;
    if (lane == 0) before = 0;
#pragma unroll
    for (uint32_t i = 0; i < D::WAVES; ++i) {
        if (i < wave) before = add_units(before, sh.tmp[i]);
        total = add_units(total, sh.tmp[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) {
        const uint32_t b = tid * EACH + i;
        if (b < a.batch) sh.unit[b] = before;
        before = add_units(before, mine[i]);
    }
    if (tid == 0) sh.unit[a.batch] = total;
    __syncthreads();
    return total;
}

// What a wave does with 32 keys, in two stretches of matrix instructions, each of which takes the time of several others: the scores of the NEXT 32 keys while
// the probabilities of this step's first 16 are worked out and taken apart, then this step's values, beside the other 16 and the next scores' maximum.  One or two waves on
// a SIMD leave it idle for every latency that the order of instructions leaves open, and the compiler's order -- a read of LDS, a wait, a product -- leaves 24 of them a step; so the
// order is fixed here: reads are AHEAD products before their own, and fences keep the vector instructions where they are.
template <typename C>
struct Step {
    typedef Rows<C, 32> R;
    static constexpr int PIECE = Deal<C>::PIECE, PITCH = Deal<C>::PITCH;
    static constexpr int KS = R::KS, KAHEAD = C::NK == 1 ? (KS < 4 ? KS : 4) : 1;
    static constexpr int VS = 2 * R::DT, VAHEAD = C::NK == 1 ? (VS < 4 ? VS : 4) : 1;
    u32x4 v[VS][C::NK];
    uint32_t piece[8][R::NP];  // of pairs of probabilities

    static __device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

    __device__ __forceinline__ void share(Rows<C, 32>& w, const float* s, float base, float& sum, int e)
    {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * e], w.c, -base)), y = __builtin_amdgcn_exp2f(fmaf(s[2 * e + 1], w.c, -base));
        sum += x + y;
        pieces<C::HALF, R::NP>(x, y, piece[e]);
#pragma unroll
        for (int n = 0; n < R::NP; ++n) asm volatile("" : "+v"(piece[e][n]));  // here, not where they are used
    }
    uint32_t at_k, at_v;  // where the lane's parts of K and V lie in a tile
    typedef __attribute__((address_space(3))) const u32x4* LdsRow;
    typedef __attribute__((address_space(3))) s16x4* LdsColumn;
    static __device__ __forceinline__ uint32_t address(const char* p) { return (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p); }

    __device__ __forceinline__ void begin()
    {
        const uint32_t j = R::row(), lane = threadIdx.x & 15, side = j / 16, g = R::group();
        at_k = j * PITCH + g * 16;
        at_v = (4 * g + (lane >> 2)) * PITCH + (2 * side + (lane >> 1 & 1)) * 16 + (lane & 1) * 8;
    }
    // Step i of the second product: 16 keys, i / DT, and a tile of dims, i % DT
    __device__ __forceinline__ void read(uint32_t lds, int i)
    {
#pragma unroll
        for (int n = 0; n < C::NK; ++n) {
            u32x2 half[2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
                half[e] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsColumn)(uintptr_t)(lds + at_v + (i / R::DT * 16 + 8 * e) * PITCH + i % R::DT * 64 + n * PIECE)));
            v[i][n] = (u32x4){half[0][0], half[0][1], half[1][0], half[1][1]};
        }
    }
    // WITH: probabilities of `old` on the way (none before the first scores)
    template <bool WITH>
    __device__ __forceinline__ void scores(Rows<C, 32>& w, uint32_t k, float* s, const float* old, float base, uint32_t lv)
    {
        u32x4 x[KS][C::NK];
        uint32_t from = k + at_k;
        asm("" : "+v"(from));  // (or sums with each step's place are kept in registers, and added to again)
        auto read_k = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < C::NK; ++n) x[i][n] = *(LdsRow)(uintptr_t)(from + i * 32 + n * PIECE);
        };
#pragma unroll
        for (int i = 0; i < KAHEAD; ++i) read_k(i);
        fence();
        float sum = 0.0f;
        typename R::Acc acc = (typename R::Acc)(0.0f);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            if (i + KAHEAD < KS) read_k(i + KAHEAD);
            u32x4 y[C::NQ];
#pragma unroll
            for (int n = 0; n < C::NQ; ++n) y[n] = w.q[n][i];
            R::template product<C::NQ>(x[i], y, acc);
            if (WITH) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e * KS / 4 == i) share(w, old, base, sum, e);
            }
            fence();
        }
        if (WITH) {
            w.l += sum;
#pragma unroll
            for (int i = 0; i < VAHEAD; ++i) read(lv, i);
            fence();
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = acc[e];
    }
    // the last step's probabilities
    __device__ __forceinline__ void shares(Rows<C, 32>& w, const float* old, float base, uint32_t lv)
    {
#pragma unroll
        for (int i = 0; i < VAHEAD; ++i) read(lv, i);
        fence();
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) share(w, old, base, sum, e);
        w.l += sum;
    }
    // o += V^T p, p of `old`; returns the lane's largest of `s`
    __device__ __forceinline__ float values(Rows<C, 32>& w, uint32_t lds, const float* old, float base, const float* s)
    {
        float mx = s[0], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < VS; ++i) {
            const int g = i / R::DT;
            u32x4 b[R::NP];
#pragma unroll
            for (int n = 0; n < R::NP; ++n) b[n] = (u32x4){piece[4 * g][n], piece[4 * g + 1][n], piece[4 * g + 2][n], piece[4 * g + 3][n]};
            if (i + VAHEAD < VS) read(lds, i + VAHEAD);
            R::template product<R::NP>(v[i], b, w.o[i % R::DT]);
#pragma unroll
            for (int e = 4; e < 8; ++e)
                if ((e - 4) * R::DT / 4 == i) share(w, old, base, sum, e);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (R::DT + e * R::DT / 16 == i) mx = fmaxf(mx, s[e]);
            fence();
        }
        w.l += sum;
        return mx;
    }
};

// Tiles from .. to - 1 (at least one) for this workgroup's rows.  KG (key groups) 1: a wave takes all keys of a tile; 2: the 32 that `half` says, of 64.  While tile t's values
// are worked on, the scores are tile t + 1's: K is a tile ahead of V in LDS, where it has three places and V two, and the next of both are on their way in
// registers.  One barrier a tile.  `ahead` has been asked for the first tile's pages.
template <typename C, int KG>
__device__ __forceinline__ void deal_tiles(const AttnArgs& a, const Row& r, uint32_t kh, Rows<C, 32>& w, const Span& span, int32_t from, int32_t to, int32_t all_hi, int64_t all_lo,
                                           bool works, uint32_t half, Ahead<C, Deal<C>::TILE>& ahead, typename Deal<C>::Shared& sh)
{
    typedef Deal<C> D;
    constexpr int TILE = D::TILE, STEPS = TILE / 32 / KG;
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), mine = KG == 1 ? 0 : 32 * half;
    typename D::S sk, sv;
    Place at_k, at_v;
    auto key_of = [&](int32_t t) { return span.at(t) * TILE; };
    auto fetch_k = [&](typename D::S& x, int32_t t) __attribute__((always_inline)) {
        at_k = place<C, TILE>(a, r, kh, key_of(t), ahead);
        x.fetch_by_wave(a.k, a, r, at_k, key_of(t), wave, tid);
    };
    auto is_mixed = [&](int32_t key0, uint32_t there) { return !(key0 + TILE <= all_hi && (key0 >= all_lo || key0 + TILE <= w.sinks)) || there != ~0u; };
    auto store_v = [&](int32_t t, uint32_t there) __attribute__((always_inline)) {
        const int buf = t & 1;
        if (is_mixed(key_of(t), there)) {
            sv.marked = true;  // (by whatever tile had this place before)
            if (sv.clear(sh.marks[buf], tid)) sh.bad[t & 3] = 1;
        }
        D::store(sv, sh.tile.v[buf], tid);
    };
    if (tid < 4) sh.bad[tid] = 0;
    uint32_t there0, there1 = ~0u, there2 = ~0u;  // of tiles t, t + 1 and t + 2
    {
        typename D::S first;
        fetch_k(first, from);
        there0 = at_k.there;
        sv.fetch_by_wave(a.v, a, r, at_k, key_of(from), wave, tid);
        ahead.ask(a, r, key_of(from + 1));
        if (from + 1 < to) {
            fetch_k(sk, from + 1);
            there1 = at_k.there;
            at_v = at_k;
            ahead.ask(a, r, key_of(from + 2));
        }
        __syncthreads();
        D::store(first, sh.tile.k[0], tid);
        store_v(from, there0);
        if (from + 1 < to) {
            D::store(sk, sh.tile.k[1], tid);
            sv.fetch_by_wave(a.v, a, r, at_v, key_of(from + 1), wave, tid);
            if (from + 2 < to) {
                fetch_k(sk, from + 2);
                there2 = at_k.there;
                at_v = at_k;
                ahead.ask(a, r, key_of(from + 3));
            }
        }
        __syncthreads();
    }
    int k0 = 0, k1 = 1, k2 = 2;  // places of tiles t, t + 1 and t + 2
    const uint32_t lds_k = Step<C>::address(sh.tile.k[0]) + mine * D::PITCH, lds_v = Step<C>::address(sh.tile.v[0]) + mine * D::PITCH;
    Step<C> step;
    step.begin();
    float s[16], base = 0.0f;
    auto hide = [&](float* x, int32_t key0, uint32_t there) __attribute__((always_inline)) {
        if (!w.all(key0, 32) || (there & 3) != 3) w.hide(x, key0, there);
    };
    if (works) {
        step.template scores<false>(w, lds_k, s, nullptr, 0.0f, 0);
        hide(s, key_of(from) + mine, there0 >> mine / 16);
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        base = w.template follow<16>(s, mx);
    }
    // Flags go round by four: that of t + 1 may be set, that of t read, and that of t + 2 is cleared.
    for (int32_t t = from; t < to; ++t) {
        uint32_t there3 = ~0u;
        if (tid == 0) sh.bad[(t + 2) & 3] = 0;
        if (t + 1 < to) {
            if (t + 2 < to) D::store(sk, sh.tile.k[k2], tid);
            store_v(t + 1, there1);
            if (t + 2 < to) {
                sv.fetch_by_wave(a.v, a, r, at_v, key_of(t + 2), wave, tid);
                if (t + 3 < to) {
                    fetch_k(sk, t + 3);
                    there3 = at_k.there;
                    at_v = at_k;
                    ahead.ask(a, r, key_of(t + 4));
                }
            }
        }
        if (works) {
            const uint32_t lv = lds_v + (t & 1) * (uint32_t)D::BYTES;
#pragma unroll
            for (int n = 0; n < STEPS; ++n) {
                const bool here = n + 1 < STEPS, more = here || t + 1 < to;
                const uint32_t next = lds_k + (here ? k0 * (uint32_t)D::BYTES + (n + 1) * 32 * D::PITCH : k1 * (uint32_t)D::BYTES);
                float x[16];
                if (more) {
                    step.template scores<true>(w, next, x, s, base, lv + n * 32 * D::PITCH);
                    if (here) hide(x, key_of(t) + 32 * (n + 1) + mine, there0 >> (2 * (n + 1) + mine / 16));
                    else hide(x, key_of(t + 1) + mine, there1 >> mine / 16);
                } else {
                    step.shares(w, s, base, lv + n * 32 * D::PITCH);
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = -INF;
                }
                const float mx = step.values(w, lv + n * 32 * D::PITCH, s, base, x);
                if (is_mixed(key_of(t), there0) && sh.bad[t & 3]) w.poison(sh.marks[t & 1] + (32 * n + mine) * C::PARTS, key_of(t) + 32 * n + mine, 32, there0 >> (2 * n + mine / 16));
                if (more) base = w.template follow<16>(x, mx);
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = x[i];
            }
        }
        const int k3 = k0;
        k0 = k1, k1 = k2, k2 = k3;
        there0 = there1, there1 = there2, there2 = there3;
        __syncthreads();
    }
}

// Which 32 rows a wave has, of `groups`, and whether it shares them with another wave, each with half of every tile: waves take turns on the four SIMDs, whose longest
// queue is the tile's time.  All of a few groups are shared, so that a SIMD has half a tile or two; of five and six, those that would be a second whole one.
struct Duty {
    uint32_t group, half, pair;  // (group WAVES: none)
    bool halves;
};
template <typename C>
__device__ __forceinline__ Duty duty_of(uint32_t wave, uint32_t groups)
{
    constexpr uint32_t WAVES = Deal<C>::WAVES, FIRST = WAVES / 2;
    if (Deal<C>::TILE != 64) return {wave, 0, 0, false};
    if (groups <= 2) return {wave < 4 ? wave % 2 : WAVES, wave / 2 % 2, wave % 2, true};
    if (groups <= FIRST) return {wave % FIRST, wave / FIRST, wave % FIRST, true};
    if (groups > FIRST + FIRST / 2 || wave < FIRST) return {wave, 0, 0, false};
    return {FIRST + (wave - FIRST) / 2, wave % 2, (wave - FIRST) / 2, true};
}

// Of two waves with the same rows the second hands its sums over to the first.
template <typename C>
__device__ __forceinline__ void deal_join_halves(Rows<C, 32>& w, const Duty& duty, typename Deal<C>::Shared& sh)
{
    typedef Rows<C, 32> R;
    const uint32_t lane = threadIdx.x & 63, pair = duty.pair;
    const bool half = duty.halves && duty.half && duty.group < Deal<C>::WAVES;
    float* const sums = sh.sums + pair * R::DT * 16 * 64 + lane;
    if (half) {
#pragma unroll
        for (int d = 0; d < R::DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[(16 * d + i) * 64] = w.o[d][i];
        sh.ml[pair][0][lane] = w.m;
        sh.ml[pair][1][lane] = w.l;
    }
    __syncthreads();
    if (half || !duty.halves) return;
    const float m = sh.ml[pair][0][lane], top = fmaxf(m, w.m), base = top == -INF ? 0.0f : top;
    const float f = __builtin_amdgcn_exp2f((w.m - base) * w.c), g = __builtin_amdgcn_exp2f((m - base) * w.c);
    w.m = top;
    w.l = w.l * f + sh.ml[pair][1][lane] * g;
#pragma unroll
    for (int d = 0; d < R::DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) w.o[d][i] = w.o[d][i] * f + sums[(16 * d + i) * 64] * g;
}

template <typename C>
__global__ __launch_bounds__(Deal<C>::THREADS, Deal<C>::WAVES / 4) void attention_deal_kernel(AttnArgs a, DealPart part)
{
    typedef Deal<C> D;
    __shared__ __attribute__((aligned(1024))) char shared[sizeof(typename D::Shared)];
    typename D::Shared& sh = *reinterpret_cast<typename D::Shared*>(shared);
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = tid & 31, h = tid >> 5 & 1;
    const uint32_t total = __builtin_amdgcn_readfirstlane(deal_units<C>(a, sh)), per = share_of(total, gridDim.x);
    // neighbouring shares on one XCD (workgroups are dealt out to 8 in turn): blocks of one key head share its keys
    const uint32_t share = gridDim.x % 8 == 0 ? blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
    uint32_t unit = share * per;  // (units are below 2^31)
    const uint32_t stop = unit + per < total ? unit + per : total;
    if (tid == 0) part.joins[2 * share] = (u32x4){0, 0, 0, 0};
    if (unit >= stop) return;
    uint32_t b = 0;
    for (uint32_t up = a.batch; up - b > 1;) {
        const uint32_t mid = (b + up) / 2;
        if (sh.unit[mid] <= unit) b = mid;
        else up = mid;
    }
    while (unit < stop) {
        while (sh.unit[b + 1] <= unit) ++b;  // (there is one: unit is below total)
        b = __builtin_amdgcn_readfirstlane(b);
        Row r;
        r.first = __builtin_amdgcn_readfirstlane(sh.token[b]);
        const uint32_t behind = __builtin_amdgcn_readfirstlane(sh.token[b + 1]);
        r.n = behind > r.first ? behind - r.first : 0;  // (not 0: the row has units)
        r.length = __builtin_amdgcn_readfirstlane(sh.length[b]);
        r.pos0 = r.length - (int32_t)r.n;
        const int32_t seq = a.seqs ? a.seqs[b] : (int32_t)b;
        r.table = a.tables + (size_t)(r.length > 0 ? seq : 0) * a.table_width;  // (read where there are keys)
        const DealRow d = deal_row<C>(a, r);
        // the block that `unit` lies in, its first unit and those of its tiles
        const DealPiece p = deal_piece(d, __builtin_amdgcn_readfirstlane(sh.unit[b]), unit, stop);
        const uint32_t kh = p.kh, block = p.block;
        const int32_t most = (int32_t)d.tiles, from = p.from, to = p.to;
        unit = p.end < stop ? p.end : stop;
        if (from >= to) continue;
        const uint32_t rows = r.n * a.group, row0 = block * d.rows, end = row0 + d.rows < rows ? row0 + d.rows : rows;
        const Duty duty = duty_of<C>(wave, (end - row0 + 31) / 32);
        const uint32_t half = duty.half, mine = row0 + 32 * duty.group;
        const Span span = span_of<true>(a, r, row0, end - 1, D::TILE);  // (a part of the last block's: only its end may come earlier)
        const bool works = mine < end;
        const int32_t until = to < span.total ? to : span.total;
        Ahead<C, D::TILE> ahead;  // (on the way together with the queries)
        if (from < until) ahead.ask(a, r, span.at(from) * D::TILE);
        Rows<C, 32> w;
        w.begin(a, r, kh, works ? mine : row0, rows);
        const int32_t all_hi = r.pos0 < 0 ? 0 : r.pos0;
        const int64_t all_lo = (int64_t)r.pos0 + (end - 1) / a.group - a.left;
        __syncthreads();  // everybody is done with the block before
        if (from < until) {
            // (a barrier for each tile on either way)
            if (D::TILE == 64 && duty.halves) deal_tiles<C, D::TILE / 32>(a, r, kh, w, span, from, until, all_hi, all_lo, works, half, ahead, sh);
            else deal_tiles<C, 1>(a, r, kh, w, span, from, until, all_hi, all_lo, works, 0, ahead, sh);
            if (D::TILE == 64) deal_join_halves<C>(w, duty, sh);
        }
        if (half == 0 && mine + j < end) {
            const float l = row_sum<32>(w.l);
            if (from == 0 && to == most) {
                const uint32_t row = mine + j, token = r.first + row / a.group, head = kh * a.group + row % a.group;
                typename C::TQ* out = static_cast<typename C::TQ*>(a.out) + (size_t)token * a.out_stride + (size_t)head * C::HD;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int dd = 0; dd < w.DT; ++dd)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (32 * dd + 8 * i < C::HD) store4(out + 32 * dd + 8 * i + 4 * h, w.quad(dd, i) * inv);
            } else {
                const size_t row = (size_t)(2 * share + (from == 0)) * D::ROWS + (mine - row0) + j;
                if (h == 0) part.mlc[row] = (f32x4){w.m, l, w.c, 0.0f};
#pragma unroll
                for (int dd = 0; dd < w.DT; ++dd)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (32 * dd + 8 * i < C::HD) store4(part.o + row * C::HD + 32 * dd + 8 * i + 4 * h, w.quad(dd, i));
            }
        }
        if (tid == 0 && from == 0 && to < most) {
            part.joins[2 * share] = (u32x4){deal_shares(p, d.tiles, per, share, gridDim.x), end - row0, 0, 0};
            part.joins[2 * share + 1] = (u32x4){r.first, row0, kh, 0};
        }
    }
}

}  // namespace attn
}  // namespace pimdl
