// Attention of a ragged batch on the matrix cores (gfx950), for one pair of types; included by a translation unit per pair.
//
// Work is cut into tiles of ROWS: row r of a sequence and key head is (token r / group, query head r % group of the key head's
// group), so query heads that share a key head share what is read of the cache.  A wave holds 32 rows and takes keys 32 at a time.
// Both products run on v_mfma_f32_32x32x16, transposed, so that a lane keeps to one row and nothing changes lanes in between:
//   S^T[key][row] = K Q^T:   A = K (32 keys x 16 dims), B = the rows' q.  Lane (row j, half h) gets keys 8 (i / 4) + 4 h + i % 4,
//                            i = 0 .. 15: a row's maximum and sum are 16 registers and one exchange between halves.
//   O^T[dim][row] += V^T P^T: the B operand of 16 keys is 8 of those very registers, in 16-bit pieces; the A operand has to hold the same keys in the
//                            same places, which are two groups of 4 consecutive keys for each half: two transposing reads of LDS
//                            (ds_read_b64_tr_b16: 16 lanes take 4 rows of 16 columns and get a column of 4 each).
// Streaming softmax: m is a running maximum of a row's raw scores (RISE below), p = 2^(c s - c m) with c = scale log2(e), l the sum of p; o and l
// are multiplied by 2^(c (m - m')) when m rises.
//
// fp32 operands are taken apart into 16-bit pieces, so that the products run at the 16-bit rate and keep 24 bits: three bf16
// pieces by truncation (exact: 8 + 8 + 8 bits), of whose nine products the six that reach 2^-24 are taken; over a cache in halves
// q (brought to 2^11 .. 2^12 by a power of two of its row) and p (times 2^7) are two halves, 22 bits and nothing subnormal that counts.
// Against v_mfma_f32_32x32x2_f32, 1 / 16 of the 16-bit rate, that is 6 / 16, 3 / 16 and 2 / 16 of the time.
#pragma once
#include <type_traits>

#include "serve_common.h"

namespace pimdl {
namespace attn {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float INF = __builtin_inff();
// The maximum that p is relative to follows the scores only when they pass it by a factor of 2^RISE: until then p and l just grow beyond 1, which
// rounds no differently, and o, 16 to 64 registers, is left alone.
constexpr float RISE = 8.0f;

// TQ: q and out; TK: keys and values
template <typename TQ_, typename TK_, int HD_, bool PAGED_>
struct Config {
    typedef TQ_ TQ;
    typedef TK_ TK;
    static constexpr int HD = HD_;
    static constexpr bool PAGED = PAGED_;
    static constexpr bool HALF = std::is_same<TK, _Float16>::value;  // the products' type: halves, or bf16
    static constexpr int NK = std::is_same<TK, float>::value ? 3 : 1;
    static constexpr int NQ = std::is_same<TQ, float>::value ? (HALF ? 2 : 3) : 1;
    static constexpr int LB = HD * 2;           // bytes of a row of one piece in LDS
    static constexpr int RB = HD * (int)sizeof(TK);  // ... in memory
    static constexpr int PARTS = HD * (int)sizeof(TK) / 16;  // 16-byte parts of a row in memory
    // p, up to 2^8 (RISE), is carried times 2^7 in halves, whose values leave room for that, and times 2^-8 otherwise: at most 1, so that a value near
    // the type's largest stays finite
    static constexpr int P_SHIFT = HALF ? 7 : -8;
};

// Order of a row's 16-byte parts in LDS: part ^ order(row).  Rows of the first product's reads are 32 consecutive ones at one part; the
// transposing reads take 4 consecutive rows at 4 parts: both meet every bank once per 16 lanes at 32, 64, 96 and 128 dims (80: twice).
template <int HD>
__device__ __forceinline__ constexpr uint32_t order(uint32_t row)
{
    if (HD == 128) return (row & 3) << 2 | (row >> 2 & 3);
    if (HD == 64) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
    if (HD == 80) return 0;
    return row >> 2 & 3;
}

template <bool HALF>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (HALF) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool HALF>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t bits(float x) { return __builtin_bit_cast(uint32_t, x); }
__device__ __forceinline__ float number(uint32_t x) { return __builtin_bit_cast(float, x); }
__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

// Two floats as N 16-bit pieces each, piece by piece.
template <bool HALF, int N>
__device__ __forceinline__ void pieces(float x, float y, uint32_t* out)
{
    if constexpr (HALF) {
        f16x2 a = {(_Float16)x, (_Float16)y};
        out[0] = __builtin_bit_cast(uint32_t, a);
        if constexpr (N == 2) {
            f16x2 b = {(_Float16)(x - (float)a[0]), (_Float16)(y - (float)a[1])};
            out[1] = __builtin_bit_cast(uint32_t, b);
        }
    } else if constexpr (N == 1) {
        bf16x2 a = {(__bf16)x, (__bf16)y};
        out[0] = __builtin_bit_cast(uint32_t, a);
    } else if constexpr (N == 2) {
        bf16x2 a = {(__bf16)x, (__bf16)y}, b = {(__bf16)(x - (float)a[0]), (__bf16)(y - (float)a[1])};
        out[0] = __builtin_bit_cast(uint32_t, a);
        out[1] = __builtin_bit_cast(uint32_t, b);
    } else {
        out[0] = high_halves(bits(x), bits(y));
        x -= number(bits(x) & 0xffff0000u);
        y -= number(bits(y) & 0xffff0000u);
        out[1] = high_halves(bits(x), bits(y));
        x -= number(bits(x) & 0xffff0000u);
        y -= number(bits(y) & 0xffff0000u);
        out[2] = high_halves(bits(x), bits(y));
    }
}

// maximum and sum over the lanes that share a row: the swapped pair holds both sides' values
template <int M>
__device__ __forceinline__ float row_max(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
    v = fmaxf(number(r[0]), number(r[1]));
    if constexpr (M == 16) {
        const auto t = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
        v = fmaxf(number(t[0]), number(t[1]));
    }
    return v;
}
template <int M>
__device__ __forceinline__ float row_sum(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
    v = number(r[0]) + number(r[1]);
    if constexpr (M == 16) {
        const auto t = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
        v = number(t[0]) + number(t[1]);
    }
    return v;
}

// Where the keys of a tile lie.  A tile begins at a multiple of 16, pages hold multiples of 16: a group of 16 keys has one base address.  The table's
// entries are asked for a tile ahead, by a load of the vector memory like the keys', which return in order (a scalar load in flight makes
// every wait for LDS a wait for all of LDS: 4 prompts of 4096 tokens 772 us with scalar loads, 673, shares being in one piece then; 860 in two): lane i % GROUPS has group i's.
template <typename C, int TILE>
struct Ahead {
    int32_t entry = 0;
    __device__ __forceinline__ void ask(const AttnArgs& a, const Row& r, int32_t key0)
    {
        if constexpr (C::PAGED) {
            const int32_t key = key0 + 16 * (int32_t)(threadIdx.x % (TILE / 16));
            entry = -1;
            if (key < r.length) entry = r.table[key >> a.page_shift];
        }
    }
};
// Keys behind the sequence or on no page are read from an address that exists; `there` has a bit for each group that is.
struct Place {
    int64_t base0, base1, base2, base3;  // bytes from k or v, of each group (not paged: base0, of the sequence)
    uint32_t there;
};

template <typename C, int TILE>
__device__ __forceinline__ Place place(const AttnArgs& a, const Row& r, uint32_t kh, int32_t key0, const Ahead<C, TILE>& ahead)
{
    Place p;
    p.there = ~0u;
    p.base0 = p.base1 = p.base2 = p.base3 = 0;
    if constexpr (C::PAGED) {
        // every lane for its own group, on the vector unit: a wave gets a scalar instruction through in four times the time
        const uint32_t page_bytes = (a.kv_heads << a.page_shift) * (uint32_t)C::RB, lane_group = threadIdx.x % (TILE / 16);
        const bool there = (uint32_t)ahead.entry < a.pages;  // (not -1)
        const uint32_t row = (kh << a.page_shift) + ((uint32_t)(key0 + 16 * (int32_t)lane_group) & ((1u << a.page_shift) - 1));
        const uint64_t base = (uint64_t)(there ? (uint32_t)ahead.entry : 0u) * page_bytes + row * (uint32_t)C::RB;
        p.there = (uint32_t)__ballot(there) | ~((1u << TILE / 16) - 1);
        auto of_group = [&](int g) {
            return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(base >> 32), g) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)base, g));
        };
        p.base0 = of_group(0);
        p.base1 = of_group(1);
        if constexpr (TILE == 64) {
            p.base2 = of_group(2);
            p.base3 = of_group(3);
        }
    } else {
        p.base0 = ((int64_t)r.first * a.kv_stride + (int64_t)kh * C::HD) * (int64_t)sizeof(typename C::TK);
    }
    return p;
}

// Copies a tile of keys or values by THREADS threads (of `wave`, where there are several) through registers: fetch() asks for it, store() puts it into
// LDS, piece by piece.
template <typename C, int TILE, int THREADS>
struct Stage {
    static constexpr int TOTAL = TILE * C::PARTS, LOADS = (TOTAL + THREADS - 1) / THREADS;
    static constexpr int PIECE = TILE * C::LB;                   // bytes of a piece in LDS
    static constexpr int BYTES = PIECE * C::NK + (C::HD % 32 ? 64 : 0);  // (a half tile of dims reads past the last row)
    u32x4 x[LOADS];
    bool marked = false;  // this thread has left marks

    __device__ __forceinline__ void fetch(const void* src, const AttnArgs& a, const Row& r, const Place& p, int32_t key0, uint32_t wave, uint32_t tid)
    {
        const char* const s = static_cast<const char*>(src);
        if constexpr (C::PAGED && 64 % C::PARTS == 0) {  // a wave's load is whole rows of one group: 1 KiB on end
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const uint32_t row = (u * THREADS + wave * 64) / C::PARTS, g = row >> 4;
                const int64_t base = g == 0 ? p.base0 : g == 1 ? p.base1 : g == 2 ? p.base2 : p.base3;
                x[u] = *reinterpret_cast<const u32x4*>(s + base + (row & 15) * C::RB + (tid & 63) * 16);
            }
        } else if constexpr (C::PAGED) {
            const int64_t step1 = p.base1 - p.base0, step2 = p.base2 - p.base1, step3 = p.base3 - p.base2;
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                const uint32_t flat = u * THREADS + tid, part = flat % C::PARTS;
                uint32_t row = flat / C::PARTS;
                if (TOTAL % THREADS && row >= TILE) row = TILE - 1;  // (not stored)
                int64_t at = p.base0 + (row & 15) * C::RB + part * 16;
                at += row < 16 ? 0 : step1;
                if constexpr (TILE == 64) {
                    at += row < 32 ? 0 : step2;
                    at += row < 48 ? 0 : step3;
                }
                x[u] = *reinterpret_cast<const u32x4*>(s + at);
            }
        } else {
            const uint32_t pitch = a.kv_stride * (uint32_t)sizeof(typename C::TK);  // (a tile is less than 4 GiB of rows)
            const char* const base = s + p.base0 + (int64_t)key0 * pitch;
            auto load = [&](int u, uint32_t last) {
                const uint32_t flat = u * THREADS + tid, row = flat / C::PARTS;
                x[u] = *reinterpret_cast<const u32x4*>(base + ((row < last ? row : last) * pitch + flat % C::PARTS * 16));
            };
            if (key0 + TILE <= r.length) {
#pragma unroll
                for (int u = 0; u < LOADS; ++u) load(u, TILE - 1);
            } else {
#pragma unroll
                for (int u = 0; u < LOADS; ++u) load(u, (uint32_t)(r.length - 1 - key0));
            }
        }
    }
    __device__ __forceinline__ void no_marks(uint8_t* marks, uint32_t tid)
    {
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
            if (TOTAL % THREADS == 0 || u * THREADS + tid < TOTAL) marks[u * THREADS + tid] = 0;
        marked = false;
    }
    // Before store() of values that some rows see and others do not: elements that are not finite become zeros and get a bit in `marks`, a
    // byte per part of a row; whether there is one
    __device__ __forceinline__ bool clear(uint8_t* marks, uint32_t tid)
    {
        // an exponent of all ones carries into the bit above it
        constexpr uint32_t ones = C::NK == 3 ? 0x7f800000u : C::HALF ? 0x7c007c00u : 0x7f807f80u;
        constexpr uint32_t carry = C::NK == 3 ? 0x00800000u : C::HALF ? 0x04000400u : 0x00800080u, sign = C::NK == 3 ? 0x80000000u : 0x80008000u;
        uint32_t any = 0;
#pragma unroll
        for (int u = 0; u < LOADS; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= (x[u][i] & ones) + carry;
        if (marked) no_marks(marks, tid);
        if (!(any & sign)) return false;
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            uint32_t found = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t bad = ((x[u][i] & ones) + carry) & sign;
                if constexpr (C::NK == 3) {
                    found |= (bad >> 31) << i;
                    if (bad) x[u][i] = 0;
                } else {
                    found |= (bad >> 15 & 1) << 2 * i | (bad >> 31) << (2 * i + 1);
                    if (bad & 0x8000u) x[u][i] &= 0xffff0000u;
                    if (bad & 0x80000000u) x[u][i] &= 0xffffu;
                }
            }
            if (TOTAL % THREADS == 0 || u * THREADS + tid < TOTAL) marks[u * THREADS + tid] = (uint8_t)found;
        }
        marked = true;
        return true;
    }
    __device__ __forceinline__ void store(char* lds, uint32_t tid) const
    {
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const uint32_t flat = u * THREADS + tid, row = flat / C::PARTS, part = flat % C::PARTS;
            if (TOTAL % THREADS && row >= TILE) continue;
            if constexpr (C::NK == 1) {
                *reinterpret_cast<u32x4*>(lds + row * C::LB + ((part ^ order<C::HD>(row)) << 4)) = x[u];
            } else {
                char* to = lds + row * C::LB + (((part >> 1) ^ order<C::HD>(row)) << 4) + (part & 1) * 8;
                uint32_t lo[3], hi[3];
                pieces<false, 3>(number(x[u][0]), number(x[u][1]), lo);
                pieces<false, 3>(number(x[u][2]), number(x[u][3]), hi);
#pragma unroll
                for (int n = 0; n < 3; ++n) *reinterpret_cast<u32x2*>(to + n * PIECE) = (u32x2){lo[n], hi[n]};
            }
        }
    }
};

// The M (32 or 16) rows of one wave and what it has of their result.  Lane (row j, group g): j = lane % M, g = lane / M.
template <typename C, int M>
struct Rows {
    static constexpr int GROUPS = 64 / M, REGS = 32 / GROUPS;  // REGS: scores of 32 keys that a lane holds
    static constexpr int STEP = 8 * GROUPS, KS = (C::HD + STEP - 1) / STEP;  // steps of the first product, in dims; of the last one of 80 dims,
    static constexpr bool REST = C::HD % STEP != 0;                          // M == 16, groups 2 and 3 repeat the dims of 0 and 1 against zeros of q
    static constexpr int DT = (C::HD + M - 1) / M;             // tiles of the second (80 dims, M == 32: of the last one only half counts)
    static constexpr int QUADS = REGS / 4, OREGS = M * M / 64, OQUADS = OREGS / 4;
    // pieces of p: two in 16 bits, 16 or 22 bits of it, so that the output alone is rounded to 16 and a token's result does not depend on how many others
    // share its call.  One piece would save many rows a third of their matrix instructions (6 prompts, window 1024, bf16: 318 us against 408) and put
    // 2.06e-3 between them and 64 bits where rounding the output takes 1.58e-3; few rows wait for memory.
    static constexpr int NP = C::NQ == 1 ? 2 : C::NQ;
    typedef typename std::conditional<M == 32, f32x16, f32x4>::type Acc;
    static constexpr int KT = M == 32 ? 1 : 2;  // accumulators of 32 keys

    u32x4 q[C::NQ][KS];
    float c;                  // scores times c are exponents of 2
    int32_t lo, hi, sinks;    // of this lane's row: keys lo .. hi - 1 and 0 .. sinks - 1 are seen
    int32_t min_hi, max_hi, min_lo, max_lo;  // over the wave's rows
    float m, l;
    Acc o[DT];

    static __device__ __forceinline__ uint32_t row() { return threadIdx.x % M; }
    static __device__ __forceinline__ uint32_t group() { return (threadIdx.x & 63) / M; }
    // which key of 32, or which dim of a tile, register i of this lane holds
    static __device__ __forceinline__ int32_t place_of(int i) { return 4 * GROUPS * (i >> 2) + 4 * (int32_t)group() + (i & 3); }

    // the 8 dims that this lane has in step s of the first product
    static __device__ __forceinline__ uint32_t dims(int s) { return STEP * s + 8 * (REST && s == KS - 1 ? group() & 1 : group()); }

    // row0: first row of the wave, rows: of the sequence and key head
    __device__ __forceinline__ void begin(const AttnArgs& a, const Row& r, uint32_t kh, uint32_t row0, uint32_t rows)
    {
        const uint32_t g = group(), mine = row0 + row() < rows ? row0 + row() : rows - 1;  // rows past the last repeat it; they are never stored
        const uint32_t token = mine / a.group, head = kh * a.group + mine % a.group;
        const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;  // c is positive, so that the largest score has the largest exponent
        c = (a.scale == 0.0f ? 1.0f : fabsf(a.scale)) * LOG2E;
        const typename C::TQ* const base = static_cast<const typename C::TQ*>(a.q) + (size_t)(r.first + token) * a.q_stride + (size_t)head * C::HD;
        if constexpr (C::NQ == 1) {
            const uint32_t flip = sign < 0.0f ? 0x80008000u : 0u, keep = sign == 0.0f ? 0u : ~0u;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                q[0][s] = (*reinterpret_cast<const u32x4*>(base + dims(s)) ^ flip) & keep;
                if (REST && s == KS - 1 && g >= 2) q[0][s] = (u32x4){0, 0, 0, 0};
            }
        } else {
            f32x4 x[2 * KS];
#pragma unroll
            for (int s = 0; s < 2 * KS; ++s) {
                x[s] = *reinterpret_cast<const f32x4*>(base + dims(s / 2) + 4 * (s & 1));
                if (REST && s / 2 == KS - 1 && g >= 2) x[s] = (f32x4){0.f, 0.f, 0.f, 0.f};
            }
            float factor = sign;
            if constexpr (C::HALF) {  // the row's largest magnitude to 2^11 .. 2^12
                float big = 0.0f;
#pragma unroll
                for (int s = 0; s < 2 * KS; ++s) big = fmaxf(fmaxf(big, fmaxf(fabsf(x[s][0]), fabsf(x[s][1]))), fmaxf(fabsf(x[s][2]), fabsf(x[s][3])));
                big = row_max<M>(big);
                int e = 11 - ((int)(bits(big) >> 23 & 255) - 127);
                e = e > 126 ? 126 : e;  // (-117 at least)
                factor *= number((uint32_t)(127 + e) << 23);
                c *= number((uint32_t)(127 - e) << 23);
            }
            c = fminf(fmaxf(c, 1.4e-45f), 3e38f);  // (0 or infinity times a hidden score would be NaN)
#pragma unroll
            for (int s = 0; s < 2 * KS; ++s) {
                uint32_t w[2][C::NQ];
                pieces<C::HALF, C::NQ>(x[s][0] * factor, x[s][1] * factor, w[0]);
                pieces<C::HALF, C::NQ>(x[s][2] * factor, x[s][3] * factor, w[1]);
#pragma unroll
                for (int n = 0; n < C::NQ; ++n) q[n][s / 2][2 * (s & 1)] = w[0][n], q[n][s / 2][2 * (s & 1) + 1] = w[1][n];
            }
        }
        auto border_hi = [&](uint32_t t) {
            const int64_t e = (int64_t)r.pos0 + t + a.right + 1;
            return (int32_t)(e < 0 ? 0 : e < r.length ? e : r.length);
        };
        auto border_lo = [&](uint32_t t) {
            const int64_t e = (int64_t)r.pos0 + t - a.left;
            return (int32_t)(e < 0 ? 0 : e < 0x7fffffff ? e : 0x7fffffff);
        };
        sinks = a.sinks < 0x7fffffffu ? (int32_t)a.sinks : 0x7fffffff;
        hi = border_hi(token);
        lo = border_lo(token);
        const uint32_t t0 = row0 / a.group, t1 = (row0 + 32 < rows ? row0 + 31 : rows - 1) / a.group;
        min_hi = border_hi(t0), max_hi = border_hi(t1), min_lo = border_lo(t0), max_lo = border_lo(t1);
        m = -INF;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = (Acc)(0.0f);
    }

    // keys key0 .. key0 + n - 1: whether some row sees some of them, whether every row sees all of them
    __device__ __forceinline__ bool some(int32_t key0, int32_t n) const { return key0 < max_hi && (key0 + n > min_lo || key0 < sinks); }
    __device__ __forceinline__ bool all(int32_t key0, int32_t n) const { return key0 + n <= min_hi && (key0 >= max_lo || key0 + n <= sinks); }
    __device__ __forceinline__ bool sees(int32_t key) const { return key < hi && (key >= lo || key < sinks); }

    // of a product of N and NK pieces those that reach the last bit of the larger count, small ones first
    template <int N>
    static __device__ __forceinline__ void product(const u32x4* x, const u32x4* y, Acc& sum)
    {
#pragma unroll
        for (int w = C::NK == 1 ? N - 1 : 2; w >= 0; --w)
#pragma unroll
            for (int n = 0; n < C::NK; ++n)
                if (w - n >= 0 && w - n < N) sum = mfma<C::HALF>(x[n], y[w - n], sum);
    }

    // scores of 32 keys, which lie in LDS from `k` on, pieces PIECE bytes apart
    template <int PIECE>
    __device__ __forceinline__ void scores(const char* k, float* s) const
    {
        const uint32_t j = row();
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            Acc acc = (Acc)(0.0f);
            const char* const at = k + (t * M + j) * C::LB;
#pragma unroll
            for (int st = 0; st < KS; ++st) {
                u32x4 x[C::NK], y[C::NQ];
#pragma unroll
                for (int n = 0; n < C::NK; ++n) x[n] = *reinterpret_cast<const u32x4*>(at + n * PIECE + (((dims(st) / 8) ^ order<C::HD>(t * M + j)) << 4));
#pragma unroll
                for (int n = 0; n < C::NQ; ++n) y[n] = q[n][st];
                product<C::NQ>(x, y, acc);
            }
#pragma unroll
            for (int i = 0; i < OREGS; ++i) s[t * OREGS + i] = acc[i];
        }
    }

    // Hides what the row does not see among 32 keys from key0 on; `there`: bits of the two groups of 16 that exist.
    __device__ __forceinline__ void hide(float* s, int32_t key0, uint32_t there) const
    {
        const int32_t k0 = key0 + 4 * (int32_t)group();
        auto at = [](int i) { return 4 * GROUPS * (i >> 2) + (i & 3); };  // (place_of without the group)
        if (key0 + 32 > min_hi) {
            const int32_t h = hi - k0;
#pragma unroll
            for (int i = 0; i < REGS; ++i) s[i] = at(i) < h ? s[i] : -INF;
        }
        if (key0 < max_lo) {
            const int32_t f = lo - k0;
            if (key0 >= sinks) {
#pragma unroll
                for (int i = 0; i < REGS; ++i) s[i] = at(i) >= f ? s[i] : -INF;
            } else {
                const int32_t e = sinks - k0;
#pragma unroll
                for (int i = 0; i < REGS; ++i) s[i] = at(i) >= f || at(i) < e ? s[i] : -INF;
            }
        }
        if (C::PAGED && (there & 3) != 3) {
#pragma unroll
            for (int i = 0; i < REGS; ++i)
                if (!(there >> (i / (REGS / 2)) & 1)) s[i] = -INF;
        }
    }

    // The N scores that a lane holds become probabilities; o and l follow the maximum.
    template <int N>
    __device__ __forceinline__ void softmax(float* s)
    {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < N; ++i) mx = fmaxf(mx, s[i]);
        mx = row_max<M>(mx);
        if (__any((mx - m) * c > RISE)) {
            const float up = (mx - m) * c > RISE ? mx : m;  // each row by its own scores: what others see must not round it differently
            const float alpha = __builtin_amdgcn_exp2f((m - (up == -INF ? 0.0f : up)) * c);  // 0 at the first keys
            m = up;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= alpha;
        }
        float base = m == -INF ? 0.0f : m * c;
        const bool far = fabsf(base) > 0x1p10f;
        if (__any(far)) {  // (rare) the rounding of m c, a factor of up to 2^(2^-15) below, would be one that counts
            const float most = far ? m : 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] -= most;
            base = far ? 0.0f : base;
        }
        base -= (float)C::P_SHIFT;
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -base));
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) sum += s[i];
        l += sum;
    }

    // o += V^T p for 32 keys, which lie in LDS from `v` on
    template <int PIECE>
    __device__ __forceinline__ void values(const char* v, const float* p)
    {
        const uint32_t i = threadIdx.x & 15, side = row() / 16, g = group();
#pragma unroll
        for (int st = 0; st < REGS / 8; ++st) {
            uint32_t w[4][NP];
#pragma unroll
            for (int e = 0; e < 4; ++e) pieces<C::HALF, NP>(p[8 * st + 2 * e], p[8 * st + 2 * e + 1], w[e]);
            u32x4 b[NP];
#pragma unroll
            for (int n = 0; n < NP; ++n) b[n] = (u32x4){w[0][n], w[1][n], w[2][n], w[3][n]};
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                u32x4 x[C::NK];
#pragma unroll
                for (int n = 0; n < C::NK; ++n) {
                    u32x2 half[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t key = 4 * GROUPS * (2 * st + e) + 4 * g + (i >> 2), part = M / 8 * d + 2 * side + (i >> 1 & 1);
                        const char* at = v + n * PIECE + key * C::LB + ((part ^ order<C::HD>(key)) << 4) + (i & 1) * 8;
                        half[e] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
                    }
                    x[n] = (u32x4){half[0][0], half[0][1], half[1][0], half[1][1]};
                }
                product<NP>(x, b, o[d]);
            }
        }
    }

    // NaN where a row sees one of the `n` keys from key0 on whose value is marked.  Keys on no page are seen by nobody.
    __device__ __forceinline__ void poison(const uint8_t* marks, int32_t key0, int32_t n, uint32_t there)
    {
        for (int32_t key = 0; key < n; ++key) {
            const bool seen = sees(key0 + key) && (there >> (key >> 4) & 1);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < OQUADS; ++i) {
                    if (M * d + 4 * GROUPS * i >= C::HD) continue;
                    const uint32_t dim = M * d + place_of(4 * i);
                    const uint32_t mark = seen ? (uint32_t)marks[key * C::PARTS + dim / (C::NK == 3 ? 4 : 8)] >> (C::NK == 3 ? 0 : dim & 4) : 0u;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (mark >> e & 1) o[d][4 * i + e] = __builtin_nanf("");
                }
        }
    }

    __device__ __forceinline__ f32x4 quad(int d, int i) const { return (f32x4){o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]}; }
};

// Results of keys that are split over workgroups: per split and row of the output (token, head) the sums, the maximum m that they are relative
// to, and l; per row c, which the first split leaves.  Joins take 2^(c (m - m')): of c m itself the rounding would be a factor of its own between large
// scores.
struct Partial {
    float* o;    // [splits][rows][head_dim]
    float* ml;   // [splits][rows][2]
    float* c;    // [rows]
    uint64_t rows;
    __device__ __forceinline__ void put(uint32_t split, uint64_t row, float m, float l, float scale) const
    {
        const uint64_t at = split * rows + row;
        ml[2 * at] = m;
        ml[2 * at + 1] = l;
        if (split == 0) c[row] = scale;
    }
};

template <typename TQ>
__device__ __forceinline__ void store4(TQ* to, f32x4 x)
{
    if constexpr (std::is_same<TQ, float>::value) {
        *reinterpret_cast<f32x4*>(to) = x;
    } else {
        struct alignas(8) Four {
            TQ v[4];
        } y = {{(TQ)x[0], (TQ)x[1], (TQ)x[2], (TQ)x[3]}};
        *reinterpret_cast<Four*>(to) = y;
    }
}

// The key tiles that a tile of rows has to look at: those of the first `sinks` keys that lie before the window, then the window's.
struct Span {
    int32_t first, sinks, total;
    __device__ __forceinline__ int32_t at(int32_t t) const { return t < sinks ? t : first + (t - sinks); }
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, const Row& r, uint32_t row0, uint32_t row1, int32_t tile)
{
    const int64_t top = (int64_t)r.pos0 + row1 / a.group + a.right + 1, low = (int64_t)r.pos0 + row0 / a.group - a.left;
    const int32_t hi = (int32_t)(top < 0 ? 0 : top < r.length ? top : r.length), lo = (int32_t)(low < 0 ? 0 : low < hi ? low : hi);
    Span s;
    s.first = lo / tile;
    const int32_t sinks = a.sinks < (uint32_t)lo ? (int32_t)a.sinks : lo, n = (sinks + tile - 1) / tile, last = (hi + tile - 1) / tile;
    s.sinks = n < s.first ? n : s.first;
    s.total = s.sinks + (last > s.first ? last - s.first : 0);
    return s;
}

// ------------------------------------------------------------------------------------------------------------
// Many rows: a workgroup takes 128 rows of a sequence and key head, its four waves 32 each, and all of them go through the same tiles of keys and
// values in LDS.  The next tile is on its way in registers while one is worked on.  128 rows read keys and values once where 64 would twice; at 32 rows a
// wave o, q, the scores and the tile to come are 168 to 256 registers, two waves per SIMD.  Bound by what those two waves leave uncovered between products and exponentials:
// whole sequences of 4096 tokens, 32 heads over 8, bf16, 719 TFLOP/s (matrix instructions, a third of them for the second piece of p, 53 % of the SIMDs' cycles,
// others 50 %); 6 prompts of up to 4096, window 1024, 404 us, 570 TFLOP/s (45 and 49 %): tiles at a window's two borders are taken whole, 1.11 times the keys that
// are seen, and a block of 14.5 tiles on average waits for its first one; fp32, 6 documents, window 257 + 256, 170 to 176 us (45 and 46 %).
// ------------------------------------------------------------------------------------------------------------
constexpr uint32_t WIDE_ROWS = 128;

template <typename C>
struct Wide {
    static constexpr int TILE = C::NK == 1 ? 64 : 32;
    typedef Stage<C, TILE, 256> S;
    struct Shared {
        alignas(16) char k[S::BYTES];
        alignas(16) char v[S::BYTES];
        uint32_t bad[2];                 // some value of the tile, or of the one before, is not finite
        uint8_t marks[TILE * C::PARTS];  // ... which
    };
};

// Blocks of `size` rows of all sequences are numbered without a sum over their lengths: those of row b of the batch, which begins at token
// `before`, start at number before * group / size + b, which leaves each row as many as it can need.
__device__ __forceinline__ uint32_t first_slot(const AttnArgs& a, uint32_t b, uint32_t before, uint32_t size)
{
    return (uint32_t)((uint64_t)before * a.group / size) + b;
}
// the row of the batch that has block `slot`, if any has
__device__ __forceinline__ uint32_t row_of_slot(const AttnArgs& a, uint32_t slot, uint32_t size)
{
    uint32_t lo = 0, up = a.batch;
    while (up - lo > 1) {
        const uint32_t mid = (lo + up) / 2;
        if (first_slot(a, mid, clamped_start(a.starts, mid, a.tokens), size) <= slot) lo = mid;
        else up = mid;
    }
    return lo;
}

template <typename C>
__device__ __forceinline__ void wide_rows(const AttnArgs& a, uint32_t block, uint32_t slots, uint32_t splits, uint32_t narrow_rows, const Partial& part, char* shared)
{
    typedef Wide<C> W;
    constexpr int TILE = W::TILE, KT = TILE / 32;
    typename W::Shared& sh = *reinterpret_cast<typename W::Shared*>(shared);
    char *const lk = sh.k, *const lv = sh.v;
    uint32_t* const bad = sh.bad;
    uint8_t* const marks = sh.marks;
    const uint32_t kh = block % a.kv_heads, rest = block / a.kv_heads, split = rest % splits, slot = slots - 1 - rest / splits;  // late rows, which see most keys, first
    const uint32_t b = __builtin_amdgcn_readfirstlane(row_of_slot(a, slot, WIDE_ROWS));
    const Row r = load_row(a.starts, a.seqs, a.tables, a.lengths, a.tokens, a.seq_count, a.table_width, a.page_shift, C::PAGED, b);
    const uint32_t rows = r.n * a.group, before = first_slot(a, b, r.first, WIDE_ROWS), row0 = (slot - before) * WIDE_ROWS;
    if (slot < before || row0 >= rows || rows <= narrow_rows) return;
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = tid & 31, h = tid >> 5 & 1;
    const uint32_t end = row0 + WIDE_ROWS < rows ? row0 + WIDE_ROWS : rows, mine = row0 + 32 * wave;
    const Span span = span_of(a, r, row0, end - 1, TILE);
    const int32_t per = (span.total + (int32_t)splits - 1) / (int32_t)splits, from = per * (int32_t)split;
    const int32_t to = from + per < span.total ? from + per : span.total;
    const bool works = mine < end;
    Rows<C, 32> w;
    w.begin(a, r, kh, works ? mine : row0, rows);
    // whether every row of the workgroup sees all of a tile
    const int32_t all_hi = [&] {
        const int64_t e = (int64_t)r.pos0 + row0 / a.group + a.right + 1;
        return (int32_t)(e < 0 ? 0 : e < r.length ? e : r.length);
    }();
    const int64_t all_lo = (int64_t)r.pos0 + (end - 1) / a.group - a.left;

    if (tid < 2) bad[tid] = 0;
    if (from < to) {
        typename W::S sk, sv;
        sv.no_marks(marks, tid);
        Ahead<C, TILE> ahead;
        ahead.ask(a, r, span.at(from) * TILE);
        const Place p = place<C, TILE>(a, r, kh, span.at(from) * TILE, ahead);
        sk.fetch(a.k, a, r, p, span.at(from) * TILE, wave, tid);
        sv.fetch(a.v, a, r, p, span.at(from) * TILE, wave, tid);
        uint32_t coming = p.there;
        ahead.ask(a, r, span.at(from + 1) * TILE);
        for (int32_t t = from; t < to; ++t) {
            const int32_t key0 = span.at(t) * TILE;
            const bool mixed = !(key0 + TILE <= all_hi && (key0 >= all_lo || key0 + TILE <= w.sinks)) || coming != ~0u;
            __syncthreads();  // everybody is done with the tile before
            if (tid == 0) bad[(t + 1) & 1] = 0;
            sk.store(lk, tid);
            if (mixed && sv.clear(marks, tid)) bad[t & 1] = 1;
            sv.store(lv, tid);
            const uint32_t there = coming;
            if (t + 1 < to) {
                const Place p = place<C, TILE>(a, r, kh, span.at(t + 1) * TILE, ahead);
                sk.fetch(a.k, a, r, p, span.at(t + 1) * TILE, wave, tid);
                sv.fetch(a.v, a, r, p, span.at(t + 1) * TILE, wave, tid);
                coming = p.there;
                ahead.ask(a, r, span.at(t + 2) * TILE);
            }
            __syncthreads();
            if (!works || !w.some(key0, TILE)) continue;
            float s[16 * KT];
#pragma unroll
            for (int n = 0; n < KT; ++n) w.template scores<W::S::PIECE>(lk + n * 32 * C::LB, s + 16 * n);
            if (!w.all(key0, TILE) || there != ~0u) {
#pragma unroll
                for (int n = 0; n < KT; ++n) w.hide(s + 16 * n, key0 + 32 * n, there >> 2 * n);
            }
            w.template softmax<16 * KT>(s);
#pragma unroll
            for (int n = 0; n < KT; ++n) w.template values<W::S::PIECE>(lv + n * 32 * C::LB, s + 16 * n);
            if (mixed && bad[t & 1]) w.poison(marks, key0, TILE, there);
        }
    }
    if (mine + j >= end || !works) return;
    const float l = row_sum<32>(w.l);
    const uint32_t row = mine + j, token = r.first + row / a.group, head = kh * a.group + row % a.group;
    if (splits == 1) {
        typename C::TQ* out = static_cast<typename C::TQ*>(a.out) + (size_t)token * a.out_stride + (size_t)head * C::HD;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < w.DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (32 * d + 8 * i < C::HD) store4(out + 32 * d + 8 * i + 4 * h, w.quad(d, i) * inv);
    } else {
        const uint64_t to_row = (uint64_t)token * a.heads + head, at = split * part.rows + to_row;
        if (h == 0) part.put(split, to_row, w.m, l, w.c);
        if (from >= to) return;  // (the joining kernel does not look at sums whose l is 0)
#pragma unroll
        for (int d = 0; d < w.DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (32 * d + 8 * i < C::HD) store4(part.o + at * C::HD + 32 * d + 8 * i + 4 * h, w.quad(d, i));
    }
}

// ------------------------------------------------------------------------------------------------------------
// Few rows (a single new token, mostly): a workgroup takes 16 rows of a sequence and key head at a time; its waves take the tiles of 32 keys in
// turn, each through LDS of its own, without barriers, and are joined at the end.  16 rows, since up to 16 query heads share a key head: 32 would double the products
// for nothing.  Bound by HBM where there are keys enough: 64 sequences of up to 8191, 32 heads over 8, bf16, 199 us, 5.5 TB/s; two of 100 000, fp16, 37 us, 6.2 TB/s.
// ------------------------------------------------------------------------------------------------------------
constexpr uint32_t NARROW_ROWS = 16;

template <typename C, int WAVES>
struct Narrow {
    typedef Stage<C, 32, 64> S;
    static constexpr int PITCH = C::HD + 1, JOIN = 16 * PITCH * 4;  // a wave's sums, rows padded against bank conflicts
    static constexpr int WAVE = ((S::BYTES > JOIN ? S::BYTES : JOIN) + 15) / 16 * 16;
    struct Shared {
        alignas(16) char lds[WAVES * WAVE];
        float ml[WAVES][16][2];  // m, and l relative to the waves' largest m
        float c[16];
        uint8_t marks[WAVES][32 * C::PARTS];
    };
};

__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// by_slot: a workgroup per block of 16 rows (first_slot); otherwise one per row of the batch, which takes its blocks one after the other
template <typename C, int WAVES>
__device__ __forceinline__ void narrow_rows_of(const AttnArgs& a, uint32_t number, uint32_t by_slot, uint32_t splits, uint32_t most_rows, const Partial& part, char* shared)
{
    typedef Narrow<C, WAVES> W;
    typename W::Shared& sh = *reinterpret_cast<typename W::Shared*>(shared);
    char* const lds = sh.lds;
    auto& ml = sh.ml;
    auto& marks = sh.marks;
    const uint32_t split = number % splits, rest = number / splits, kh = rest % a.kv_heads, slot = rest / a.kv_heads;
    const uint32_t b = by_slot ? __builtin_amdgcn_readfirstlane(row_of_slot(a, slot, NARROW_ROWS)) : slot;
    const Row r = load_row(a.starts, a.seqs, a.tables, a.lengths, a.tokens, a.seq_count, a.table_width, a.page_shift, C::PAGED, b);
    const uint32_t rows = r.n * a.group;
    if (rows > most_rows) return;
    uint32_t block = 0, blocks = (rows + NARROW_ROWS - 1) / NARROW_ROWS;
    if (by_slot) {
        const uint32_t before = first_slot(a, b, r.first, NARROW_ROWS);
        if (slot < before || slot - before >= blocks) return;
        block = slot - before;
        blocks = block + 1;
    }
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15;
    char* const mine = lds + wave * W::WAVE;
    for (; block < blocks; ++block) {
        const uint32_t row0 = block * NARROW_ROWS, end = row0 + NARROW_ROWS < rows ? row0 + NARROW_ROWS : rows;
        const Span span = span_of(a, r, row0, end - 1, 32);
        int32_t per = (span.total + (int32_t)splits - 1) / (int32_t)splits;
        if (per < WAVES) per = WAVES;  // a tile for each wave
        const int32_t from = per * (int32_t)split, to = from + per < span.total ? from + per : span.total;
        if (splits > 1 && from >= to) {  // nothing left for this split
            if (tid < end - row0) {
                const uint32_t row = row0 + tid;
                part.put(split, (uint64_t)(r.first + row / a.group) * a.heads + kh * a.group + row % a.group, -INF, 0.0f, 1.0f);
            }
            continue;
        }
        int32_t t = from + (int32_t)wave;
        typename W::S sk, sv;
        sv.no_marks(marks[wave], lane);
        Place now;
        Ahead<C, 32> ahead;
        if (t < to) {  // (before the rows' q: the first keys take longest)
            ahead.ask(a, r, span.at(t) * 32);
            now = place<C, 32>(a, r, kh, span.at(t) * 32, ahead);
            sk.fetch(a.k, a, r, now, span.at(t) * 32, 0, lane);
            sv.fetch(a.v, a, r, now, span.at(t) * 32, 0, lane);
            ahead.ask(a, r, span.at(t + WAVES) * 32);
        }
        Rows<C, 16> w;
        w.begin(a, r, kh, row0, rows);
        for (; t < to; t += WAVES) {
            const int32_t key0 = span.at(t) * 32;
            const uint32_t there = now.there;
            const bool mixed = !w.all(key0, 32) || there != ~0u, more = t + WAVES < to;
            sk.store(mine, lane);
            if (more) {
                now = place<C, 32>(a, r, kh, span.at(t + WAVES) * 32, ahead);
                sk.fetch(a.k, a, r, now, span.at(t + WAVES) * 32, 0, lane);
            }
            wave_sync();
            float s[8];
            w.template scores<W::S::PIECE>(mine, s);
            wave_sync();
            if (mixed) w.hide(s, key0, there);
            bool bad = false;
            if (mixed) bad = __any(sv.clear(marks[wave], lane));
            sv.store(mine, lane);
            if (more) {
                sv.fetch(a.v, a, r, now, span.at(t + WAVES) * 32, 0, lane);
                ahead.ask(a, r, span.at(t + 2 * WAVES) * 32);
            }
            w.template softmax<8>(s);
            wave_sync();
            w.template values<W::S::PIECE>(mine, s);
            if (bad) w.poison(marks[wave], key0, 32, there);
            wave_sync();
        }
        // join the waves: all relative to the largest maximum
        const float l = row_sum<16>(w.l);
        if (lane < 16) ml[wave][j][0] = w.m;
        __syncthreads();
        float top = -INF;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top = fmaxf(top, ml[i][j][0]);
        const float f = __builtin_amdgcn_exp2f((w.m - (top == -INF ? 0.0f : top)) * w.c);
        if (lane < 16) ml[wave][j][1] = l * f;
        if (tid < 16) sh.c[j] = w.c;
        float* const sums = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int d = 0; d < w.DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[j * W::PITCH + 16 * d + w.place_of(i)] = w.o[d][i] * f;
        __syncthreads();
        // HD consecutive columns of a row by consecutive threads
        for (uint32_t x = tid; x < (end - row0) * (C::HD / 4); x += WAVES * 64) {
            const uint32_t row = x / (C::HD / 4), col = x % (C::HD / 4) * 4;
            f32x4 y = {0.f, 0.f, 0.f, 0.f};
            float mx = -INF, sum = 0.0f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                const float* from_wave = reinterpret_cast<const float*>(lds + i * W::WAVE) + row * W::PITCH + col;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] += from_wave[e];
                mx = fmaxf(mx, ml[i][row][0]);
                sum += ml[i][row][1];
            }
            const uint32_t token = r.first + (row0 + row) / a.group, head = kh * a.group + (row0 + row) % a.group;
            if (splits == 1) {
                store4(static_cast<typename C::TQ*>(a.out) + (size_t)token * a.out_stride + (size_t)head * C::HD + col, sum == 0.0f ? (f32x4){0.f, 0.f, 0.f, 0.f} : y * (1.0f / sum));
            } else {
                const uint64_t to_row = (uint64_t)token * a.heads + head;
                if (col == 0) part.put(split, to_row, mx, sum, sh.c[row]);
                store4(part.o + (split * part.rows + to_row) * C::HD + col, y);
            }
        }
        __syncthreads();
    }
}

// What one call launches, decided by launch_attention.
struct Plan {
    bool wide, narrow;
    uint32_t slots;                       // blocks of 128 rows
    uint32_t wide_splits, narrow_splits;
    uint32_t narrow_rows;                 // rows of a sequence and key head up to which they are taken 16 at a time
    bool by_slot;                         // ... in workgroups of 16 rows each
    Partial part;
};

// Waves of a workgroup that takes 16 rows, alone in its launch: eight, where their LDS fits.  us with four / eight: one sequence of 777 keys, 12 heads, fp32 over
// fp16, 9.7 / 8.1; one text of 128 tokens 6.6 / 6.7, two sequences of 100 000 keys 49.0 / 48.4, 64 of up to 8191 197 / 198.
template <typename C>
constexpr int NARROW_WAVES = C::NK == 3 && C::HD > 64 ? 4 : 8;

template <typename C>
__global__ __launch_bounds__(NARROW_WAVES<C> * 64, C::NK == 1 && C::HD <= 64 ? 4 : NARROW_WAVES<C> / 4) void attention_narrow_kernel(AttnArgs a, uint32_t by_slot, uint32_t splits, uint32_t most_rows,
                                                                                                     Partial part)
{
    __shared__ __attribute__((aligned(1024))) char shared[sizeof(typename Narrow<C, NARROW_WAVES<C>>::Shared)];
    narrow_rows_of<C, NARROW_WAVES<C>>(a, blockIdx.x, by_slot, splits, most_rows, part, shared);
}

// Blocks of 128 rows, and behind them, for those sequences of the batch that have few, blocks of 16: these wait for memory most of the time, those for
// the matrix cores, so they share the device better than one launch after the other (16 sequences, half of them with one token: 245 us in two
// launches, 214 in one, shares being in one piece then).
template <typename C>
__global__ __launch_bounds__(256, (C::NK == 3 && C::HD > 80) || (C::NQ > 1 && C::HD > 96) ? 1 : 2) void attention_wide_kernel(AttnArgs a, uint32_t wide_blocks, uint32_t slots, uint32_t splits,
                                                                                                         uint32_t narrow_splits, uint32_t narrow_rows, Partial part)
{
    constexpr size_t WIDE = sizeof(typename Wide<C>::Shared), NARROW = C::PAGED ? sizeof(typename Narrow<C, 4>::Shared) : 0;
    __shared__ __attribute__((aligned(1024))) char shared[WIDE > NARROW ? WIDE : NARROW];
    if (!C::PAGED || blockIdx.x < wide_blocks) {
        wide_rows<C>(a, blockIdx.x, slots, splits, narrow_rows, part, shared);
    } else {
        if constexpr (C::PAGED) narrow_rows_of<C, 4>(a, blockIdx.x - wide_blocks, 0, narrow_splits, narrow_rows, part, shared);
    }
}

template <typename C>
int launch(Ctx* ctx, const AttnArgs& a, const Plan& p)
{
    if (p.wide) {
        const uint32_t wide = p.slots * a.kv_heads * p.wide_splits, narrow = p.narrow ? a.batch * a.kv_heads * p.narrow_splits : 0;
        hipLaunchKernelGGL((attention_wide_kernel<C>), dim3(wide + narrow), dim3(256), 0, ctx->stream, a, wide, p.slots, p.wide_splits, p.narrow_splits,
                           p.narrow ? p.narrow_rows : 0, p.part);
        return hip_check(ctx, hipGetLastError(), "attention_wide_kernel launch");
    }
    const uint32_t slots = p.by_slot ? (uint32_t)((uint64_t)a.tokens * a.group / NARROW_ROWS) + a.batch : a.batch;
    hipLaunchKernelGGL((attention_narrow_kernel<C>), dim3(slots * a.kv_heads * p.narrow_splits), dim3(NARROW_WAVES<C> * 64), 0, ctx->stream, a,
                       (uint32_t)p.by_slot, p.narrow_splits, p.narrow_rows, p.part);
    return hip_check(ctx, hipGetLastError(), "attention_narrow_kernel launch");
}

template <typename TQ, typename TK, bool PAGED>
int launch_heads(Ctx* ctx, const AttnArgs& a, const Plan& p)
{
    switch (a.head_dim) {
    case 32: return launch<Config<TQ, TK, 32, PAGED>>(ctx, a, p);
    case 64: return launch<Config<TQ, TK, 64, PAGED>>(ctx, a, p);
    case 80: return launch<Config<TQ, TK, 80, PAGED>>(ctx, a, p);
    case 96: return launch<Config<TQ, TK, 96, PAGED>>(ctx, a, p);
    default: return launch<Config<TQ, TK, 128, PAGED>>(ctx, a, p);
    }
}

// a translation unit each
int launch_f32(Ctx* ctx, const AttnArgs& a, const Plan& p);
int launch_f32_f16(Ctx* ctx, const AttnArgs& a, const Plan& p);
int launch_f32_bf16(Ctx* ctx, const AttnArgs& a, const Plan& p);
int launch_f16(Ctx* ctx, const AttnArgs& a, const Plan& p);
int launch_bf16(Ctx* ctx, const AttnArgs& a, const Plan& p);

}  // namespace attn
}  // namespace pimdl
