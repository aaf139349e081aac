// Attention of a ragged batch over a window or a paged cache for gfx950 (MI355X): see pimdl_attention_window and
// pimdl_attention_paged.
#include "serve_common.h"

namespace pimdl {

namespace {

constexpr float LOG2E = 1.4426950408889634f;

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
// Any head size up to 256, any stride and alignment: a wave takes one query of one head, a lane a key at a time for the scores and up to
// four columns of the output, with the running maximum m and sum l of a streaming softmax in between: a block of 64 keys
// with maximum m' gives o = o 2^(m - m') + sum p v, l = l 2^(m - m') + sum p, p = 2^(s - m').
// ---------------------------------------------------------------------------------------------
template <typename TQ, typename TK, bool PAGED>
__global__ __launch_bounds__(256) void attention_plain_kernel(AttnArgs a)
{
    __shared__ float qs[4][256];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t item = (uint64_t)blockIdx.x * 4 + wave;
    const uint32_t t = (uint32_t)(item / a.heads), h = (uint32_t)(item % a.heads);
    if (t >= a.tokens) return;
    const uint32_t b = row_of_token(a.starts, a.batch, a.tokens, t);
    const Row r = load_row(a.starts, a.seqs, a.tables, a.lengths, a.tokens, a.seq_count, a.table_width, a.page_shift, PAGED, b);
    if (t < r.first || t - r.first >= r.n) return;  // a row of no sequence
    const uint32_t hd = a.head_dim, kh = h / a.group;
    const TQ* q = static_cast<const TQ*>(a.q) + (size_t)t * a.q_stride + (size_t)h * hd;
    for (uint32_t d = lane; d < hd; d += 64) qs[wave][d] = to_float(q[d]);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();

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
    float m = -__builtin_inff(), l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
    auto keys = [&](int32_t from, int32_t to) {
        for (int32_t j0 = from; j0 < to; j0 += 64) {
            const int32_t j = j0 + (int32_t)lane;
            float s = -__builtin_inff();
            int64_t at = -1;
            if (j < to && (at = row_at(j)) >= 0) {
                float dot = 0.0f;
                for (uint32_t d = 0; d < hd; ++d) dot = fmaf(qs[wave][d], to_float(k[at + d]), dot);
                s = dot * a.scale * LOG2E;
            }
            const float mx = fmaxf(m, wave_max(s));
            const float base = mx == -__builtin_inff() ? 0.0f : mx;  // (nothing yet but scores of -infinity)
            const float p = exp2f(s - base), alpha = exp2f(m - base);
            m = mx;
            l = l * alpha + wave_sum(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] *= alpha;
            const int32_t count = to - j0 < 64 ? to - j0 : 64;
            for (int32_t jj = 0; jj < count; ++jj) {
                const float pj = __shfl(p, jj);
                const int64_t row = ((int64_t)__shfl((int)(at >> 32), jj) << 32) | (uint32_t)__shfl((int)at, jj);
                if (row < 0) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (lane + 64 * i < hd) o[i] = fmaf(pj, to_float(v[row + lane + 64 * i]), o[i]);
            }
        }
    };
    keys(0, sinks);
    keys(lo, hi);
    TQ* out = static_cast<TQ*>(a.out) + (size_t)t * a.out_stride + (size_t)h * hd;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < hd) out[lane + 64 * i] = (TQ)(l == 0.0f ? 0.0f : o[i] * inv);
}

template <typename TQ, typename TK>
int launch_plain(Ctx* ctx, const AttnArgs& a)
{
    const uint32_t grid = (uint32_t)(((uint64_t)a.tokens * a.heads + 3) / 4);
    if (a.paged) hipLaunchKernelGGL((attention_plain_kernel<TQ, TK, true>), dim3(grid), dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((attention_plain_kernel<TQ, TK, false>), dim3(grid), dim3(256), 0, ctx->stream, a);
    return hip_check(ctx, hipGetLastError(), "attention_plain_kernel launch");
}

}  // namespace

int launch_attention(Ctx* ctx, const AttnArgs& a)
{
    if (a.tokens == 0 || a.batch == 0) return PIMDL_OK;
    if (a.dtype == PIMDL_BF16) return launch_plain<__bf16, __bf16>(ctx, a);
    if (a.dtype == PIMDL_F16) return launch_plain<_Float16, _Float16>(ctx, a);
    if (a.cache_dtype == PIMDL_BF16) return launch_plain<float, __bf16>(ctx, a);
    if (a.cache_dtype == PIMDL_F16) return launch_plain<float, _Float16>(ctx, a);
    return launch_plain<float, float>(ctx, a);
}

}  // namespace pimdl
