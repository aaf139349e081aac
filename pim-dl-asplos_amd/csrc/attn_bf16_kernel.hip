// Attention on the matrix cores: bf16.
#include "attn_body.h"

int pimdl::attn::launch_bf16(Ctx* ctx, const AttnArgs& a, const Plan& p)
{
    return a.paged ? launch_heads<__bf16, __bf16, true>(ctx, a, p) : launch_heads<__bf16, __bf16, false>(ctx, a, p);
}
