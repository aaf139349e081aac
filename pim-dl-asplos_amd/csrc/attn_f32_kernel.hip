// Attention on the matrix cores: fp32.
#include "attn_body.h"

int pimdl::attn::launch_f32(Ctx* ctx, const AttnArgs& a, const Plan& p)
{
    return a.paged ? launch_heads<float, float, true>(ctx, a, p) : launch_heads<float, float, false>(ctx, a, p);
}
