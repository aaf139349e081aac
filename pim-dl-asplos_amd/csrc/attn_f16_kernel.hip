// Attention on the matrix cores: halves.
#include "attn_body.h"

int pimdl::attn::launch_f16(Ctx* ctx, const AttnArgs& a, const Plan& p)
{
    return a.paged ? launch_heads<_Float16, _Float16, true>(ctx, a, p) : launch_heads<_Float16, _Float16, false>(ctx, a, p);
}
