// Attention on the matrix cores: fp32 over a cache in halves.
#include "attn_body.h"

int pimdl::attn::launch_f32_f16(Ctx* ctx, const AttnArgs& a, const Plan& p)
{
    return launch_heads<float, _Float16, true>(ctx, a, p);  // (a window's tensors have one type)
}
