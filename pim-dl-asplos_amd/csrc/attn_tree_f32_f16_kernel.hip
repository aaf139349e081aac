// Attention of trees of drafted tokens on the matrix cores: fp32 over a cache in halves.
#include "attn_body.h"

int pimdl::attn::launch_tree_f32_f16(Ctx* ctx, const AttnArgs& a, const Plan& p) { return launch_heads<float, _Float16, true, true>(ctx, a, p); }
