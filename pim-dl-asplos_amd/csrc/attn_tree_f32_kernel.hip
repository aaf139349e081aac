// Attention of trees of drafted tokens on the matrix cores: fp32.
#include "attn_body.h"

int pimdl::attn::launch_tree_f32(Ctx* ctx, const AttnArgs& a, const Plan& p) { return launch_heads<float, float, true, true>(ctx, a, p); }
