// Attention of trees of drafted tokens on the matrix cores: bf16.
#include "attn_body.h"

int pimdl::attn::launch_tree_bf16(Ctx* ctx, const AttnArgs& a, const Plan& p) { return launch_heads<__bf16, __bf16, true, true>(ctx, a, p); }
