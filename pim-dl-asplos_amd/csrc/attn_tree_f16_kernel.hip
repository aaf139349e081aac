// Attention of trees of drafted tokens on the matrix cores: halves.
#include "attn_body.h"

int pimdl::attn::launch_tree_f16(Ctx* ctx, const AttnArgs& a, const Plan& p) { return launch_heads<_Float16, _Float16, true, true>(ctx, a, p); }
