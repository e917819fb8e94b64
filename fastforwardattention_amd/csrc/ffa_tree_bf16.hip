// Attention of a group of new tokens, bf16 (templates in ffa_tree_kernels.h).
#include "ffa_tree_kernels.h"

namespace ffa {

int launch_tree_bf16(const TreeParams& P, int head_dim, const TreePlan& plan, void* stream) {
    return launch_tree_type<bf16_t>(P, head_dim, plan, stream);
}

}  // namespace ffa
