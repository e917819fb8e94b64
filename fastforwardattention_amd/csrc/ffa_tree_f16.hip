// Attention of a group of new tokens, fp16 (templates in ffa_tree_kernels.h).
#include "ffa_tree_kernels.h"

namespace ffa {

int launch_tree_f16(const TreeParams& P, int head_dim, const TreePlan& plan, void* stream) {
    return launch_tree_type<uint16_t>(P, head_dim, plan, stream);
}

}  // namespace ffa
