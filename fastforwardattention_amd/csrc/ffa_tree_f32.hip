// Attention of a group of new tokens, fp32 (templates in ffa_tree_kernels.h).
#include "ffa_tree_kernels.h"

namespace ffa {

int launch_tree_f32(const TreeParams& P, int head_dim, int row_tiles, void* stream) {
    return launch_tree_type<float>(P, head_dim, row_tiles, stream);
}

}  // namespace ffa
