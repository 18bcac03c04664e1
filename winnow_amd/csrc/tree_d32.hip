// Tree attention at head_dim 32.
#include "wn_tree_kernels.h"

namespace wn {
TreeKernels tree_kernels_32(bool exact, int bw_k, int bw_v) { return tree_kernels_for<32>(exact, bw_k, bw_v); }
}  // namespace wn
