// Tree attention at head_dim 256.
#include "wn_tree_kernels.h"

namespace wn {
TreeKernels tree_kernels_256(bool exact, int bw_k, int bw_v) { return tree_kernels_for<256>(exact, bw_k, bw_v); }
}  // namespace wn
