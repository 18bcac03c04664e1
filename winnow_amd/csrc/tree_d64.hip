// Tree attention at head_dim 64.
#include "wn_tree_kernels.h"

namespace wn {
TreeKernels tree_kernels_64(bool exact) { return exact ? tree_kernels<64, true>() : tree_kernels<64, false>(); }
}  // namespace wn
