// Tree attention at head_dim 16.
#include "wn_tree_kernels.h"

namespace wn {
TreeKernels tree_kernels_16(bool exact) { return exact ? tree_kernels<16, true>() : tree_kernels<16, false>(); }
}  // namespace wn
