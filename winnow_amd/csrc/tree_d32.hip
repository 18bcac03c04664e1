// Tree attention at head_dim 32.
#include "wn_tree_kernels.h"

namespace wn {
TreeKernels tree_kernels_32(bool exact) { return exact ? tree_kernels<32, true>() : tree_kernels<32, false>(); }
}  // namespace wn
