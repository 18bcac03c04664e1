// Tree attention at head_dim 256.
#include "wn_tree_kernels.h"

namespace wn {
TreeKernels tree_kernels_256(bool exact) { return exact ? tree_kernels<256, true>() : tree_kernels<256, false>(); }
}  // namespace wn
