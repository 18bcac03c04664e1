// Tree attention at head_dim 128.
#include "wn_tree_kernels.h"

namespace wn {
TreeKernels tree_kernels_128(bool exact) { return exact ? tree_kernels<128, true>() : tree_kernels<128, false>(); }
}  // namespace wn
