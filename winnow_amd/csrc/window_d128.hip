// Windowed attention at head_dim 128.
#include "wn_tree_kernels.h"

namespace wn {
WindowKernels window_kernels_128(bool exact, int bw_k, int bw_v) { return tree_kernels_for<128, true>(exact, bw_k, bw_v); }
}  // namespace wn
