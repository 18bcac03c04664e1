// Windowed attention at head_dim 16.
#include "wn_tree_kernels.h"

namespace wn {
WindowKernels window_kernels_16(bool exact, int bw_k, int bw_v) { return tree_kernels_for<16, true>(exact, bw_k, bw_v); }
}  // namespace wn
