// Windowed attention at head_dim 32.
#include "wn_tree_kernels.h"

namespace wn {
WindowKernels window_kernels_32(bool exact, int bw_k, int bw_v) { return tree_kernels_for<32, true>(exact, bw_k, bw_v); }
}  // namespace wn
