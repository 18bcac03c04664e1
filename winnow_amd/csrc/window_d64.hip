// Windowed attention at head_dim 64.
#include "wn_window_rows.h"

namespace wn {
WindowKernels window_kernels_64(bool exact, int bw_k, int bw_v) { return window_kernels_for<64>(exact, bw_k, bw_v); }
}  // namespace wn
