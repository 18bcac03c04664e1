// Windowed attention at head_dim 256.
#include "wn_window_rows.h"

namespace wn {
WindowKernels window_kernels_256(bool exact, int bw_k, int bw_v) { return window_kernels_for<256>(exact, bw_k, bw_v); }
}  // namespace wn
