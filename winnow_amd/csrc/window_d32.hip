// Windowed attention at head_dim 32.
#include "wn_window_rows.h"

namespace wn {
WindowKernels window_kernels_32(bool exact, int bw_k, int bw_v) { return window_kernels_for<32>(exact, bw_k, bw_v); }
}  // namespace wn
