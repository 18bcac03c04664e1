// Windowed attention at head_dim 128.
#include "wn_window_rows.h"

namespace wn {
WindowKernels window_kernels_128(bool exact, int bw_k, int bw_v) { return window_kernels_for<128>(exact, bw_k, bw_v); }
}  // namespace wn
