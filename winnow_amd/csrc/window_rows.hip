// The row scans (wn_decode_rows.h) of the windowed attention's single-token step.
#include "wn_decode_rows.h"

namespace wn {

SplitKernel pick_window_rows(int bw_k, int bw_v, int n_rep, bool tf32) {
  const int ng = n_rep >= 1 && n_rep <= 4 ? 1 : n_rep >= 5 && n_rep <= 8 ? 2 : 0;
  if (ng == 0) return SplitKernel{};
  SplitKernel k;
  if (tf32) k = ng == 1 ? rows_tf_for<1, true>(bw_k, bw_v) : rows_tf_for<2, true>(bw_k, bw_v);
  if (!k.fn) k = ng == 1 ? rows16_for<1, false, true>(bw_k, bw_v) : rows16_for<2, false, true>(bw_k, bw_v);
  return k;
}

}  // namespace wn
