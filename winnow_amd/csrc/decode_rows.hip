// The row scans of the packed decode (wn_decode_rows.h).
#include "wn_decode_rows.h"

namespace wn {

SplitKernel pick_split_rows_tf(int bw_k, int bw_v, int n_rep) {
  const int ng = n_rep >= 1 && n_rep <= 4 ? 1 : n_rep >= 5 && n_rep <= 8 ? 2 : 0;
  if (ng == 0) return SplitKernel{};
  return ng == 1 ? rows_tf_for<1>(bw_k, bw_v) : rows_tf_for<2>(bw_k, bw_v);
}

SplitKernel pick_split_pair(int bw_k, int bw_v, int n_rep) {
  if (n_rep < 1 || n_rep > 4) return SplitKernel{};
  return rows16_for<2, true>(bw_k, bw_v);
}

SplitKernel pick_split_rows(int bw_k, int bw_v, int n_rep) {
  const int ng = n_rep <= 4 ? 1 : n_rep <= 8 ? 2 : 0;
  if (ng == 0) return SplitKernel{};
  return ng == 1 ? rows16_for<1>(bw_k, bw_v) : rows16_for<2>(bw_k, bw_v);
}

}  // namespace wn
