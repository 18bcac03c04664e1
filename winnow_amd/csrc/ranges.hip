// Range checks of the small metadata that a host mirror holds, before a launch that reads pages by
// it. Host code only: the same comparisons in numpy take 8 to 12 us a call, here under 2 with the
// call itself.
#include <cstdint>

#include "wn_common.h"

extern "C" int wn_positions_in_range(const int32_t* start, int lengths, int n, const int32_t* page_table,
                                     int64_t table_stride_b, int B, int max_pages, int num_pages, int S) {
  if (!start || !page_table || B < 0 || max_pages < 0 || S <= 0 || n < 0) return 0;
  for (int b = 0; b < B; ++b) {
    const int64_t lo = lengths ? 0 : start[b], hi = lengths ? start[b] : int64_t(start[b]) + n;
    if (lo < 0 || hi < 0 || hi > int64_t(max_pages) * S) return 0;
    const int32_t* row = page_table + b * table_stride_b;
    for (int64_t c = lo / S; c * S < hi; ++c)
      if (row[c] < 0 || row[c] >= num_pages) return 0;
  }
  return 1;
}

extern "C" int wn_window_in_range(const int32_t* lens, const int32_t* page_table, int64_t table_stride_b, int B, int max_pages,
                                  int num_pages, int S, int Q, int window, int sinks) {
  if (!lens || !page_table || B < 0 || max_pages < 0 || S <= 0 || Q < 0 || window < 1 || sinks < 0) return 0;
  for (int b = 0; b < B; ++b) {
    const int64_t L = lens[b];
    if (L < 0 || L > int64_t(max_pages) * S) return 0;
    const int64_t lo = L - Q + 1 > window ? L - Q + 1 - window : 0, sink = sinks < L ? sinks : L;
    const int32_t* row = page_table + b * table_stride_b;
    for (int64_t c = 0; c * S < sink; ++c)
      if (row[c] < 0 || row[c] >= num_pages) return 0;
    for (int64_t c = lo / S; c * S < L; ++c)
      if (row[c] < 0 || row[c] >= num_pages) return 0;
  }
  return 1;
}

extern "C" int wn_parents_in_order(const int32_t* parents, int64_t parents_stride_b, int B, int T) {
  if (!parents || B < 0 || T < 0) return 0;
  for (int b = 0; b < B; ++b)
    for (int i = 0; i < T; ++i) {
      const int32_t p = parents[b * parents_stride_b + i];
      if (p < -1 || p >= i) return 0;
    }
  return 1;
}

extern "C" int wn_tree_prepare(const int32_t* lens, const int32_t* page_table, int64_t table_stride_b, int table_pages,
                               const int32_t* parents, int64_t parents_stride_b, int B, int Hq, int Hkv, int T, int D, int S,
                               int bw_k, int bw_v, int exact, int num_pages, int max_pages, int* plan) {
  return plan && wn_positions_in_range(lens, 1, 0, page_table, table_stride_b, B, table_pages, num_pages, S) &&
         wn_parents_in_order(parents, parents_stride_b, B, T) &&
         wn_tree_plan(B, Hq, Hkv, T, D, S, bw_k, bw_v, exact, max_pages, lens, plan, plan + 1, plan + 2) == 0;
}

extern "C" int wn_window_prepare(const int32_t* lens, const int32_t* page_table, int64_t table_stride_b, int table_pages, int B, int Hq,
                                 int Hkv, int Q, int D, int S, int bw_k, int bw_v, int exact, int wide, int num_pages, int max_pages,
                                 int window, int sinks, int* plan) {
  return plan && wn_window_in_range(lens, page_table, table_stride_b, B, table_pages, num_pages, S, Q, window, sinks) &&
         wn_window_plan(B, Hq, Hkv, Q, D, S, bw_k, bw_v, exact, wide, max_pages, window, sinks, lens, plan, plan + 1) == 0;
}
