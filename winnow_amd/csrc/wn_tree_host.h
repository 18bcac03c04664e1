// What the host sides of the tree attention (tree.hip) and the windowed attention (window.hip) share.
#pragma once

#include <algorithm>
#include <map>
#include <mutex>
#include <utility>

#include "wn_tree.h"

namespace wn {

// Query rows per kv head, padded to whole work-groups.
template <class Args>
int tree_nrp(const TreeScanOf<Args>& s, int64_t rows) { return int((rows + s.rows - 1) / s.rows * s.rows); }

inline int64_t align256(int64_t x) { return (x + 255) & ~int64_t(255); }

struct TreeLayout {
  int64_t qh, ql, qs, vis, acc, ml, total;
};

inline TreeLayout tree_layout(int B, int Hkv, int nrp, int T, int D, int num_splits) {
  TreeLayout l;
  const int64_t rows = int64_t(B) * Hkv * nrp;
  l.qh = 0;
  l.ql = l.qh + align256(rows * D * 2);
  l.qs = l.ql + align256(rows * D * 2);
  l.vis = l.qs + align256(rows * 4);
  l.acc = l.vis + align256(int64_t(B) * T * 8);
  l.ml = l.acc + align256(rows * num_splits * D * 4);
  l.total = l.ml + align256(rows * num_splits * 2 * 4);
  return l;
}

// Resident work-groups of a scan on the current device (0: the query failed), asked for
// once per device, kernel and LDS size; the kernel is allowed that much LDS.
template <class Args>
int tree_slots(const TreeScanOf<Args>& s, int lds) {
  static std::mutex mu;
  static std::map<std::pair<std::pair<int, void (*)(Args)>, int>, int> cache;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find({{dev, s.fn}, lds});
  if (it != cache.end()) return it->second;
  int per_cu = 0;
  const void* f = reinterpret_cast<const void*>(s.fn);
  if ((lds && hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) ||
      hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, f, s.threads, lds) != hipSuccess)
    return 0;
  const int n = per_cu * device_cus();
  cache[{{dev, s.fn}, lds}] = n;
  return n;
}

template <class Args>
int tree_lds(const TreeScanOf<Args>& s, int bw_k, int bw_v) {
  if (s.waves) return 0;  // static
  return std::max(s.give, s.lds + (s.tables ? s.tables : tree_table_bytes(bw_k) + tree_table_bytes(bw_v)));
}

}  // namespace wn
