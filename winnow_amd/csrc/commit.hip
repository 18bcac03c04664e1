// Keeping the accepted branch of a drafted tree in a paged cache.
//
// The rows of drafted node path[b, i] (position start[b] + path[b, i]) move to position
// start[b] + i for i < counts[b], K and V, codes and norms, in every layer and kv head, and
// lengths[b] = start[b] + counts[b]. Rows only change place: no arithmetic.
//
// Bound: latency. A step moves some hundred bytes per (layer, sequence, head, side), each
// behind the lookups of its positions and pages; one wave per such group keeps them all in
// flight at once (a full batch: 8,192 waves). A row may be the target of one move and the
// source of another, so a wave reads every source of a block of columns before it writes;
// blocks of columns are independent of each other.
#include <algorithm>

#include "wn_common.h"

namespace wn {
namespace {

constexpr int kUnits = 4;  // pieces of a row that a lane holds

struct CommitSide {
  uint8_t* pages;
  uint16_t* norms;             // null: an unquantized cache
  int64_t sl, sp, sh;          // layer, page and head strides, bytes
  int64_t nl, np, nh;          // of the norms, elements
  int row;                     // bytes of a row
  int unit;                    // bytes moved at a time: 16, 8, 4, 2 or 1
};

struct CommitArgs {
  CommitSide side[2];
  const int32_t* table;
  int64_t tsb;
  const int32_t* start;
  const int32_t* path;
  int64_t psb;
  const int32_t* counts;
  int32_t* lengths;
  int B, Hkv, A, nodes, log2S, num_pages, max_pages;
};

// The page and slot of a position; false where the table or the pool has none.
__device__ __forceinline__ bool commit_row(const CommitArgs& a, const int32_t* trow, int64_t pos, int64_t* page, int* slot) {
  const int64_t col = pos >> a.log2S;
  if (pos < 0 || col >= a.max_pages) return false;
  const int32_t pid = trow[col];
  *page = pid;
  *slot = int(pos & ((1 << a.log2S) - 1));
  return pid >= 0 && pid < a.num_pages;
}

template <class T>
__device__ __forceinline__ void commit_rows(const CommitArgs& a, const CommitSide& s, uint8_t* base, const int64_t* src,
                                            const int64_t* dst, int n, int lane) {
  const int cols = s.row / int(sizeof(T)), most = 64 * kUnits / n;  // columns of a block
  for (int c0 = 0; c0 < cols; c0 += most) {
    const int w = min(most, cols - c0), total = n * w;
    T v[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int u = lane + 64 * k;
      if (u < total && src[u / w] >= 0) v[k] = *reinterpret_cast<const T*>(base + src[u / w] + int64_t(c0 + u % w) * sizeof(T));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // read before written, over all lanes of the wave
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int u = lane + 64 * k;
      if (u < total && src[u / w] >= 0) *reinterpret_cast<T*>(base + dst[u / w] + int64_t(c0 + u % w) * sizeof(T)) = v[k];
    }
  }
}

__global__ __launch_bounds__(64) void commit_kernel(CommitArgs a) {
  __shared__ int64_t src[64], dst[64];  // byte offsets of a layer's head; -1: nothing to move
  const int lane = threadIdx.x;
  const int b = blockIdx.x / a.Hkv, kvh = blockIdx.x % a.Hkv, layer = blockIdx.y;
  const CommitSide& s = a.side[blockIdx.z];
  const int n = min(max(a.counts[b], 0), a.A);
  if (blockIdx.z == 0 && layer == 0 && kvh == 0 && lane == 0) a.lengths[b] = a.start[b] + n;
  if (n == 0) return;  // the whole work-group
  uint16_t norm = 0;
  uint16_t* norm_to = nullptr;
  src[lane] = -1;
  if (lane < n) {
    const int32_t* trow = a.table + b * a.tsb;
    const int node = a.path[b * a.psb + lane];
    const int64_t pos = a.start[b];
    int64_t sp, dp;
    int ss, ds;
    if (node >= 0 && node < a.nodes && node != lane && commit_row(a, trow, pos + node, &sp, &ss) &&
        commit_row(a, trow, pos + lane, &dp, &ds)) {
      src[lane] = sp * s.sp + int64_t(ss) * s.row;
      dst[lane] = dp * s.sp + int64_t(ds) * s.row;
      if (s.norms) {
        uint16_t* base = s.norms + layer * s.nl + kvh * s.nh;
        norm = base[sp * s.np + ss];
        norm_to = base + dp * s.np + ds;
      }
    }
  }
  __syncthreads();
  asm volatile("s_waitcnt vmcnt(0)" : "+v"(norm)::"memory");  // every norm is read
  if (norm_to) *norm_to = norm;
  uint8_t* base = s.pages + layer * s.sl + kvh * s.sh;
  switch (s.unit) {
    case 16: commit_rows<uint4>(a, s, base, src, dst, n, lane); break;
    case 8: commit_rows<uint2>(a, s, base, src, dst, n, lane); break;
    case 4: commit_rows<uint32_t>(a, s, base, src, dst, n, lane); break;
    case 2: commit_rows<uint16_t>(a, s, base, src, dst, n, lane); break;
    default: commit_rows<uint8_t>(a, s, base, src, dst, n, lane);
  }
}

}  // namespace
}  // namespace wn

extern "C" int wn_commit_kv(
    uint8_t* k_pages, int64_t k_stride_l, int64_t k_stride_p, int64_t k_stride_h, int k_row,
    uint8_t* v_pages, int64_t v_stride_l, int64_t v_stride_p, int64_t v_stride_h, int v_row,
    uint16_t* k_norms, int64_t kn_stride_l, int64_t kn_stride_p, int64_t kn_stride_h,
    uint16_t* v_norms, int64_t vn_stride_l, int64_t vn_stride_p, int64_t vn_stride_h,
    const int32_t* page_table, int64_t table_stride_b, const int32_t* start_pos,
    const int32_t* path, int64_t path_stride_b, const int32_t* counts, int32_t* lengths,
    int layers, int B, int Hkv, int S, int A, int nodes, int num_pages, int max_pages, void* stream) {
  using namespace wn;
  clear_error();
  WN_REQUIRE(layers >= 0 && B >= 0 && Hkv > 0 && k_row > 0 && v_row > 0 && num_pages > 0 && max_pages > 0, WN_E_INVALID,
             "commit: bad sizes layers=%d B=%d Hkv=%d rows=%d/%d", layers, B, Hkv, k_row, v_row);
  WN_REQUIRE(A > 0 && nodes > 0 && A <= nodes && nodes <= 64, WN_E_INVALID, "commit: need 1 <= A <= nodes <= 64 (A=%d, nodes=%d)", A, nodes);
  WN_REQUIRE(is_pow2(S), WN_E_INVALID, "commit: page size %d is not a power of two", S);
  if (layers == 0 || B == 0) return WN_OK;
  WN_REQUIRE(k_pages && v_pages && !k_norms == !v_norms && page_table && start_pos && path && counts && lengths, WN_E_INVALID,
             "commit: null operand");
  WN_REQUIRE(lengths != start_pos, WN_E_INVALID, "commit: lengths may not be start_pos itself");
  WN_REQUIRE(layers <= 65535 && int64_t(B) * Hkv < (int64_t(1) << 31), WN_E_INVALID, "commit: grid too large");
  auto unit = [](const void* p, int64_t l, int64_t pg, int64_t h, int row) {
    const uint64_t all = reinterpret_cast<uintptr_t>(p) | uint64_t(l) | uint64_t(pg) | uint64_t(h) | uint64_t(row) | 16;
    return int(all & (~all + 1));  // the lowest bit set
  };
  CommitArgs a;
  a.side[0] = CommitSide{k_pages, k_norms, k_stride_l, k_stride_p, k_stride_h, kn_stride_l, kn_stride_p, kn_stride_h, k_row,
                         unit(k_pages, k_stride_l, k_stride_p, k_stride_h, k_row)};
  a.side[1] = CommitSide{v_pages, v_norms, v_stride_l, v_stride_p, v_stride_h, vn_stride_l, vn_stride_p, vn_stride_h, v_row,
                         unit(v_pages, v_stride_l, v_stride_p, v_stride_h, v_row)};
  a.table = page_table;
  a.tsb = table_stride_b;
  a.start = start_pos;
  a.path = path;
  a.psb = path_stride_b;
  a.counts = counts;
  a.lengths = lengths;
  a.B = B;
  a.Hkv = Hkv;
  a.A = A;
  a.nodes = nodes;
  a.log2S = ilog2(S);
  a.num_pages = num_pages;
  a.max_pages = max_pages;
  hipLaunchKernelGGL(commit_kernel, dim3(unsigned(B) * unsigned(Hkv), unsigned(layers), 2), dim3(64), 0,
                     static_cast<hipStream_t>(stream), a);
  return check_launch("wn_commit_kv");
}
