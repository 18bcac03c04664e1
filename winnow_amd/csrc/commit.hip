// Keeping the accepted branch of a drafted tree in a paged cache.
//
// The rows of drafted node path[b, i] (position start[b] + path[b, i]) move to position
// start[b] + i for i < counts[b], K and V, codes and norms, in every layer and kv head, and
// lengths[b] = start[b] + counts[b]. Rows only change place: no arithmetic.
//
// Bound: latency. A step moves some hundred bytes per (layer, sequence, head, side), each
// behind the lookups of its positions and pages; one wave per such group keeps them all in
// flight at once (a full batch: 8,192 waves) and asks in three round trips: for the counts,
// paths and starts, for both pages of every node, for rows and norms together. No load sits
// behind a branch, where the compiler waits for each: 28 layers, 4 heads, 5 rows 3.2 us (16.7 with
// the branches), 32 layers x 16 sequences x 8 heads, 12 rows 6.7 (19.6), x 24, 7 rows of 256 bytes
// 8.9 (22.8). A row may be the target of one move and the
// source of another, so a wave reads every source of a block of columns before it writes;
// blocks of columns are independent of each other.
#include <algorithm>

#include "wn_common.h"

namespace wn {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kUnits = 4;  // pieces of rows that a lane holds

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

__device__ __forceinline__ int commit_log2(int x) { return x > 1 ? 32 - __builtin_clz(x - 1) : 0; }  // up

// Blocks of 2^lg columns of all n rows (lg from 2 on: n is at most 64), each read before it is written.
template <class T>
__device__ __forceinline__ void commit_rows(const CommitSide& s, uint8_t* base, const int64_t* src, const int64_t* dst,
                                            int n, int lane, uint16_t norm, uint16_t* norm_to) {
  const int cols = s.row / int(sizeof(T)), lg = min(min(commit_log2(cols), 6), commit_log2(64 * kUnits) - commit_log2(n));
  for (int c0 = 0; c0 < cols; c0 += 1 << lg) {
    const int64_t col = c0 + (lane & ((1 << lg) - 1));
    T v[kUnits];
    int64_t to[kUnits];
    bool live[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int row = (lane + 64 * k) >> lg, at = min(row, 63);
      const int64_t from = src[at];
      live[k] = row < n && col < cols && from >= 0;
      to[k] = dst[at] + col * int64_t(sizeof(T));
      // no branch around a load, which would wait for it: a lane without a row reads the layer's first
      v[k] = *reinterpret_cast<const T*>(base + (live[k] ? from + col * int64_t(sizeof(T)) : 0));
    }
    // read before written, over all lanes of the wave; the norms, asked for before, are here too
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (c0 == 0 && norm_to) *norm_to = norm;
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      if (live[k]) *reinterpret_cast<T*>(base + to[k]) = v[k];
    }
  }
}

__global__ __launch_bounds__(64) void commit_kernel(CommitArgs a) {
  __shared__ int64_t src[64], dst[64];  // byte offsets of a layer's head; -1: nothing to move
  const int lane = threadIdx.x;
  const int b = blockIdx.x / a.Hkv, kvh = blockIdx.x % a.Hkv, layer = blockIdx.y;
  const CommitSide s = a.side[blockIdx.z];
  // every argument in one round trip, not each where it is first used
  asm volatile("" ::"s"(s.pages), "s"(s.norms), "s"(s.sl), "s"(s.sp), "s"(s.sh), "s"(s.nl), "s"(s.np), "s"(s.nh), "s"(s.row),
               "s"(s.unit), "s"(a.table), "s"(a.tsb), "s"(a.path), "s"(a.psb), "s"(a.num_pages), "s"(a.max_pages), "s"(a.nodes),
               "s"(a.log2S));
  const int node = a.path[b * a.psb + min(lane, a.A - 1)], count = a.counts[b], start = a.start[b];
  const int n = min(max(count, 0), a.A);
  if (blockIdx.z == 0 && layer == 0 && kvh == 0 && lane == 0) a.lengths[b] = start + n;
  if (n == 0) return;  // the whole work-group
  // the pages of both positions; none where the table or the pool has none
  const int64_t from = int64_t(start) + node, to = int64_t(start) + lane;
  const int64_t positions = int64_t(a.max_pages) << a.log2S;
  const bool move = lane < n && node >= 0 && node < a.nodes && node != lane && start >= 0 && from < positions && to < positions;
  const int32_t* trow = a.table + b * a.tsb;
  int32_t sp = -1, dp = -1;
  if (move) {
    sp = trow[from >> a.log2S];
    dp = trow[to >> a.log2S];
  }
  const int mask = (1 << a.log2S) - 1, ss = int(from) & mask, ds = int(to) & mask;
  const bool found = sp >= 0 && sp < a.num_pages && dp >= 0 && dp < a.num_pages;
  const int64_t from_at = found ? sp * s.sp + int64_t(ss) * s.row : -1, to_at = dp * s.sp + int64_t(ds) * s.row;
  uint16_t* norms = s.norms + layer * s.nl + kvh * s.nh;
  // as below: no branch around a load
  const uint16_t norm = *(found && s.norms ? norms + (sp * s.np + ss) : reinterpret_cast<const uint16_t*>(a.counts));
  uint16_t* norm_to = found && s.norms ? norms + (dp * s.np + ds) : nullptr;
  src[lane] = from_at;
  dst[lane] = to_at;
  __builtin_amdgcn_wave_barrier();  // one wave: its LDS accesses are in order, and no load is waited for
  uint8_t* base = s.pages + layer * s.sl + kvh * s.sh;
  switch (s.unit) {
    case 16: commit_rows<u32x4>(s, base, src, dst, n, lane, norm, norm_to); break;
    case 8: commit_rows<u32x2>(s, base, src, dst, n, lane, norm, norm_to); break;
    case 4: commit_rows<uint32_t>(s, base, src, dst, n, lane, norm, norm_to); break;
    case 2: commit_rows<uint16_t>(s, base, src, dst, n, lane, norm, norm_to); break;
    default: commit_rows<uint8_t>(s, base, src, dst, n, lane, norm, norm_to);
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
  WN_REQUIRE(layers > 0 && B >= 0 && Hkv > 0 && k_row > 0 && v_row > 0 && num_pages > 0 && max_pages > 0, WN_E_INVALID,
             "commit: bad sizes layers=%d B=%d Hkv=%d rows=%d/%d", layers, B, Hkv, k_row, v_row);
  WN_REQUIRE(A > 0 && nodes > 0 && A <= nodes && nodes <= 64, WN_E_INVALID, "commit: need 1 <= A <= nodes <= 64 (A=%d, nodes=%d)", A, nodes);
  WN_REQUIRE(is_pow2(S), WN_E_INVALID, "commit: page size %d is not a power of two", S);
  if (B == 0) return WN_OK;
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
