// Attention of a tree of drafted tokens over paged packed K/V for gfx950: up to 64
// drafted tokens (nodes) per sequence, whose K and V are the last T positions of the
// cache. Node i sees every position before the tree and, among the nodes, itself and
// its ancestors; with s = scale q . k_hat and k_hat = n_K (c_K Pi_K),
//   out = softmax(s) v_hat = (sum_j p_j n_V,j c_V,j) Pi_V / sum_j p_j,
// so the query is rotated once (q' = q Pi_K^T), keys and values are read as codes and
// norms, and the value sum is rotated back once per row.
//
// Three launches on the caller's stream:
//   1. tree_rotate_kernel  q' of every row (row r of a (sequence, kv head) is node
//                          r / n_rep, head r % n_rep of the group) as fp16, or as two
//                          fp16 terms, with a power-of-two scale per row; and every
//                          node's 64-bit word of visible nodes, from the parents;
//   2. tree_scan_kernel    a work-group per (split of the batch's tokens, kv head, row block):
//                          online softmax over its chunks, an (acc, m, l) partial per row
//                          (tree_rows.hip holds the scan of long contexts);
//   3. tree_merge_kernel   per row the max-stable merge of its splits, 1/l, Pi_V, cast.
//
// The scan, per chunk of 64 tokens (32 at head_dim 256): all threads turn the packed rows
// into fp16 tiles in LDS, K as [token][dim] and V as [dim][token], each code looked up
// once per work-group in a table of (high, low) fp16 terms of 2^8 c, or, for 4-bit codes and
// single terms, of a byte's two codes at once; then wave (rg, tg) takes row group rg and token
// group tg. Per 16 x 16 tile (lane 16 g + c) scores have A = K (row c = token tile_row(t, c),
// k-slots = 8 dims) and B = q' (column c = query row), so that a lane's score registers of tiles
// 2ks, 2ks + 1 are the consecutive tokens 32 ks + 8 g .. + 7 of one row: as the value product's
// B operand P never leaves the registers, and A is one 16-byte read of the V tile. Blocks of 16,
// 32 or 64 rows and more per wave and work-group by how many rows a kv head has: a chunk is
// decoded once for a whole block.
//
// What bounds it is instruction issue (decoding: six instructions a code by single lookups, three
// by pairs; the softmax: thirteen a score) beside the matrix instructions, and, for few rows,
// latency. Whole scans on a 256-CU device, medians of traces, two terms a factor and one: 8
// sequences of 500 to 6,000 tokens, 28 heads over 4, 26 nodes, 4 bits: 68 us and 40; 16 of 32,768,
// 32 heads over 8, 16 nodes, 4 bits: 520 to 650 us (twelve in a row lower the clock) and 245, with
// two terms up to 0.8 PFLOP/s of fp16 products: of 520 us at 2.4 GHz the vector instructions fill
// 45% and the products 31%; 4 of 15,000 to 20,000, 64 heads over 8, 64 nodes, 4 and 6 bits: 520 to 620 and 285; one of
// 300, 32 heads over 8, 8 nodes: 12 and 10, of which a chunk takes 2.
//
// Precision. EX = true, the callers' default for every type: every factor is a sum of two fp16
// terms (22 bits), and each product the three larger of their four products (what is left out is
// below 2^-22 of a term): fp32 accuracy. EX = false, where the caller allows TF32-class products:
// one fp16 term per factor (rounded to nearest, off by 2^-11 of it at most, the bits of a TF32
// factor), a third of the matrix work. Sums, maxima and partials are fp32 either way.
#pragma once

#include <cstdint>
#include <utility>

#include "wn_common.h"

namespace wn {

struct TreeArgs {
  const _Float16* qh;  // (B Hkv nrp, D) high terms of q' 2^e
  const _Float16* ql;  // low terms (EX)
  const float* qs;     // (B Hkv nrp) scale log2(e) 2^-(e + 8)
  const float* qf;     // (B Hkv nrp, 128) scale log2(e) q' in place of the three (row scan)
  const uint64_t* vis; // (B T) visible nodes of a node
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const uint16_t* k_norms;
  const uint16_t* v_norms;
  const float* cb_k;
  const float* cb_v;
  const int32_t* table;
  const int32_t* seq_lens;
  float* part_acc;             // (items, 16, D), item = ((b Hkv + kvh) nsplit + s) nrp / 16 + row block
  float* part_ml;              // (items, 16, 2): maximum (log2 units), sum
  int64_t ksp, ksh, vsp, vsh;  // page strides, bytes
  int64_t knp, knh, vnp, vnh;  // norm strides, elements
  int64_t tsb;                 // page-table row stride, elements
  int B, Hkv, n_rep, T, nrp, ncg, nsplit, span, log2S, max_pages, num_pages, bwk, bwv;
};

// Tokens of a split of a sequence of L: `span` (a multiple of 64), more where nsplit of them do not
// cover it. Long and short sequences then have splits of one size, and as many as they need.
__host__ __device__ inline int tree_span(int L, int nsplit, int span) {
  const int even = int((int64_t(L) + nsplit - 1) / nsplit + 63) / 64 * 64;
  return span > even ? span : even;
}

// Splits of a sequence of L, and where split s of them ends. A sequence may come as near to 2^31 as
// 257 positions and a span too, so that their sum, or a whole last split, would pass it.
__host__ __device__ inline int tree_count(int L, int span) { return L > 0 ? (L - 1) / span + 1 : 0; }
__host__ __device__ inline int tree_end(int L, int span, int s) {
  const int rest = L - s * span;
  return rest < span ? L : s * span + span;
}

// Of both scans:
constexpr float kTreeRescale = 8.0f;  // a maximum moves when a score exceeds it by more
constexpr int kTreeNoScale = -64;     // value scale before the first norm

#ifdef __HIPCC__
// g with x < 2^g for a non-negative finite fp16 x > 0, the least such.
__device__ __forceinline__ int tree_exponent(uint32_t bits) {
  return bits >> 10 ? int(bits >> 10) - 14 : 8 - __builtin_clz(bits);
}

// The largest of the four lanes 16 apart, in each of them.
__device__ __forceinline__ float tree_max16(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  x = fmaxf(__builtin_bit_cast(float, uint32_t(a[0])), __builtin_bit_cast(float, uint32_t(a[1])));
  const auto b = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, uint32_t(b[0])), __builtin_bit_cast(float, uint32_t(b[1])));
}

// Split j of the batch, its splits counted sequence after sequence: its sequence and place there.
// False past the last one. Every lane of a wave takes part.
__device__ __forceinline__ bool tree_split(const TreeArgs& a, int lane, int j, int* b, int* s) {
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int L = b0 + lane < a.B ? min(max(a.seq_lens[b0 + lane], 0), a.max_pages << a.log2S) : 0;
    const int own = tree_count(L, tree_span(L, a.nsplit, a.span));
    int upto = own;  // of this lane's sequence and those before it
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      upto += lane >= o ? x : 0;
    }
    const int all = __builtin_amdgcn_readlane(upto, 63);
    if (j < before + all) {
      const int k = __builtin_popcountll(__ballot(before + upto <= j));
      *b = b0 + k;
      *s = j - before - __builtin_amdgcn_readlane(upto - own, k);
      return true;
    }
    before += all;
  }
  return false;
}

// Addresses of the rows of 16-token groups. Lane (kind, i) of the wave's first 16 holds the address of
// group i's K rows, V rows, K norms or V norms (kind 0 .. 3): formed by one product a chunk, and read
// from there into scalars, where a scalar product per group and kind took a sixth of the scan's
// instructions.
// Of global memory, by type: through a pointer that the compiler must take for any memory's, every wait
// for LDS waits for the rows too.
using TreeBytes = const __attribute__((address_space(1))) uint8_t*;
struct TreeRows {
  uint64_t base, stride;  // of the kind: pool + head, bytes per page
  uint32_t token;         // bytes per token
  uint64_t at;            // of the group
  __device__ __forceinline__ void init(const TreeArgs& a, int lane, int kvh, uint32_t nbk, uint32_t nbv) {
    const int kind = lane >> 2 & 3;
    base = kind == 0   ? reinterpret_cast<uint64_t>(a.k_pages) + uint64_t(kvh) * uint64_t(a.ksh)
           : kind == 1 ? reinterpret_cast<uint64_t>(a.v_pages) + uint64_t(kvh) * uint64_t(a.vsh)
           : kind == 2 ? reinterpret_cast<uint64_t>(a.k_norms) + uint64_t(kvh) * uint64_t(a.knh) * 2
                       : reinterpret_cast<uint64_t>(a.v_norms) + uint64_t(kvh) * uint64_t(a.vnh) * 2;
    stride = uint64_t(kind == 0 ? a.ksp : kind == 1 ? a.vsp : kind == 2 ? a.knp * 2 : a.vnp * 2);
    token = kind == 0 ? nbk : kind == 1 ? nbv : 2;
  }
  __device__ __forceinline__ void set(uint32_t page, int slot) {
    at = base + uint64_t(page) * stride + uint32_t(slot) * token;
  }
  __device__ __forceinline__ TreeBytes rows(int kind, int group) const {  // wave-uniform
    const int l = 4 * kind + group;
    return TreeBytes(uint64_t(uint32_t(__builtin_amdgcn_readlane(int(at >> 32), l))) << 32 |
                                            uint32_t(__builtin_amdgcn_readlane(int(uint32_t(at)), l)));
  }
  __device__ __forceinline__ TreeBytes rows_lane(int kind, int group) const {  // by the lane
    const int l = 4 * kind + group;
    return TreeBytes(uint64_t(uint32_t(__shfl(int(at >> 32), l, 64))) << 32 |
                                            uint32_t(__shfl(int(uint32_t(at)), l, 64)));
  }
};
#endif

struct TreeRotArgs {
  const void* q;
  int64_t qsb, qsh, qsq;  // element strides of q (B, Hq, T, D)
  const float* pi;
  const int32_t* parents;
  int64_t psb;  // parents' row stride, elements
  _Float16* qh;
  _Float16* ql;
  float* qs;
  float* qf;  // not null: fp32 rows, no terms
  uint64_t* vis;
  float scale;  // scale log2(e)
  int Hkv, n_rep, T, nrp, q_dtype, exact;
  int vec;  // q's base and strides are multiples of 16 bytes
};

struct TreeMergeArgs {
  const float* part_acc;
  const float* part_ml;
  const float* pi_v;
  void* out;  // (B, Hq, T, D) contiguous
  const int32_t* seq_lens;
  int out_dtype, Hkv, n_rep, T, nrp, nsplit, span, max_len;
};

using TreeScanFn = void (*)(TreeArgs);
using TreeRotFn = void (*)(TreeRotArgs);
using TreeMergeFn = void (*)(TreeMergeArgs);

template <class Args>
struct TreeScanOf {
  void (*fn)(Args) = nullptr;
  int rows = 0, threads = 0;  // query rows and threads of a work-group
  int lds = 0, tables = 0;    // LDS bytes without the codebook tables; theirs (0: by the widths)
  int give = 0;               // LDS bytes that the hand-over at the end takes
  int waves = 0;              // > 0: the row scan, so many waves a work-group, each with its own rows
};
using TreeScan = TreeScanOf<TreeArgs>;

template <class Args, class MergeArgs>
struct TreeKernelsOf {
  TreeScanOf<Args> scan[4];  // for up to 32, up to 64, more rows per kv head; the windowed attention's for many
  TreeRotFn rotate = nullptr;
  int rotate_threads = 0;
  void (*merge[2])(MergeArgs) = {};  // of four and of sixteen rows a work-group
};
using TreeKernels = TreeKernelsOf<TreeArgs, TreeMergeArgs>;

// Bytes of one side's codebook table in LDS: 2^bw entries of (high, low), a copy per bank
// (16 of 6-bit tables, 8 of 8-bit ones: their size).
__host__ __device__ constexpr int tree_copies(int bw) { return bw <= 5 ? 32 : bw == 6 ? 16 : 8; }
__host__ __device__ constexpr int tree_table_bytes(int bw) { return (4 << bw) * tree_copies(bw); }

// The row scan (tree_rows.hip): head_dim 128, 4 and 6-bit K and V, single-term products.
TreeScan tree_rows_scan(int bw_k, int bw_v);

TreeKernels tree_kernels_16(bool exact, int bw_k, int bw_v);
TreeKernels tree_kernels_32(bool exact, int bw_k, int bw_v);
TreeKernels tree_kernels_64(bool exact, int bw_k, int bw_v);
TreeKernels tree_kernels_128(bool exact, int bw_k, int bw_v);
TreeKernels tree_kernels_256(bool exact, int bw_k, int bw_v);

// The windowed attention (window.hip): the same scan, rows and merge, with another choice of keys.
// The T queries of a sequence are its last T positions; the one at position p sees the positions
// j <= p with p - j < window or j < sinks.
struct WindowArgs : TreeArgs {
  int window, sinks;
};

struct WindowMergeArgs : TreeMergeArgs {
  int window, sinks, rows_block, chunk;  // rows of a scan's work-group, tokens of its chunk
  int tiles;  // of sixteen rows of a unit, over all of them
};

// Of window_rotate_kernel and window_merge_kernel: a wave per 16 columns, four at least.
__host__ __device__ constexpr int window_row_threads(int D) { return 4 * D > 256 ? 4 * D : 256; }

// The chunks that the queries of rows r0 .. r0 + rows - 1 of a (sequence, kv head) look at: those that
// hold sinks, then those from the first query's window to the last query. `total` of them, counted as
// if what lies between had been cut out: chunk c is the sequence's c < sink ? c : c + skip. Splits
// take `span` of them each.
struct WindowSpan {
  int lo, hi;  // positions: first of the window, one past the last
  int p_lo, p_hi;  // of the first and last query
  int total, sink, skip, span;
  __host__ __device__ int chunk(int c) const { return c < sink ? c : c + skip; }
};
__host__ __device__ inline WindowSpan window_span(int L, int T, int n_rep, int r0, int rows, int ch, int window, int sinks, int nsplit,
                                                  int span) {
  const auto lesser = [](int a, int b) { return a < b ? a : b; };
  const auto greater = [](int a, int b) { return a > b ? a : b; };
  WindowSpan w;
  w.p_lo = L - T + r0 / n_rep;
  w.p_hi = L - T + lesser(T - 1, (r0 + rows - 1) / n_rep);
  w.hi = greater(w.p_hi + 1, 0);
  w.lo = greater(greater(w.p_lo, 0) - window + 1, 0);
  w.sink = (lesser(sinks, w.hi) + ch - 1) / ch;
  w.skip = greater(w.lo / ch - w.sink, 0);
  w.total = (w.hi + ch - 1) / ch - w.skip;
  const int even = (w.total + nsplit - 1) / nsplit;
  w.span = greater(span / ch, even);
  return w;
}

struct WindowKernels : TreeKernelsOf<WindowArgs, WindowMergeArgs> {
  void (*rotate_many)(TreeRotArgs, int) = nullptr;  // of many tiles of sixteen rows, from head_dim 128 on
};
WindowKernels window_kernels_16(bool exact, int bw_k, int bw_v);
WindowKernels window_kernels_32(bool exact, int bw_k, int bw_v);
WindowKernels window_kernels_64(bool exact, int bw_k, int bw_v);
WindowKernels window_kernels_128(bool exact, int bw_k, int bw_v);
WindowKernels window_kernels_256(bool exact, int bw_k, int bw_v);

}  // namespace wn
