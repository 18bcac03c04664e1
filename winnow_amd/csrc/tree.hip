// Host side of the tree attention (wn_tree.h).
#include <algorithm>

#include "wn_tree_host.h"

namespace wn {
namespace {

constexpr int kTreeNodes = 64;
// Tiles of 16 rows from which a work-group merges a whole one (4 rows each below: 16 tiles merged from
// 10 splits took 7.7 us a tile to a work-group, 6.0 us in fours).
constexpr int64_t kMergeTiles = 256;

TreeKernels pick_tree(int D, bool exact, int bw_k, int bw_v) {
  switch (D) {
    case 16: return tree_kernels_16(exact, bw_k, bw_v);
    case 32: return tree_kernels_32(exact, bw_k, bw_v);
    case 64: return tree_kernels_64(exact, bw_k, bw_v);
    case 128: return tree_kernels_128(exact, bw_k, bw_v);
    case 256: return tree_kernels_256(exact, bw_k, bw_v);
    default: return TreeKernels{};
  }
}

// Whether the row scan serves (head_dim 128, single-term products, 4 and 6-bit widths, `wide`: rows and
// norms laid out for its loads, see rows_wide). `tokens`: positions that the page table holds, over the
// batch and kv heads (not the lengths: those of a captured call change between replays, and short
// sequences behind a wide table pay what the figures for few tokens show). A wave of it needs long splits
// (it starts with 128 KB of tables), and every 32 rows look codes up again, which the tile scan does
// once per row block, by byte-pair tables if both sides have 4 bits. Whole calls, tile and row scan, us:
//   4/4 bits, 32 rows:  256 k tokens 45 / 48, 512 k 60 / 56, 1 M 96 / 74
//             64 rows:  256 k 59 / 60, 512 k 81 / 75, 1 M 122 / 101;  128 rows: 512 k 101 / 101
//   4/6 bits, 32 rows:  64 k tokens 37 / 45, 128 k 46 / 43, 256 k 60 / 48, 1 M 148 / 79
//             64 rows:  64 k 46 / 46, 128 k 62 / 53;  128 rows: 64 k 58 / 52, 1 M 277 / 184
bool rows_serve(int D, bool exact, bool wide, int bw_k, int bw_v, int64_t rows, int64_t tokens) {
  if (D != 128 || exact || !wide || (bw_k != 4 && bw_k != 6) || (bw_v != 4 && bw_v != 6)) return false;
  return bw_k + bw_v == 8 ? rows <= 64 && tokens >= 524288 : std::max<int64_t>(rows, 32) * tokens >= 4194304;
}

// The row scan reads K by 16 bytes (4 bits) or 8, and four norms at once.
bool rows_wide(int bw_k, const void* k_pages, int64_t k_stride_p, int64_t k_stride_h, const void* k_norms, int64_t kn_stride_p,
               int64_t kn_stride_h, const void* v_norms, int64_t vn_stride_p, int64_t vn_stride_h) {
  const int k = bw_k == 4 ? 16 : 8;
  return aligned(k_pages, k) && k_stride_p % k == 0 && k_stride_h % k == 0 && aligned(k_norms, 8) && aligned(v_norms, 8) &&
         kn_stride_p % 4 == 0 && kn_stride_h % 4 == 0 && vn_stride_p % 4 == 0 && vn_stride_h % 4 == 0;
}

TreeScan tree_variant(int D, bool exact, bool wide, int bw_k, int bw_v, int64_t rows, int64_t tokens) {
  if (rows_serve(D, exact, wide, bw_k, bw_v, rows, tokens)) return tree_rows_scan(bw_k, bw_v);
  return pick_tree(D, exact, bw_k, bw_v).scan[rows <= 32 ? 0 : rows <= 64 ? 1 : 2];
}

bool tree_shape(int B, int Hq, int Hkv, int T, int D) {
  return B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && T > 0 && T <= kTreeNodes && valid_head_dim(D) &&
         int64_t(Hq / Hkv) * T <= (1 << 20);
}

}  // namespace
}  // namespace wn

extern "C" int wn_tree_plan(int B, int Hq, int Hkv, int T, int D, int S, int bw_k, int bw_v, int exact, int max_pages,
                            const int32_t* lens, int* num_splits, int* span, int* parts) {
  using namespace wn;
  clear_error();
  WN_REQUIRE(tree_shape(B, Hq, Hkv, T, D) && max_pages > 0 && int64_t(max_pages) * S <= INT32_MAX - 256 && num_splits && span &&
                 parts,
             WN_E_INVALID, "wn_tree_plan: bad sizes B=%d Hq=%d Hkv=%d T=%d D=%d max_pages=%d", B, Hq, Hkv, T, D, max_pages);
  WN_REQUIRE(is_pow2(S) && S >= 16 && valid_bw(bw_k) && valid_bw(bw_v), WN_E_UNSUPPORTED,
             "wn_tree_plan: (S=%d, bw_k=%d, bw_v=%d) not compiled", S, bw_k, bw_v);
  const int64_t rows = int64_t(Hq / Hkv) * T;
  const TreeScan scan = tree_variant(D, exact != 0, true, bw_k, bw_v, rows, int64_t(B) * Hkv * max_pages * S);
  const int groups = tree_slots(scan, tree_lds(scan, bw_k, bw_v));
  WN_REQUIRE(groups > 0, WN_E_LAUNCH, "wn_tree_plan: cannot query the device occupancy");
  const int64_t slots = groups * int64_t(std::max(1, scan.waves));
  const int64_t heads = int64_t(Hkv) * (tree_nrp(scan, rows) / scan.rows);
  const int n = lens ? B : 1;
  const int64_t each = lens ? 1 : std::max(B, 1);  // sequences per entry of lens
  int64_t longest = 1;
  auto chunks = [&](int b) { return (std::min<int64_t>(std::max(lens ? lens[b] : max_pages * S, 1), int64_t(max_pages) * S) + 63) / 64; };
  for (int b = 0; b < n; ++b) longest = std::max(longest, chunks(b));
  // For one to four rounds of the slots, the smallest split whose count over the batch fits; the
  // least of rounds times (split and its fixed cost: tables, query, partials, about four chunks).
  int64_t best = 0, best_cost = 0;
  for (int64_t rounds = 1; rounds <= 4; ++rounds) {
    int64_t lo = 1, hi = longest;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      int64_t count = 0;
      for (int b = 0; b < n; ++b) count += (chunks(b) + mid - 1) / mid;
      if (count * each * heads <= rounds * slots) hi = mid;
      else lo = mid + 1;
    }
    const int64_t cost = rounds * (lo + 4);
    if (!best || cost < best_cost) {
      best = lo;
      best_cost = cost;
    }
  }
  best = std::max(best, (longest + 255) / 256);
  *span = int(64 * best);
  *num_splits = int((longest + best - 1) / best);
  int64_t count = 0;
  for (int b = 0; b < n; ++b) count += (chunks(b) + best - 1) / best;
  *parts = int(std::min<int64_t>(count * each, INT32_MAX));
  return WN_OK;
}

extern "C" int64_t wn_tree_workspace_bytes(int B, int Hq, int Hkv, int T, int D, int num_splits) {
  using namespace wn;
  if (!tree_shape(B, Hq, Hkv, T, D) || num_splits <= 0) return -1;
  // the most that any scan of this shape takes
  const int64_t rows = int64_t(Hq / Hkv) * T;
  return tree_layout(B, Hkv, tree_nrp(tree_variant(D, false, false, 8, 8, rows, 0), rows), T, D, num_splits).total;
}

extern "C" int wn_tree_attention(
    const void* q, int q_dtype, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
    const float* pi_k, const float* pi_v, const float* codebook_k, const float* codebook_v,
    const uint8_t* k_pages, int64_t k_stride_p, int64_t k_stride_h,
    const uint8_t* v_pages, int64_t v_stride_p, int64_t v_stride_h,
    const uint16_t* k_norms, int64_t kn_stride_p, int64_t kn_stride_h,
    const uint16_t* v_norms, int64_t vn_stride_p, int64_t vn_stride_h,
    const int32_t* page_table, int64_t table_stride_b, const int32_t* seq_lens,
    const int32_t* parents, int64_t parents_stride_b,
    void* out, int out_dtype, void* workspace, int64_t workspace_bytes,
    int B, int Hq, int Hkv, int T, int D, int S, int bw_k, int bw_v, int num_pages, int max_pages,
    float scale, int exact, int num_splits, int span, int parts, void* stream, void* ev_begin, void* ev_end) {
  using namespace wn;
  clear_error();
  WN_REQUIRE(tree_shape(B, Hq, Hkv, T, D), WN_E_INVALID,
             "tree: need B>=0, Hq%%Hkv==0, 1<=T<=%d, D a power of two 16..256 (B=%d Hq=%d Hkv=%d T=%d D=%d)", kTreeNodes,
             B, Hq, Hkv, T, D);
  WN_REQUIRE(valid_bw(bw_k) && valid_bw(bw_v), WN_E_UNSUPPORTED, "tree: bit widths %d/%d not compiled", bw_k, bw_v);
  WN_REQUIRE(is_pow2(S) && S >= 16, WN_E_INVALID, "tree: page size %d is not a power of two >= 16", S);
  WN_REQUIRE(q_dtype >= WN_F32 && q_dtype <= WN_BF16 && out_dtype >= WN_F32 && out_dtype <= WN_BF16, WN_E_INVALID,
             "tree: dtype codes %d/%d", q_dtype, out_dtype);
  WN_REQUIRE(num_splits > 0 && num_splits <= 4096 && span > 0 && span % 64 == 0 && parts > 0, WN_E_INVALID,
             "tree: num_splits %d, span %d, parts %d", num_splits, span, parts);
  WN_REQUIRE(num_pages > 0 && max_pages > 0 && int64_t(max_pages) * S <= INT32_MAX - 256, WN_E_INVALID,
             "tree: num_pages %d, max_pages %d", num_pages, max_pages);
  if (B == 0) return WN_OK;
  WN_REQUIRE(q && pi_k && pi_v && codebook_k && codebook_v && k_pages && v_pages && k_norms && v_norms && page_table &&
                 seq_lens && parents && out,
             WN_E_INVALID, "tree: null operand");
  WN_REQUIRE(aligned(k_pages, 4) && aligned(v_pages, 4) && k_stride_p % 4 == 0 && k_stride_h % 4 == 0 &&
                 v_stride_p % 4 == 0 && v_stride_h % 4 == 0,
             WN_E_INVALID, "tree: pages need a 4-byte aligned base and strides");
  WN_REQUIRE(k_stride_p >= 0 && v_stride_p >= 0 && k_stride_h >= 0 && v_stride_h >= 0 && kn_stride_p >= 0 &&
                 kn_stride_h >= 0 && vn_stride_p >= 0 && vn_stride_h >= 0 && table_stride_b >= 0 && parents_stride_b >= 0,
             WN_E_INVALID, "tree: negative stride");
  WN_REQUIRE(aligned(pi_k, 16) && aligned(q, q_dtype == WN_F32 ? 4 : 2) && aligned(out, out_dtype == WN_F32 ? 4 : 2),
             WN_E_INVALID, "tree: Pi_K 16-byte aligned, q and out aligned to their type");
  const int n_rep = Hq / Hkv;
  const int64_t rows = int64_t(n_rep) * T;
  const TreeKernels k = pick_tree(D, exact != 0, bw_k, bw_v);
  const bool rows_ok = rows_wide(bw_k, k_pages, k_stride_p, k_stride_h, k_norms, kn_stride_p, kn_stride_h, v_norms, vn_stride_p, vn_stride_h);
  const TreeScan scan = tree_variant(D, exact != 0, rows_ok, bw_k, bw_v, rows, int64_t(B) * Hkv * max_pages * S);
  const int nrp = tree_nrp(scan, rows), ncg = nrp / scan.rows;
  const TreeLayout lay = tree_layout(B, Hkv, nrp, T, D, num_splits);
  WN_REQUIRE(workspace && workspace_bytes >= lay.total && aligned(workspace, 256), WN_E_WORKSPACE,
             "tree: workspace needs %lld bytes, 256-aligned (got %lld)", (long long)lay.total, (long long)workspace_bytes);
  // The tile scan's work-groups for the planned splits, in eights (a unit's row blocks on one XCD);
  // the row scan's waves for every split that could be.
  const int64_t tiles = int64_t(B) * Hkv * (nrp / 16), units = std::min<int64_t>(parts, int64_t(B) * num_splits) * Hkv;
  const int64_t groups = scan.waves ? (int64_t(B) * Hkv * num_splits * ncg + scan.waves - 1) / scan.waves : (units + 7) / 8 * 8 * ncg;
  WN_REQUIRE(tiles < (int64_t(1) << 31) && groups < (int64_t(1) << 31), WN_E_INVALID, "tree: grid too large");
  const int lds = tree_lds(scan, bw_k, bw_v);
  WN_REQUIRE(tree_slots(scan, lds) > 0, WN_E_LAUNCH, "tree: cannot query the device occupancy");

  char* ws = static_cast<char*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  TreeRotArgs ra;
  ra.q = q;
  ra.qsb = q_stride_b;
  ra.qsh = q_stride_h;
  ra.qsq = q_stride_t;
  ra.pi = pi_k;
  ra.parents = parents;
  ra.psb = parents_stride_b;
  ra.qh = reinterpret_cast<_Float16*>(ws + lay.qh);
  ra.ql = reinterpret_cast<_Float16*>(ws + lay.ql);
  ra.qs = reinterpret_cast<float*>(ws + lay.qs);
  ra.qf = scan.waves ? reinterpret_cast<float*>(ws + lay.qh) : nullptr;  // in the two terms' place
  ra.vis = reinterpret_cast<uint64_t*>(ws + lay.vis);
  ra.scale = float(double(scale) * 1.4426950408889634);
  ra.Hkv = Hkv;
  ra.n_rep = n_rep;
  ra.T = T;
  ra.nrp = nrp;
  ra.q_dtype = q_dtype;
  ra.exact = exact != 0;
  const int per = q_dtype == WN_F32 ? 4 : 8;  // elements of 16 bytes
  ra.vec = aligned(q, 16) && q_stride_b % per == 0 && q_stride_h % per == 0 && q_stride_t % per == 0;
  hipLaunchKernelGGL(k.rotate, dim3(unsigned(tiles)), dim3(k.rotate_threads), 0, st, ra);

  TreeArgs a;
  a.qh = ra.qh;
  a.ql = ra.ql;
  a.qs = ra.qs;
  a.qf = ra.qf;
  a.vis = ra.vis;
  a.k_pages = k_pages;
  a.v_pages = v_pages;
  a.k_norms = k_norms;
  a.v_norms = v_norms;
  a.cb_k = codebook_k;
  a.cb_v = codebook_v;
  a.table = page_table;
  a.seq_lens = seq_lens;
  a.part_acc = reinterpret_cast<float*>(ws + lay.acc);
  a.part_ml = reinterpret_cast<float*>(ws + lay.ml);
  a.ksp = k_stride_p;
  a.ksh = k_stride_h;
  a.vsp = v_stride_p;
  a.vsh = v_stride_h;
  a.knp = kn_stride_p;
  a.knh = kn_stride_h;
  a.vnp = vn_stride_p;
  a.vnh = vn_stride_h;
  a.tsb = table_stride_b;
  a.B = B;
  a.Hkv = Hkv;
  a.n_rep = n_rep;
  a.T = T;
  a.nrp = nrp;
  a.ncg = ncg;
  a.nsplit = num_splits;
  a.span = span;
  a.log2S = ilog2(S);
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  a.bwk = bw_k;
  a.bwv = bw_v;
  if (ev_begin) (void)hipEventRecord(static_cast<hipEvent_t>(ev_begin), st);
  hipLaunchKernelGGL(scan.fn, dim3(unsigned(groups)), dim3(scan.threads), lds, st, a);
  if (ev_end) (void)hipEventRecord(static_cast<hipEvent_t>(ev_end), st);

  TreeMergeArgs ma{a.part_acc, a.part_ml, pi_v, out, seq_lens, out_dtype, Hkv, n_rep, T, nrp, num_splits, span, max_pages * S};
  const int64_t wide = int64_t(B) * Hkv * ((rows + 15) / 16);
  if (wide >= kMergeTiles) hipLaunchKernelGGL(k.merge[1], dim3(unsigned(wide)), dim3(1024), 0, st, ma);
  else hipLaunchKernelGGL(k.merge[0], dim3(unsigned(int64_t(B) * Hkv * ((rows + 3) / 4))), dim3(1024), 0, st, ma);
  return check_launch("wn_tree_attention");
}
