// Attention over paged packed K/V under a sliding window with sinks, for gfx950: the Q queries of a
// sequence are its last Q positions, and the one at position p sees the positions j <= p with
// p - j < window or j < sinks,
//   out = softmax(scale q . k_hat) v_hat,   k_hat = n_K (c_K Pi_K),   v_hat = n_V (c_V Pi_V).
//
// Host side. What lies between the sinks and the window is passed over, in chunks of 64 positions or in pages:
// a call costs the window and up to three of these, not the context. Two scans:
//
// * the tree attention's (wn_tree.h, wn_tree_kernels.h), compiled for this choice of keys: q' = q Pi_K^T
//   once, a scan of the chunks that some query of a row block sees (window_span), split where there are
//   few blocks, and a merge with Pi_V. It serves every shape. 512 queries at a window of 4,096, 32 heads
//   over 8, fp32 accuracy: 113 us of the call's 133 (125 of 157 in the first calls after a pause), 0.9 PFLOP/s of fp16 products (three a factor). Vector instructions (softmax, decoding) issue in
//   54% of its cycles, products in 45%.
// * one query at head_dim 128: the decode's row scan (wn_decode_rows.h) over the pages in view, laid out
//   side by side by the launch that rotates the query (window_view, decode.hip). It reads these pages whole
//   and masks what is out of view of them. 32 sequences at a window of 8,192, 32 heads over 8, 4 bits,
//   pages of 16: 71 us, 3.9 TB/s; a step of one user at 1,024: 20 us, three launches' latency. Pages much
//   longer than the window are where the tile scan, which passes over chunks, would read less: 32 sequences at
//   a window of 64, us by row scan and tile scan: pages of 16 23 and 28, of 1,024 33 and 28, of 4,096 48 and 28.
#include "wn_decode.h"
#include "wn_tree_host.h"

namespace wn {
namespace {

WindowKernels pick_window(int D, bool exact, int bw_k, int bw_v) {
  switch (D) {
    case 16: return window_kernels_16(exact, bw_k, bw_v);
    case 32: return window_kernels_32(exact, bw_k, bw_v);
    case 64: return window_kernels_64(exact, bw_k, bw_v);
    case 128: return window_kernels_128(exact, bw_k, bw_v);
    case 256: return window_kernels_256(exact, bw_k, bw_v);
    default: return WindowKernels{};
  }
}

int window_chunk(int D) { return D == 256 ? 32 : 64; }  // tokens of a scan's chunk

// The tile scan for so many rows per kv head and (sequence, kv head) pairs. Blocks of 256 rows decode a
// chunk for twice the rows of blocks of 128, in 1.7 times the time (7.6 and 4.5 us a chunk): where that
// many fewer serve, and there are enough of them to go round. Calls of 32 heads over 8, 4 bits, us, 128 and
// 256 rows: 2,048 rows at a window of 4,096 175 and 155, 8,000 rows 241 and 205, 192 rows of 8 sequences 162
// and 140, of one 53 and 55; 384 rows 60 and 64; 512 68 and 66; 336 rows, 4 kv heads 49 and 57.
int window_variant(int64_t rows, int64_t pairs) {
  if (rows <= 64) return rows <= 32 ? 0 : 1;
  const int64_t small = (rows + 127) / 128, large = (rows + 255) / 256;
  return 17 * large <= 10 * small && pairs * small >= 32 ? 3 : 2;
}

bool window_shape(int B, int Hq, int Hkv, int Q, int D) {
  return B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Q > 0 && valid_head_dim(D) && int64_t(Hq / Hkv) * Q <= (1 << 20);
}

}  // namespace
}  // namespace wn

extern "C" int wn_window_plan(int B, int Hq, int Hkv, int Q, int D, int S, int bw_k, int bw_v, int exact, int wide, int max_pages,
                              int window, int sinks, const int32_t* lens, int* num_splits, int* span) {
  using namespace wn;
  clear_error();
  WN_REQUIRE(window_shape(B, Hq, Hkv, Q, D) && max_pages > 0 && int64_t(max_pages) * S <= INT32_MAX - 256 && window > 0 && sinks >= 0 &&
                 num_splits && span,
             WN_E_INVALID, "wn_window_plan: bad sizes B=%d Hq=%d Hkv=%d Q=%d D=%d max_pages=%d window=%d sinks=%d", B, Hq, Hkv, Q, D,
             max_pages, window, sinks);
  WN_REQUIRE(is_pow2(S) && S >= 16 && valid_bw(bw_k) && valid_bw(bw_v), WN_E_UNSUPPORTED,
             "wn_window_plan: (S=%d, bw_k=%d, bw_v=%d) not compiled", S, bw_k, bw_v);
  const int n_rep = Hq / Hkv, ch = window_chunk(D);
  const int64_t rows = int64_t(n_rep) * Q;
  // One query at head_dim 128 takes the decode's row scan wherever that is compiled, whatever its size. Calls
  // of 32 heads over 8 at 4 bits, us, row scan and tile scan: 1 sequence at 256 tokens in view 19.8 and 20.0, at
  // 8,192 28 and 29; 8 at 1,024 23 and 30, at 4,096 29 and 51; 32 at 8,192 75 and 224.
  if (Q == 1 && wide) {
    const int waves = window_rows_waves(Hq, Hkv, D, bw_k, bw_v, exact == 0);
    if (waves > 0) {
      *num_splits = waves;
      *span = 0;
      return WN_OK;
    }
  }
  const auto scan = pick_window(D, exact != 0, bw_k, bw_v).scan[window_variant(rows, int64_t(B) * Hkv)];
  const int64_t slots = tree_slots(scan, tree_lds(scan, bw_k, bw_v));
  WN_REQUIRE(slots > 0, WN_E_LAUNCH, "wn_window_plan: cannot query the device occupancy");
  const int blocks = tree_nrp(scan, rows) / scan.rows;
  const int n = lens ? B : 1;
  const int64_t each = (lens ? 1 : std::max(B, 1)) * int64_t(Hkv) * blocks;  // work-groups per entry of lens and split
  // chunks of a sequence's last row block, or, where rows fill only part of that and so span fewer positions,
  // the more of its and the one's before: the others have as many, fewer, or by where they begin one more
  auto chunks = [&](int b) {
    const int L = int(std::min<int64_t>(std::max(lens ? lens[b] : max_pages * S, 0), int64_t(max_pages) * S));
    int64_t most = 1;
    for (int blk = blocks - 1; blk >= 0 && blk >= blocks - (rows % scan.rows ? 2 : 1); --blk)
      most = std::max<int64_t>(most, window_span(L, Q, n_rep, blk * scan.rows, scan.rows, ch, window, sinks, 1, ch).total);
    return most;
  };
  int64_t longest = 1;
  for (int b = 0; b < n; ++b) longest = std::max(longest, chunks(b));
  // For one to four rounds of the slots, the smallest split whose count over the batch fits; the least
  // of rounds times (split and its fixed cost: tables, query, partials, about four chunks).
  int64_t best = 0, best_cost = 0;
  for (int64_t rounds = 1; rounds <= 4; ++rounds) {
    int64_t lo = 1, hi = longest;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      int64_t count = 0;
      for (int b = 0; b < n; ++b) count += (chunks(b) + mid - 1) / mid;
      if (count * each <= rounds * slots) hi = mid;
      else lo = mid + 1;
    }
    const int64_t cost = rounds * (lo + 4);
    if (!best || cost < best_cost) {
      best = lo;
      best_cost = cost;
    }
  }
  best = std::max(best, (longest + 255) / 256);
  if (ch < 64) best = (best + 1) / 2 * 2;
  *span = int(ch * best);
  *num_splits = int((longest + best - 1) / best);
  return WN_OK;
}

extern "C" int64_t wn_window_workspace_bytes(int B, int Hq, int Hkv, int Q, int D, int S, int max_pages, int window, int sinks,
                                             int num_splits, int span) {
  using namespace wn;
  if (!window_shape(B, Hq, Hkv, Q, D) || !is_pow2(S) || max_pages <= 0 || window <= 0 || sinks < 0 || num_splits <= 0 || span < 0) return -1;
  if (span == 0) return Q == 1 && D == 128 ? window_rows_workspace(B, Hq, Hkv, S, max_pages, window, sinks, num_splits) : -1;
  const int64_t rows = int64_t(Hq / Hkv) * Q;
  const auto scan = pick_window(D, false, 8, 8).scan[window_variant(rows, int64_t(B) * Hkv)];
  return tree_layout(B, Hkv, tree_nrp(scan, rows), 0, D, num_splits).total;
}

extern "C" int wn_window_attention(
    const void* q, int q_dtype, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_q,
    const float* pi_k, const float* pi_v, const float* codebook_k, const float* codebook_v,
    const uint8_t* k_pages, int64_t k_stride_p, int64_t k_stride_h,
    const uint8_t* v_pages, int64_t v_stride_p, int64_t v_stride_h,
    const uint16_t* k_norms, int64_t kn_stride_p, int64_t kn_stride_h,
    const uint16_t* v_norms, int64_t vn_stride_p, int64_t vn_stride_h,
    const int32_t* page_table, int64_t table_stride_b, const int32_t* seq_lens,
    void* out, int out_dtype, void* workspace, int64_t workspace_bytes,
    int B, int Hq, int Hkv, int Q, int D, int S, int bw_k, int bw_v, int num_pages, int max_pages,
    int window, int sinks, float scale, int exact, int num_splits, int span, void* stream, void* ev_begin, void* ev_end) {
  using namespace wn;
  clear_error();
  WN_REQUIRE(window_shape(B, Hq, Hkv, Q, D), WN_E_INVALID,
             "window: need B>=0, Hq%%Hkv==0, Q>0, n_rep*Q<=2^20, D a power of two 16..256 (B=%d Hq=%d Hkv=%d Q=%d D=%d)", B, Hq, Hkv, Q, D);
  WN_REQUIRE(valid_bw(bw_k) && valid_bw(bw_v), WN_E_UNSUPPORTED, "window: bit widths %d/%d not compiled", bw_k, bw_v);
  WN_REQUIRE(is_pow2(S) && S >= 16, WN_E_INVALID, "window: page size %d is not a power of two >= 16", S);
  WN_REQUIRE(q_dtype >= WN_F32 && q_dtype <= WN_BF16 && out_dtype >= WN_F32 && out_dtype <= WN_BF16, WN_E_INVALID,
             "window: dtype codes %d/%d", q_dtype, out_dtype);
  WN_REQUIRE(window > 0 && sinks >= 0, WN_E_INVALID, "window: window %d (at least 1), sinks %d", window, sinks);
  WN_REQUIRE(span == 0 ? num_splits > 0 && Q == 1 && D == 128 : num_splits > 0 && num_splits <= 4096 && span > 0 && span % 64 == 0,
             WN_E_INVALID, "window: num_splits %d, span %d", num_splits, span);
  WN_REQUIRE(num_pages > 0 && max_pages > 0 && int64_t(max_pages) * S <= INT32_MAX - 256, WN_E_INVALID,
             "window: num_pages %d, max_pages %d", num_pages, max_pages);
  if (B == 0) return WN_OK;
  WN_REQUIRE(q && pi_k && pi_v && codebook_k && codebook_v && k_pages && v_pages && k_norms && v_norms && page_table && seq_lens && out,
             WN_E_INVALID, "window: null operand");
  WN_REQUIRE(aligned(k_pages, 4) && aligned(v_pages, 4) && k_stride_p % 4 == 0 && k_stride_h % 4 == 0 && v_stride_p % 4 == 0 &&
                 v_stride_h % 4 == 0,
             WN_E_INVALID, "window: pages need a 4-byte aligned base and strides");
  WN_REQUIRE(k_stride_p >= 0 && v_stride_p >= 0 && k_stride_h >= 0 && v_stride_h >= 0 && kn_stride_p >= 0 && kn_stride_h >= 0 &&
                 vn_stride_p >= 0 && vn_stride_h >= 0 && table_stride_b >= 0,
             WN_E_INVALID, "window: negative stride");
  WN_REQUIRE(aligned(pi_k, 16) && aligned(q, q_dtype == WN_F32 ? 4 : 2) && aligned(out, out_dtype == WN_F32 ? 4 : 2), WN_E_INVALID,
             "window: Pi_K 16-byte aligned, q and out aligned to their type");
  if (span == 0)
    return window_rows_attention(WindowStep{q, q_dtype, q_stride_b, q_stride_h, pi_k, pi_v, codebook_k, codebook_v, k_pages, v_pages,
                                            k_stride_p, k_stride_h, v_stride_p, v_stride_h, k_norms, v_norms, kn_stride_p, kn_stride_h,
                                            vn_stride_p, vn_stride_h, page_table, table_stride_b, seq_lens, out, out_dtype, workspace,
                                            workspace_bytes, B, Hq, Hkv, S, bw_k, bw_v, num_pages, max_pages, window, sinks, scale,
                                            exact == 0, num_splits, stream, ev_begin, ev_end});
  const int n_rep = Hq / Hkv;
  const int64_t rows = int64_t(n_rep) * Q;
  const WindowKernels k = pick_window(D, exact != 0, bw_k, bw_v);
  const auto scan = k.scan[window_variant(rows, int64_t(B) * Hkv)];
  const int nrp = tree_nrp(scan, rows), ncg = nrp / scan.rows;
  const TreeLayout lay = tree_layout(B, Hkv, nrp, 0, D, num_splits);
  WN_REQUIRE(workspace && workspace_bytes >= lay.total && aligned(workspace, 256), WN_E_WORKSPACE,
             "window: workspace needs %lld bytes, 256-aligned (got %lld)", (long long)lay.total, (long long)workspace_bytes);
  // work-groups in eights: a unit's row blocks, which read much the same rows, on one XCD
  const int64_t tiles = int64_t(B) * Hkv * (nrp / 16), groups = (int64_t(B) * num_splits * Hkv + 7) / 8 * 8 * ncg;
  WN_REQUIRE(grid_fits(tiles, k.rotate_threads) && grid_fits(groups, scan.threads), WN_E_INVALID, "window: grid too large");
  const int lds = tree_lds(scan, bw_k, bw_v);
  WN_REQUIRE(tree_slots(scan, lds) > 0, WN_E_LAUNCH, "window: cannot query the device occupancy");

  char* ws = static_cast<char*>(workspace);
  hipStream_t st = static_cast<hipStream_t>(stream);
  TreeRotArgs ra{};
  ra.q = q;
  ra.qsb = q_stride_b;
  ra.qsh = q_stride_h;
  ra.qsq = q_stride_q;
  ra.pi = pi_k;
  ra.qh = reinterpret_cast<_Float16*>(ws + lay.qh);
  ra.ql = reinterpret_cast<_Float16*>(ws + lay.ql);
  ra.qs = reinterpret_cast<float*>(ws + lay.qs);
  ra.scale = float(double(scale) * 1.4426950408889634);
  ra.Hkv = Hkv;
  ra.n_rep = n_rep;
  ra.T = Q;
  ra.nrp = nrp;
  ra.q_dtype = q_dtype;
  ra.exact = exact != 0;
  const int per = q_dtype == WN_F32 ? 4 : 8;  // elements of 16 bytes
  ra.vec = aligned(q, 16) && q_stride_b % per == 0 && q_stride_h % per == 0 && q_stride_q % per == 0;
  const int threads = window_row_threads(D);
  const int64_t stay = int64_t(std::max(1, device_cus())) * (1024 / threads);  // 1,024 threads a compute unit
  if (k.rotate_many && tiles * D >= (1 << 17))  // wn_window_rows.h has both sides
    hipLaunchKernelGGL(k.rotate_many, dim3(unsigned(std::min(tiles, stay))), dim3(threads), 0, st, ra, int(tiles));
  else hipLaunchKernelGGL(k.rotate, dim3(unsigned(tiles)), dim3(k.rotate_threads), 0, st, ra);

  WindowArgs a{};
  a.qh = ra.qh;
  a.ql = ra.ql;
  a.qs = ra.qs;
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
  a.T = Q;
  a.nrp = nrp;
  a.ncg = ncg;
  a.nsplit = num_splits;
  a.span = span;
  a.log2S = ilog2(S);
  a.max_pages = max_pages;
  a.num_pages = num_pages;
  a.bwk = bw_k;
  a.bwv = bw_v;
  a.window = window;
  a.sinks = sinks;
  if (ev_begin) (void)hipEventRecord(static_cast<hipEvent_t>(ev_begin), st);
  hipLaunchKernelGGL(scan.fn, dim3(unsigned(groups)), dim3(scan.threads), lds, st, a);
  if (ev_end) (void)hipEventRecord(static_cast<hipEvent_t>(ev_end), st);

  WindowMergeArgs ma{};
  ma.part_acc = a.part_acc;
  ma.part_ml = a.part_ml;
  ma.pi_v = pi_v;
  ma.out = out;
  ma.seq_lens = seq_lens;
  ma.out_dtype = out_dtype;
  ma.Hkv = Hkv;
  ma.n_rep = n_rep;
  ma.T = Q;
  ma.nrp = nrp;
  ma.nsplit = num_splits;
  ma.span = span;
  ma.max_len = max_pages * S;
  ma.window = window;
  ma.sinks = sinks;
  ma.rows_block = scan.rows;
  ma.chunk = window_chunk(D);
  const int64_t wide = int64_t(B) * Hkv * ((rows + 15) / 16);
  ma.tiles = int(wide);
  // few splits, or many rows: wn_window_rows.h has both sides
  if (num_splits <= 8 || wide >= 128)
    hipLaunchKernelGGL(k.merge[1], dim3(unsigned(std::min(wide, stay))), dim3(threads), 0, st, ma);
  else hipLaunchKernelGGL(k.merge[0], dim3(unsigned(int64_t(B) * Hkv * ((rows + 3) / 4))), dim3(1024), 0, st, ma);
  return check_launch("wn_window_attention");
}
