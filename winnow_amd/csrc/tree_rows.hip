// Tree attention (wn_tree.h) at head_dim 128 with 4 and 6-bit K and V and single-term products:
// one wave takes 32 query rows of a (sequence, kv head) against its split's 64-token chunks, every
// code going from the packed row through an LDS codebook table straight into a matrix-instruction
// operand (wn_rows.h). Nothing is shared between waves, so no wave waits for another, and no tile is
// written to LDS and read back: 740 wave instructions per chunk of 32 rows (64 of them matrix
// instructions, 128 table reads), where the tile kernel (wn_tree_kernels.h) spends 2,300 on 64 rows.
// Two waves share a SIMD. What bounds it is instruction issue: 16 sequences of 32,768 tokens, 8 kv
// heads, 64 rows, 4 bits: 245 us, 0.56 PFLOP/s (tile kernel: 388 us). 64 rows a wave (128
// accumulators, one wave per SIMD) took 318: a lookup then feeds four matrix instructions, but nothing
// fills the waits.
#include "wn_rows.h"
#include "wn_tree.h"

namespace wn {
namespace {

template <int NCT>
__device__ __forceinline__ void rows_scale(PfState<NCT>& st, const float (&f)[NCT]) {
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) st.acc[ct][mt] *= f[ct];
}

template <int BWK, int BWV, int NCT, int WPB>
__global__ __launch_bounds__(64 * WPB) __attribute__((amdgpu_waves_per_eu(WPB / 4, WPB / 4))) void tree_rows_kernel(TreeArgs a) {
  using Lay = PfLds<BWK, BWV>;
  constexpr int NR = 16 * NCT;
  __shared__ __align__(16) char lds[Lay::total];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wig = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Unit (split of the batch, kv head) times row blocks of NR; a work-group's waves take neighbouring
  // ones. The grid has a wave for every split there could be (a loop over units, as the tile kernel
  // has, keeps its values in registers that this kernel lacks: it spilled, 327 us for 251 at 8 x
  // 32,000 tokens), the last of which find none.
  const int64_t w0 = int64_t(blockIdx.x) * WPB, w = w0 + wig;
  int b, s;
  if (!tree_split(a, lane, int(w0 / a.ncg) / a.Hkv, &b, &s)) return;  // the whole work-group
  stage_table_tf<BWK, 64 * WPB>(a.cb_k, lds + Lay::k_off, tid);
  stage_table_tf<BWV, 64 * WPB>(a.cb_v, lds + Lay::v_off, tid);
  __syncthreads();  // the only block-wide barrier: waves run independently from here
  const int cb = int(w % a.ncg), unit = int(w / a.ncg), kvh = unit % a.Hkv;
  if (!tree_split(a, lane, unit / a.Hkv, &b, &s)) return;  // wave-uniform

  PfState<NCT> st;
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) st.acc[ct][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    st.m[ct] = -INFINITY;
    st.l[ct] = 0.f;
  }
  st.gs = kTreeNoScale;

  const int L = min(max(const_view(a.seq_lens)[b], 0), a.max_pages << a.log2S);
  const int hist = L - a.T;  // position of node 0
  const int span = tree_span(L, a.nsplit, a.span);
  {
    const int t_lo = s * span, t_hi = tree_end(L, span, s), n = (t_hi - t_lo + 63) >> 6, col_hi = (t_hi - 1) >> a.log2S;
    const int32_t* trow = a.table + int64_t(b) * a.tsb;
    const uint32_t last_page = uint32_t(a.num_pages - 1);
    auto tiles = [&](int c0) {
      PfTiles tl = pf_tiles(a, trow, c0, col_hi);
#pragma unroll
      for (int t = 0; t < 4; ++t) tl.pid[t] = min(tl.pid[t], last_page);
      return tl;
    };

    // B operands of the scores: column c of tile ct = row 16 ct + c of the block, K-step k = dims
    // 32 g + 8 k .. + 7 of q' 2^e, rounded to nearest; e from the block's largest finite value
    // (below 2^15 then), so a row that is not finite leaves the others alone
    const float* q0 = a.qf + ((int64_t(b) * a.Hkv + kvh) * a.nrp + cb * NR + c) * 128 + 32 * g;
    float top = 0.f;
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const f32x4 x = reinterpret_cast<const f32x4*>(q0 + 16 * 128 * ct)[k];
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(x[j]) < INFINITY ? fabsf(x[j]) : 0.f);
      }
    int qe;
    frexpf(wave_max(top), &qe);
    const int e = min(15 - qe, 110);
    const float sc = ldexpf(1.f, -(e + 8)), up = ldexpf(1.f, e);
    h8 qb[NCT][4];
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f32x4 x0 = reinterpret_cast<const f32x4*>(q0 + 16 * 128 * ct)[2 * k];
        const f32x4 x1 = reinterpret_cast<const f32x4*>(q0 + 16 * 128 * ct)[2 * k + 1];
#pragma unroll
        for (int j = 0; j < 8; ++j) qb[ct][k][j] = _Float16((j < 4 ? x0[j & 3] : x1[j & 3]) * up);
      }


    TabTf<BWK> cbk = make_tab_tf<BWK>(lds, Lay::k_off, lane);
    TabTf<BWV> cbv = make_tab_tf<BWV>(lds, Lay::v_off, lane);
    // the next chunk's K rows load once the scores have read this chunk's, its norms after the
    // weights, its V rows after the values
    PfK<BWK> K;
    PfV<BWV> V;
    PfN N;
    {
      const PfTiles tl = tiles(t_lo);
      pf_load_k<BWK>(a, tl, kvh, lane, K);
      pf_load_n(a, tl, kvh, lane, N);
      pf_load_v<BWV>(a, tl, kvh, lane, V);
    }
    for (int ch = 0; ch < n; ++ch) {
      const int c0 = t_lo + 64 * ch;
      const PfTiles nx = tiles(min(c0 + 64, t_lo + 64 * (n - 1)));  // the last chunk again at the end
      f32x4 d[NCT][4];  // register i of tile t: token 16 t + 4 g + i of column c
      pf_scores<BWK, NCT>(K, cbk, qb, d);
      pf_load_k<BWK>(a, nx, kvh, lane, K);

      const bool full = c0 + 64 <= hist;  // before the tree: every row sees every token
      uint32_t bad = 0;                   // tokens whose value norm is not finite
      if (!full) {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          // what lies past the sequence may hold anything
          const int sh = 16 * (k & 1);
          const uint32_t v = N.nv[k >> 1] >> sh & 0x7fffu;
          const bool out = c0 + 16 * (k >> 2) + 4 * g + (k & 3) >= t_hi;
          if (!out && v >= 0x7c00u) bad |= 1u << k;
          if (out || v >= 0x7c00u) N.nv[k >> 1] &= ~(0xffffu << sh);
          if (out) N.nk[k >> 1] &= ~(0xffffu << sh);
        }
      }
      // value scale: every n_V < 2^(7 + gs), so 2^kTreeRescale n_V 2^-gs < 2^15 in fp16; it follows
      // the norms' magnitude
      {
        u16x2 hi = __builtin_bit_cast(u16x2, N.nv[0] & 0x7fff7fffu);
#pragma unroll
        for (int k = 1; k < 8; ++k) hi = __builtin_elementwise_max(hi, __builtin_bit_cast(u16x2, N.nv[k] & 0x7fff7fffu));
        uint32_t size = max(uint32_t(hi[0]), uint32_t(hi[1]));
        size = size < 0x7c00u ? size : 0;
        if (__any(f16_to_f32(uint16_t(size)) >= ldexpf(1.f, 7 + st.gs))) {  // wave-uniform, rare
          const uint32_t most = __builtin_bit_cast(uint16_t, _Float16(wave_max(f16_to_f32(uint16_t(size)))));
          if (most && tree_exponent(most) - 7 > st.gs) {
            const int to = tree_exponent(most) - 7;
            float f[NCT];
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
              f[ct] = ldexpf(1.f, st.gs - to);
              st.l[ct] *= f[ct];
            }
            st.gs = to;
            rows_scale<NCT>(st, f);
          }
        }
      }
      // scores less the row's maximum and gs, so that p 2^-gs = 2^d
      const float gsf = float(st.gs);
      float nks[16], tops[NCT];
#pragma unroll
      for (int k = 0; k < 16; ++k) nks[k] = half_at(N.nk, k) * sc;
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        const float m0 = (st.m[ct] == -INFINITY ? 0.f : st.m[ct]) + gsf;
        tops[ct] = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) d[ct][t][i] = fmaf(d[ct][t][i], nks[4 * t + i], -m0);
      }
      if (!full) {
        // some of the chunk's tokens are nodes, seen by their descendants only, or lie past the
        // sequence; a value norm that is not finite makes the rows that see it NaN and no other
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
          const int node = (cb * NR + 16 * ct + c) / a.n_rep;
          const uint64_t vis = node < a.T ? a.vis[int64_t(b) * a.T + node] : 0;
          const int at = hist - c0;  // the tree's first position in the chunk (or before it)
          const uint64_t word = at >= 0 ? (vis << at | ((uint64_t(1) << at) - 1)) : at > -64 ? vis >> -at : 0;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t seen = uint32_t(word >> (16 * t + 4 * g));
#pragma unroll
            for (int i = 0; i < 4; ++i)
              d[ct][t][i] = !(seen >> i & 1) ? -INFINITY : (bad >> (4 * t + i) & 1) ? __builtin_nanf("") : d[ct][t][i];
          }
        }
      }
      bool move[NCT], any = false;
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) tops[ct] = fmaxf(tops[ct], d[ct][t][i]);
        tops[ct] = tree_max16(tops[ct]) + gsf;
        move[ct] = tops[ct] > kTreeRescale || (st.m[ct] == -INFINITY && tops[ct] > -INFINITY);
        any = any || move[ct];
      }
      if (__any(any)) {
        float alpha[NCT];
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
          const bool fresh = st.m[ct] == -INFINITY;
          const float shift = move[ct] ? tops[ct] : 0.f;
          alpha[ct] = move[ct] ? (fresh ? 0.f : __builtin_amdgcn_exp2f(-tops[ct])) : 1.f;
          st.m[ct] = move[ct] ? (fresh ? 0.f : st.m[ct]) + tops[ct] : st.m[ct];
          st.l[ct] *= alpha[ct];
#pragma unroll
          for (int t = 0; t < 4; ++t) d[ct][t] -= shift;
        }
        rows_scale<NCT>(st, alpha);
      }
      // weights p n_V 2^-gs into the value B operands: K-step ks takes this lane's own score
      // registers, tokens (2 ks, i) at k-slots i and (2 ks + 1, i) at 4 + i; l sums p 2^-gs
      h8 pb[NCT][2];
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float p = __builtin_amdgcn_exp2f(d[ct][2 * ks + (j >> 2)][j & 3]);
            st.l[ct] += p;
            pb[ct][ks][j] = _Float16(p * half_at(N.nv, 8 * ks + j));
          }
      pf_load_n(a, nx, kvh, lane, N);
      pf_merge_pairs<BWV>(V, lane);
      pf_values<BWV, NCT>(V, cbv, pb, st);
      pf_load_v<BWV>(a, nx, kvh, lane, V);
    }
  }
  const float lf = ldexpf(1.f, st.gs);
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) st.l[ct] *= lf;
  pf_write<NCT>(a, st, (((int64_t(b) * a.Hkv + kvh) * a.nsplit + s) * a.ncg + cb) * NR, lane);
}

template <int BWK, int BWV>
TreeScan rows_scan() {
  return TreeScan{tree_rows_kernel<BWK, BWV, 2, 8>, 32, 512, 0, 0, 0, 8};
}

}  // namespace

TreeScan tree_rows_scan(int bw_k, int bw_v) {
  if (bw_k == 4) return bw_v == 4 ? rows_scan<4, 4>() : rows_scan<4, 6>();
  return bw_v == 4 ? rows_scan<6, 4>() : rows_scan<6, 6>();
}

}  // namespace wn
