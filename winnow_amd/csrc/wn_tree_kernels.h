// The kernels of the tree attention (wn_tree.h), templates on the head dim.
#pragma once

#include <type_traits>

#include "wn_tree.h"

namespace wn {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kTreeCb = 256.0f;  // codebook values are scaled by 2^8

template <int D>
struct TreeGeo {
  static constexpr int DP = D < 32 ? 32 : D;        // K dims, padded to one K-step
  static constexpr int KS = DP / 32, MT = D / 16;   // score K-steps, value M-tiles
  static constexpr int CH = D == 256 ? 32 : 64;     // tokens per chunk
  static constexpr int NG = CH / 16;                // 16-token groups, each within a page (S >= 16)
  // An operand read takes one 16-byte column of sixteen rows at once, the banks hold 256 bytes:
  // K tile rows have their columns swapped by a key of the token that is another one (or another
  // part of the banks) for each of a score tile's rows; rows shorter than 128 bytes are padded.
  // V tile rows likewise by a key of the dim, which the writes (eight dim groups, two columns) spread
  // over eight columns too. Read at 4.5 clocks a wave and CU; a key of eight rows only: 8.2.
  static constexpr int KROW = DP >= 64 ? 2 * DP : 2 * DP + 16;
  static constexpr int VROW = 2 * CH;
  static constexpr int KT = CH * KROW, VT = D * VROW;
  __device__ static uint32_t k_key(int tok) {
    return DP >= 128 ? (tok & 3) | (tok >> 1 & 12) : (tok >> 1 & 1) | (tok >> 2 & 6);
  }
  __device__ static uint32_t k_at(int tok, int col) {
    if constexpr (DP >= 64) return uint32_t(tok * KROW) + ((uint32_t(col) ^ k_key(tok)) << 4);
    else return uint32_t(tok * KROW + (col << 4));
  }
  __device__ static uint32_t v_key(int row) { return CH == 64 ? (row >> 1 & 7) ^ (row >> 4 & 3) : (row >> 2 & 3) ^ (row >> 4 & 1); }
  __device__ static uint32_t v_at(int row, int col) { return uint32_t(row * VROW) + ((uint32_t(col) ^ v_key(row)) << 4); }
};

// Token of row c of score tile t.
__device__ __forceinline__ int tree_tok(int t, int c) { return 32 * (t >> 1) + 8 * (c >> 2) + 4 * (t & 1) + (c & 3); }

// The raw words of one group of eight codes: the one or two 4-byte words that hold bytes
// [o, o + bw) of a block; no other word is read.
struct TreeRaw {
  uint32_t lo, hi;
};
template <int BW>
__device__ __forceinline__ TreeRaw tree_raw(TreeBytes block, uint32_t o, int bw) {
  using Words = const __attribute__((address_space(1))) uint32_t*;
  TreeRaw r;
  r.lo = *Words(block + (o & ~3u));
  // the same word again where one holds them all: a branch would wait for the load before it
  if constexpr (BW == 4) r.hi = 0;
  else r.hi = *Words(block + ((o + uint32_t(bw) - 1) & ~3u));
  return r;
}

// Table entries (high | low << 16) of the eight codes of a group that starts at byte o.
template <int BW>
__device__ __forceinline__ void tree_entries(TreeRaw r, uint32_t o, const char* tab, uint32_t lane, uint32_t (&e)[8]) {
  constexpr int COP = tree_copies(BW);
  const uint32_t own = (lane & uint32_t(COP - 1)) << 2, sh = 8 * (o & 3);
  const uint64_t w = BW == 4 ? uint64_t(r.lo) : (uint64_t(r.hi) << 32 | r.lo) >> sh;
  const uint32_t lo = uint32_t(w), hi = uint32_t(w >> 32);
#pragma unroll
  for (int m = 0; m < 8; ++m) {
    const int bit = BW * m;
    uint32_t c;
    if (bit + BW <= 32) c = lo >> bit;
    else if (bit >= 32) c = hi >> (bit - 32);
    else c = __builtin_amdgcn_alignbit(hi, lo, bit);
    c &= (1u << BW) - 1u;
    e[m] = *reinterpret_cast<const uint32_t*>(tab + (c * uint32_t(4 * COP) | own));
  }
}

// (low halves of a and b) and (high halves)
__device__ __forceinline__ uint32_t pack_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t pack_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// f(width) with the width as a constant; W: the width where the kernel is compiled for one.
template <int W, class F>
__device__ __forceinline__ void tree_by_width(int bw, F&& f) {
  if constexpr (W != 0) {
    f(std::integral_constant<int, W>{});
  } else {
    switch (bw) {  // wave-uniform
      case 2: f(std::integral_constant<int, 2>{}); break;
      case 3: f(std::integral_constant<int, 3>{}); break;
      case 4: f(std::integral_constant<int, 4>{}); break;
      case 5: f(std::integral_constant<int, 5>{}); break;
      case 6: f(std::integral_constant<int, 6>{}); break;
      default: f(std::integral_constant<int, 8>{}); break;
    }
  }
}

// A codebook as (high, low) fp16 terms of 2^8 c, in copies.
template <int NTHR>
__device__ __forceinline__ void tree_stage_table(const float* cb, int bw, char* dst, int tid) {
  const int cop = tree_copies(bw), n = (1 << bw) * cop;
  for (int i = tid; i < n; i += NTHR) {
    const float x = cb[i / cop] * kTreeCb;
    const _Float16 h = _Float16(x), l = _Float16(x - float(h));
    reinterpret_cast<uint32_t*>(dst)[i] =
        uint32_t(__builtin_bit_cast(uint16_t, h)) | uint32_t(__builtin_bit_cast(uint16_t, l)) << 16;
  }
}

// A 4-bit codebook by the byte: the fp16 values of 2^8 c of a byte's two codes, in copies. One
// lookup then serves two codes. Eight copies, 8 KB: a lookup takes 4.4 clocks a wave and CU
// (sixteen copies: 4.2; a copy per bank, 32 KB: 3.0).
constexpr int kPairCopies = 8, kPairBytes = 256 * kPairCopies * 4;
template <int NTHR>
__device__ __forceinline__ void tree_stage_pairs(const float* cb, char* dst, int tid) {
  for_strided<256 * kPairCopies, NTHR>(tid, [&](int i) {
    const int v = i / kPairCopies;
    const _Float16 a = _Float16(cb[v & 15] * kTreeCb), b = _Float16(cb[v >> 4] * kTreeCb);
    reinterpret_cast<uint32_t*>(dst)[i] =
        uint32_t(__builtin_bit_cast(uint16_t, a)) | uint32_t(__builtin_bit_cast(uint16_t, b)) << 16;
  });
}
// Entry of byte J of x.
template <int J>
__device__ __forceinline__ uint32_t tree_pair(uint32_t x, const char* tab, uint32_t own) {
  constexpr int SH = 5;  // 4 kPairCopies bytes an entry
  static_assert(4 * kPairCopies == 1 << SH, "");
  const uint32_t at = (J == 0 ? x << SH : x >> (8 * J - SH)) & (255u << SH);
  return *reinterpret_cast<const uint32_t*>(tab + (at | own));
}

// Largest of the sixteen lanes of a row, in each of them.
__device__ __forceinline__ uint32_t tree_row_max(uint32_t x) {
  x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), 0x128, 0xf, 0xf, true)));  // row_ror:8, 4, 2, 1
  x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), 0x124, 0xf, 0xf, true)));
  x = max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), 0x122, 0xf, 0xf, true)));
  return max(x, uint32_t(__builtin_amdgcn_mov_dpp(int(x), 0x121, 0xf, 0xf, true)));
}

template <int D, bool EX, int NCT, int RG, int TG>
struct TreeCfg {
  using G = TreeGeo<D>;
  static constexpr int NW = RG * TG, NTHR = 64 * NW, ROWS = 16 * NCT * RG;
  static constexpr int NTW = G::CH / 16 / TG;  // score tiles of a wave
  static constexpr int PL = EX ? 2 : 1;        // planes of a tile
  // dequantization items of a chunk: K (token, 8 dims), dims fastest; V (token pair, 8 dims), a
  // wave taking the 8 pairs of GPW groups of 16 tokens times DGL groups of dims
  static constexpr int KI = G::CH * D / 8, NK = (KI + NTHR - 1) / NTHR;
  static constexpr int DGL = D / 8 < 8 ? D / 8 : 8, GPW = 8 / DGL;
  static constexpr int VGB = (G::NG + GPW - 1) / GPW, VC = VGB * (D / 8 / DGL), NV = (VC + NW - 1) / NW;
  static constexpr int k_off = 0, v_off = k_off + PL * G::KT, n_off = v_off + PL * G::VT;
  // norms: K then V, fp16; then the largest V norm of each group of tokens
  static constexpr int m_off = n_off + 4 * G::CH, tab_off = m_off + 16;
  // the waves of token group 1 hand over (acc, m, l) in the tiles' place, sixteen rows at a time
  static constexpr int give = RG * 16 * (D + 2) * 4;
  static_assert(TG == 1 || give <= tab_off, "hand-over fits");
  static_assert(NTW % 2 == 0 && tab_off % 16 == 0 && TG <= 2, "whole value K-steps");
};

// Bits 0 .. x - 1 of 64.
__device__ __forceinline__ uint64_t tree_below(int x) { return x <= 0 ? 0 : x >= 64 ? ~uint64_t(0) : (uint64_t(1) << x) - 1; }

// WIN: the windowed attention; a work-group is one split of one row block of a (sequence, kv head).
template <int D, bool EX, int NCT, int RG, int TG, int W, bool WIN = false>
__global__ __launch_bounds__(64 * RG * TG, 2) void tree_scan_kernel(std::conditional_t<WIN, WindowArgs, TreeArgs> a) {
  using C = TreeCfg<D, EX, NCT, RG, TG>;
  using G = TreeGeo<D>;
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wig = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wig % RG, tg = wig / RG;
  const int bwk = W ? W : a.bwk, bwv = W ? W : a.bwv;
  constexpr bool PAIR = W == 4 && !EX;
  [[maybe_unused]] WindowSpan ws;
  if constexpr (WIN) {
    const int u = (int(blockIdx.x >> 3) / a.ncg) * 8 + int(blockIdx.x & 7), b = u / (a.nsplit * a.Hkv);
    if (b >= a.B) return;  // the whole work-group, here and below
    const int L = min(max(const_view(a.seq_lens)[b], 0), a.max_pages << a.log2S);
    ws = window_span(L, a.T, a.n_rep, int(blockIdx.x >> 3) % a.ncg * C::ROWS, C::ROWS, G::CH, a.window, a.sinks, a.nsplit, a.span);
    if (int64_t(u / a.Hkv % a.nsplit) * ws.span >= ws.total) return;
  }
  char* tabk = lds + C::tab_off;
  char* tabv = tabk + (PAIR ? kPairBytes : tree_table_bytes(bwk));
  if constexpr (PAIR) {
    tree_stage_pairs<C::NTHR>(a.cb_k, tabk, tid);
    tree_stage_pairs<C::NTHR>(a.cb_v, tabv, tid);
  } else {
    tree_stage_table<C::NTHR>(a.cb_k, bwk, tabk, tid);
    tree_stage_table<C::NTHR>(a.cb_v, bwv, tabv, tid);
  }
  // Unit (split of the batch, kv head), and its row block of ROWS. Work-groups go to the eight XCDs
  // in turn: a unit's row blocks, which read the same rows, share one, and units go round. A grid of
  // fewer units than there are (lengths that have grown since it was planned) goes over them again.
  const int cg = int(blockIdx.x >> 3) % a.ncg, step = int(gridDim.x) / a.ncg;
  for (int u = (int(blockIdx.x >> 3) / a.ncg) * 8 + int(blockIdx.x & 7);; u += step) {
    int b, s;
    if constexpr (WIN) {
      b = u / (a.nsplit * a.Hkv);
      s = u / a.Hkv % a.nsplit;
      if (b >= a.B) break;  // the grid holds every unit once: the second turn ends here
    } else if (!tree_split(a, lane, u / a.Hkv, &b, &s)) {
      break;  // the whole work-group
    }
    if constexpr (D < G::DP) {
      // the K tile's padded dims are zero, for each unit again: what the one before handed over at its
      // end (below) lies in the tiles' place, and as fp16 it may be NaN, which the query's zeros keep
      constexpr int PAD = (G::DP - D) / 2;  // words of a row
      for (int i = tid; i < C::PL * G::CH * PAD; i += C::NTHR) {
        const int row = i / PAD;
        char* at = lds + C::k_off + row / G::CH * G::KT + row % G::CH * G::KROW;
        reinterpret_cast<uint32_t*>(at + 2 * D)[i % PAD] = 0;
      }
    }
    const int kvh = u % a.Hkv;
    const int L = min(max(const_view(a.seq_lens)[b], 0), a.max_pages << a.log2S);
    int ch_lo, ch_hi;  // WIN: as ws counts them
    if constexpr (WIN) {
      ch_lo = s * ws.span;
      ch_hi = min(ch_lo + ws.span, ws.total);
    } else {
      const int span = tree_span(L, a.nsplit, a.span);
      ch_lo = s * (span / G::CH);
      ch_hi = (tree_end(L, span, s) + G::CH - 1) / G::CH;
    }
    const int hist = L - a.T;  // position of node 0
    const int rows = a.n_rep * a.T, r0 = cg * C::ROWS + rg * 16 * NCT;  // the wave's first row
    const int64_t row0 = (int64_t(b) * a.Hkv + kvh) * a.nrp + r0;

    f32x4 acc[NCT][G::MT];
    float m[NCT], l[NCT], sc[NCT];
    h8 qh[NCT][G::KS], ql[EX ? NCT : 1][EX ? G::KS : 1];
    int gs = kTreeNoScale;  // values are scaled by 2^(8 - gs)
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
#pragma unroll
      for (int mt = 0; mt < G::MT; ++mt) acc[ct][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[ct] = -INFINITY;
      l[ct] = 0.f;
      const int64_t row = row0 + 16 * ct + c;
      sc[ct] = a.qs[row];
#pragma unroll
      for (int k = 0; k < G::KS; ++k) {
        const bool pad = D < 32 && g >= D / 8;  // dims past D
        qh[ct][k] = pad ? h8{} : *reinterpret_cast<const h8*>(a.qh + row * D + 32 * k + 8 * g);
        if constexpr (EX) ql[ct][k] = pad ? h8{} : *reinterpret_cast<const h8*>(a.ql + row * D + 32 * k + 8 * g);
      }
    }

    {
      int t_hi = min(G::CH * ch_hi, L);
      if constexpr (WIN) t_hi = ws.hi;
      const int col_hi = (t_hi - 1) >> a.log2S, smask = (1 << a.log2S) - 1;
      const int32_t* trow = a.table + int64_t(b) * a.tsb;
      const uint32_t nbk = uint32_t(D * bwk / 8), nbv = uint32_t(D * bwv / 8), last_page = uint32_t(a.num_pages - 1);
      // The rows of each 16-token group of a chunk (S >= 16: they lie in one page). Tokens past the
      // range read its last page (and are masked), so every address is one of the pool.
      TreeRows at;
      at.init(a, lane, kvh, nbk, nbv);
      auto page_ids = [&](int c0) { return uint32_t(trow[min((c0 + 16 * (lane & 3 & (G::NG - 1))) >> a.log2S, col_hi)]); };
      auto pages = [&](uint32_t ids, int c0) { at.set(min(ids, last_page), (c0 + 16 * (lane & 3)) & smask); };
      // Item j of this thread: K (token tok, 8 dims dg), V (tokens 2 tp, 2 tp + 1, 8 dims dg); its
      // group of tokens, wave-uniform from 64 dims on, and whether there is one. A row's address is
      // its group's (scalar) plus the token's within the group (the same for every j).
      constexpr bool UNI = D >= 64, DP64 = D >= 64;
      auto k_item = [&](int j, int* grp, int* tok, int* dg) {
        const int it = tid + C::NTHR * j;
        *tok = it / (D / 8);
        *dg = it % (D / 8);
        *grp = UNI ? (64 * wig + C::NTHR * j) / (D / 8) >> 4 : *tok >> 4;
        return C::KI % C::NTHR == 0 || it < C::KI;
      };
      auto v_item = [&](int j, int* grp, int* tp, int* dg) {
        const int combo = wig + C::NW * j, half = UNI ? 0 : (lane >> 3) / C::DGL;
        *grp = (combo % C::VGB) * C::GPW + half;
        *tp = 8 * *grp + (lane & 7);
        *dg = (combo / C::VGB) * C::DGL + (lane >> 3) % C::DGL;
        return C::VC % C::NW == 0 || combo < C::VC;
      };
      auto block = [&](int kind, int grp) { return UNI ? at.rows(kind, grp) : at.rows_lane(kind, grp); };
      // byte of an item's codes within its group's block of 16 rows
      auto k_off = [&](int tok, int dg) { return uint32_t(tok & 15) * nbk + uint32_t(dg * bwk); };
      auto v_off = [&](int tp, int dg) { return uint32_t(2 * tp & 15) * nbv + uint32_t(dg * bwv); };

      // AHEAD sets of raw rows: chunk n is stored from one while n + 1 travels in the other, and
      // n + 2 is loaded into the first as soon as it is stored (at any widths a row takes twice the
      // registers: one set). Loads are issued on every step, the last ones' again at the end: behind
      // a branch each step's waits would have to cover the path without.
      constexpr int AHEAD = W ? 2 : 1;
      TreeRaw kr[AHEAD][C::NK], vr[AHEAD][C::NV][2];
      uint16_t nr[AHEAD];
      auto load = [&](auto set) {
        constexpr int P = decltype(set)::value;
#pragma unroll
        for (int j = 0; j < C::NK; ++j) {
          int grp, tok, dg;
          if (k_item(j, &grp, &tok, &dg)) kr[P][j] = tree_raw<W>(block(0, grp), k_off(tok, dg), bwk);
        }
#pragma unroll
        for (int j = 0; j < C::NV; ++j) {
          int grp, tp, dg;
          if (!v_item(j, &grp, &tp, &dg)) continue;
          const TreeBytes v = block(1, grp);
          vr[P][j][0] = tree_raw<W>(v, v_off(tp, dg), bwv);
          vr[P][j][1] = tree_raw<W>(v, v_off(tp, dg) + nbv, bwv);
        }
        if (C::NW <= G::NG || wig < G::NG) {  // wave w: the norms of group w, K in lanes 0..15, V in 16..31
          nr[P] = ((const __attribute__((address_space(1))) uint16_t*)(lane & 16 ? at.rows(3, wig) : at.rows(2, wig)))[c];
        }
      };
      uint32_t k_to, v_to;  // LDS addresses of the first items
      {
        int grp, tok, tp, dg;
        k_item(0, &grp, &tok, &dg);
        k_to = uint32_t(C::k_off) + G::k_at(tok, dg);
        v_item(0, &grp, &tp, &dg);
        v_to = uint32_t(C::v_off) + G::v_at(8 * dg, tp >> 2) + 4 * (tp & 3);
      }
      auto store = [&](auto set, int c0) {
        constexpr int P = decltype(set)::value;
        // recomputed from these two each chunk: held as loop invariants, the addresses of every
        // write would take some thirty registers
        asm volatile("" : "+v"(k_to), "+v"(v_to));
        const uint32_t own = uint32_t(lane & (kPairCopies - 1)) << 2;
        // An item's address from the first one's: TOK tokens further on, the key swapped by their
        // bits (steps of 8 and more tokens add to the same bits of the first item's token only where
        // that has none: up to 64 items of a wave lie in one group of 16); eight groups of dims
        // further on, the V tile's key is the same
        auto k_dst = [&](int j, int tok, int dg) {
          constexpr int TOK = C::NTHR / (D / 8);
          if (TOK >= 16 && DP64) return lds + (k_to ^ (G::k_key(TOK * j) << 4)) + uint32_t(TOK * j * G::KROW);
          return lds + C::k_off + G::k_at(tok, dg);
        };
        auto v_dst = [&](int j, int d, int tp, int dg) {
          if (j == 0 || (G::CH == 64 && C::VGB == C::NW))
            return lds + (v_to ^ uint32_t(G::CH == 64 ? d >> 1 << 4 : d >> 2 << 4)) + (d + 8 * C::DGL * j) * G::VROW;
          return lds + C::v_off + G::v_at(8 * dg + d, tp >> 2) + 4 * (tp & 3);
        };
        tree_by_width<W>(bwk, [&](auto bw) {
          constexpr int BW = decltype(bw)::value;
#pragma unroll
          for (int j = 0; j < C::NK; ++j) {
            int grp, tok, dg;
            if (!k_item(j, &grp, &tok, &dg)) continue;
            char* dst = k_dst(j, tok, dg);
            if constexpr (PAIR) {
              const uint32_t x = kr[P][j].lo;
              *reinterpret_cast<u32x4*>(dst) =
                  u32x4{tree_pair<0>(x, tabk, own), tree_pair<1>(x, tabk, own), tree_pair<2>(x, tabk, own), tree_pair<3>(x, tabk, own)};
            } else {
              uint32_t e[8];
              tree_entries<BW>(kr[P][j], k_off(tok, dg), tabk, lane, e);
              *reinterpret_cast<u32x4*>(dst) = u32x4{pack_lo(e[0], e[1]), pack_lo(e[2], e[3]), pack_lo(e[4], e[5]), pack_lo(e[6], e[7])};
              if constexpr (EX)
                *reinterpret_cast<u32x4*>(dst + G::KT) = u32x4{pack_hi(e[0], e[1]), pack_hi(e[2], e[3]), pack_hi(e[4], e[5]), pack_hi(e[6], e[7])};
              if (j & 1) __builtin_amdgcn_sched_barrier(0);  // the lookups of two items in flight
            }
          }
        });
        __builtin_amdgcn_sched_barrier(0);
        tree_by_width<W>(bwv, [&](auto bw) {
          constexpr int BW = decltype(bw)::value;
#pragma unroll
          for (int j = 0; j < C::NV; ++j) {
            int grp, tp, dg;
            if (!v_item(j, &grp, &tp, &dg)) continue;
            if constexpr (PAIR) {
              // byte i of `even`: the codes of dim 2 i of both tokens; of `odd`, of dim 2 i + 1
              constexpr uint32_t m = 0x0f0f0f0fu;
              const uint32_t x = vr[P][j][0].lo, y = vr[P][j][1].lo;
              const uint32_t even = (x & m) | (y << 4 & ~m), odd = (x >> 4 & m) | (y & ~m);
              const uint32_t e[8] = {tree_pair<0>(even, tabv, own), tree_pair<0>(odd, tabv, own), tree_pair<1>(even, tabv, own),
                                     tree_pair<1>(odd, tabv, own),  tree_pair<2>(even, tabv, own), tree_pair<2>(odd, tabv, own),
                                     tree_pair<3>(even, tabv, own), tree_pair<3>(odd, tabv, own)};
#pragma unroll
              for (int d = 0; d < 8; ++d) *reinterpret_cast<uint32_t*>(v_dst(j, d, tp, dg)) = e[d];
            } else {
              uint32_t e0[8], e1[8];
              tree_entries<BW>(vr[P][j][0], v_off(tp, dg), tabv, lane, e0);
              tree_entries<BW>(vr[P][j][1], v_off(tp, dg) + nbv, tabv, lane, e1);
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                char* dst = v_dst(j, d, tp, dg);
                *reinterpret_cast<uint32_t*>(dst) = pack_lo(e0[d], e1[d]);
                if constexpr (EX) *reinterpret_cast<uint32_t*>(dst + G::VT) = pack_hi(e0[d], e1[d]);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        });
        if (C::NW <= G::NG || wig < G::NG) {
          // what lies past the sequence may hold anything
          bool own = c0 + 16 * wig + c < t_hi;
          // nor may what no query of the block sees: its pages may be another's by now
          if constexpr (WIN) own = own && (c0 + 16 * wig + c >= ws.lo || c0 + 16 * wig + c < a.sinks);
          const uint32_t n = own ? nr[P] : 0, size = n & 0x7fffu;
          const uint32_t top = tree_row_max(size < 0x7c00u ? size : 0);  // of the finite ones
          if (lane < 32) reinterpret_cast<uint16_t*>(lds + C::n_off)[(lane >> 4) * G::CH + 16 * wig + c] = uint16_t(n);
          if (lane == 16) reinterpret_cast<uint32_t*>(lds + C::m_off)[wig] = top;
        }
      };

      // LDS addresses of the products' operands: from 64 dims on the XORs of a few registers
      uint32_t kb[G::KS], vb[4];
      const int w0 = 16 * C::NTW * tg;  // the wave's first token of a chunk
#pragma unroll
      for (int k = 0; k < G::KS; ++k) kb[k] = uint32_t(C::k_off) + G::k_at(w0 + tree_tok(0, c), 4 * k + g);
#pragma unroll
      for (int i = 0; i < 4; ++i) vb[i] = (uint32_t(C::v_off) + G::v_at(c, (w0 >> 3) + g)) ^ uint32_t(i << 4);
      // tile t of K-step k: tokens tree_tok(t, 0) further on (bits 2 and 5: not the key's)
      auto k_addr = [&](int t, int k) { return kb[k] + uint32_t(tree_tok(t, 0) * G::KROW); };
      // row 16 mt + c, column (w0 >> 3) + 4 ks + g: mt's part of the key and ks are swaps
      auto v_addr = [&](int mt, int ks) {
        if constexpr (G::CH == 64) return (vb[mt & 3] ^ uint32_t(ks << 6)) + uint32_t(16 * mt * G::VROW);
        else return vb[mt & 1] + uint32_t(16 * mt * G::VROW);
      };
      const int c_last = G::CH * (ch_hi - 1);
      auto next = [&](int c0) { return min(c0, c_last); };  // the last chunk again past the end
      // position of chunk ch, the last one again past the end
      auto at_chunk = [&](int ch) {
        if constexpr (WIN) return G::CH * ws.chunk(min(ch, ch_hi - 1));
        else return next(G::CH * ch);
      };
      constexpr std::integral_constant<int, 0> even;
      constexpr std::integral_constant<int, AHEAD - 1> odd;
      const int c_first = WIN ? at_chunk(ch_lo) : G::CH * ch_lo;
      pages(page_ids(c_first), c_first);
      load(even);
      if constexpr (AHEAD == 2) {
        pages(page_ids(at_chunk(ch_lo + 1)), at_chunk(ch_lo + 1));
        load(odd);
      }
      uint32_t ids = page_ids(at_chunk(ch_lo + AHEAD));
      auto chunk = [&](auto set, int ch) {
        const int c0 = WIN ? at_chunk(ch) : G::CH * ch;
        __syncthreads();  // the last chunk's tiles are read (at first: the tables are staged)
        store(set, c0);
        // the page ids of the chunk after are asked for ahead of the rows: waiting for them next
        // time waits for no row
        pages(ids, at_chunk(ch + AHEAD));
        ids = page_ids(at_chunk(ch + AHEAD + 1));
        load(set);
        __syncthreads();
        if (r0 >= rows) return;  // padding: the wave has only its part of the tiles to do

        // a wave that takes the whole chunk for 32 rows does so in halves, for their registers
        constexpr int HV = WIN && RG == 8 ? C::NTW / 2 : 1, NT = C::NTW / HV;
#pragma unroll
        for (int hf = 0; hf < HV; ++hf) {
        // scores of the wave's tokens: register i of tile t is token w0 + tree_tok(t, 4 g + i)
        f32x4 d[NCT][NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) d[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        // two tiles at a time, so that an accumulator's next product is 2 NCT instructions off
#pragma unroll
        for (int t0 = 0; t0 < NT; t0 += 2)
#pragma unroll
          for (int k = 0; k < G::KS; ++k) {
            const char* kp[2] = {lds + k_addr(NT * hf + t0, k), lds + k_addr(NT * hf + t0 + 1, k)};
            h8 kh[2], kl[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              kh[t] = *reinterpret_cast<const h8*>(kp[t]);
              if constexpr (EX) kl[t] = *reinterpret_cast<const h8*>(kp[t] + G::KT);
            }
            auto products = [&](const h8 (&x)[2], const auto& y) {
#pragma unroll
              for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int ct = 0; ct < NCT; ++ct)
                  d[ct][t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[t], y[ct][k], d[ct][t0 + t], 0, 0, 0);
            };
            products(kh, qh);
            if constexpr (EX) {
              products(kl, qh);
              products(kh, ql);
            }
          }
        __builtin_amdgcn_sched_barrier(0);
        // value scale: every n_V < 2^(7 + gs), so 2^kTreeRescale n_V 2^-gs < 2^15 in fp16; it
        // follows the norms' magnitude (n_V = 2^-20 keeps its bits)
        constexpr int KV = NT / 2;
        {
          const uint32_t* gm = reinterpret_cast<const uint32_t*>(lds + C::m_off);
          uint32_t top = gm[0];
#pragma unroll
          for (int i = 1; i < G::NG; ++i) top = max(top, gm[i]);
          top = __builtin_amdgcn_readfirstlane(int(top));
          if (top && tree_exponent(top) - 7 > gs) {  // wave-uniform, rare after the first chunk
            const int to = tree_exponent(top) - 7;
            const float f = ldexpf(1.f, gs - to);
            gs = to;
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
              l[ct] *= f;
#pragma unroll
              for (int mt = 0; mt < G::MT; ++mt) acc[ct][mt] *= f;
            }
          }
        }
        // norms of the wave's tokens, eight consecutive ones per K-step of the values
        h8 nk[KV], nv[KV];
#pragma unroll
        for (int ks = 0; ks < KV; ++ks) {
          const uint16_t* np = reinterpret_cast<const uint16_t*>(lds + C::n_off) + w0 + 32 * (KV * hf + ks) + 8 * g;
          nk[ks] = *reinterpret_cast<const h8*>(np);
          nv[ks] = *reinterpret_cast<const h8*>(np + G::CH);
        }
        // scores less the row's maximum and gs, so that p 2^-gs = 2^x. masked: some of the chunk's
        // tokens are nodes, seen by their descendants only, or lie past the sequence; a value norm
        // that is not finite there makes the rows that see it NaN and no other
        const float gsf = float(gs);
        float x[NCT][KV][8], top[NCT];
        auto scores = [&](auto masked) {
          constexpr bool MASK = decltype(masked)::value;
          bool bad[KV][8];
          if constexpr (MASK) {
#pragma unroll
            for (int ks = 0; ks < KV; ++ks)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float v = float(nv[ks][j]);
                bad[ks][j] = !(fabsf(v) < INFINITY);
                if (bad[ks][j]) nv[ks][j] = _Float16(0.f);
              }
          }
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
            uint32_t seen[KV];  // bit j: token 8 g + j of the K-step
            if constexpr (MASK) {
              int row = r0 + 16 * ct + c;
              asm volatile("" : "+v"(row));  // not ahead of the loop: once per split
              const int node = row / a.n_rep;
              uint64_t word;
              if constexpr (WIN) {
                const int p = hist + node, from = max(max(p, 0) - a.window + 1, 0);
                word = node < a.T ? tree_below(p - c0 + 1) & (~tree_below(from - c0) | tree_below(a.sinks - c0)) : 0;
              } else {
                const uint64_t vis = node < a.T ? a.vis[int64_t(b) * a.T + node] : 0;
                const int at = hist - c0;  // the tree's first position in the chunk (or before it)
                word = at >= 0 ? (vis << at | ((uint64_t(1) << at) - 1)) : at > -64 ? vis >> -at : 0;
              }
#pragma unroll
              for (int ks = 0; ks < KV; ++ks) seen[ks] = uint32_t(word >> (w0 + 32 * (KV * hf + ks) + 8 * g)) & 0xffu;
            }
            const float m0 = (m[ct] == -INFINITY ? 0.f : m[ct]) + gsf;
            top[ct] = -INFINITY;
#pragma unroll
            for (int ks = 0; ks < KV; ++ks)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                float y = fmaf(d[ct][2 * ks + (j >> 2)][j & 3] * sc[ct], float(nk[ks][j]), -m0);
                if (MASK) y = !(seen[ks] >> j & 1) ? -INFINITY : bad[ks][j] ? __builtin_nanf("") : y;
                x[ct][ks][j] = y;
                top[ct] = fmaxf(top[ct], y);
              }
          }
        };
        bool whole = c0 + G::CH <= hist;  // every row sees the chunk
        if constexpr (WIN) whole = c0 + G::CH <= ws.p_lo + 1 && (c0 > ws.p_hi - a.window || c0 + G::CH <= a.sinks);
        if (whole) scores(std::integral_constant<bool, false>{});
        else scores(std::integral_constant<bool, true>{});
        // a row's maximum moves when a score exceeds it by more than kTreeRescale, and on its first key
        bool move[NCT], any = false;
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
          top[ct] = tree_max16(top[ct]) + gsf;
          move[ct] = top[ct] > kTreeRescale || (m[ct] == -INFINITY && top[ct] > -INFINITY);
          any = any || move[ct];
        }
        if (__any(any)) {
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) {
            const bool fresh = m[ct] == -INFINITY;
            const float shift = move[ct] ? top[ct] : 0.f;
            const float alpha = move[ct] ? (fresh ? 0.f : __builtin_amdgcn_exp2f(-top[ct])) : 1.f;
            m[ct] = move[ct] ? (fresh ? 0.f : m[ct]) + top[ct] : m[ct];
            l[ct] *= alpha;
#pragma unroll
            for (int mt = 0; mt < G::MT; ++mt) acc[ct][mt] *= alpha;
#pragma unroll
            for (int ks = 0; ks < KV; ++ks)
#pragma unroll
              for (int j = 0; j < 8; ++j) x[ct][ks][j] -= shift;
          }
        }
        // weights p n_V 2^-gs (l sums p 2^-gs)
        h8 ph[NCT][KV], pl[EX ? NCT : 1][EX ? KV : 1];
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
          for (int ks = 0; ks < KV; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float p = __builtin_amdgcn_exp2f(x[ct][ks][j]);
              l[ct] += p;
              float w = p * float(nv[ks][j]);
              // one rounded product for both terms: fused with the conversion (which rounds the exact
              // product) the high term could differ from the one that the low term makes up for
              if constexpr (EX) asm("" : "+v"(w));
              ph[ct][ks][j] = _Float16(w);
              if constexpr (EX) pl[ct][ks][j] = _Float16(w - float(ph[ct][ks][j]));
            }
        __builtin_amdgcn_sched_barrier(0);
        // values: A row c of M-tile mt = dim 16 mt + c, k-slots of lane group g = tokens 32 ks + 8 g .. + 7
        constexpr int MP = G::MT > 1 ? 2 : 1;  // M-tiles at a time, as above
#pragma unroll
        for (int m0 = 0; m0 < G::MT; m0 += MP)
#pragma unroll
          for (int ks = 0; ks < KV; ++ks) {
            h8 vh[MP], vl[MP];
#pragma unroll
            for (int i = 0; i < MP; ++i) {
              const char* vp = lds + v_addr(m0 + i, KV * hf + ks);
              vh[i] = *reinterpret_cast<const h8*>(vp);
              if constexpr (EX) vl[i] = *reinterpret_cast<const h8*>(vp + G::VT);
            }
            auto products = [&](const h8 (&x)[MP], const auto& y) {
#pragma unroll
              for (int i = 0; i < MP; ++i)
#pragma unroll
                for (int ct = 0; ct < NCT; ++ct)
                  acc[ct][m0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i], y[ct][ks], acc[ct][m0 + i], 0, 0, 0);
            };
            products(vh, ph);
            if constexpr (EX) {
              products(vl, ph);
              products(vh, pl);
            }
          }
        }
      };
      for (int ch = ch_lo; ch < ch_hi; ch += AHEAD) {
        chunk(even, ch);
        if (AHEAD == 2 && ch + 1 < ch_hi) chunk(odd, ch + 1);
      }
    }

    const float f = ldexpf(1.f, gs - 8), lf = ldexpf(1.f, gs);
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      l[ct] *= lf;
      l[ct] += __shfl_xor(l[ct], 16, 64);
      l[ct] += __shfl_xor(l[ct], 32, 64);
#pragma unroll
      for (int mt = 0; mt < G::MT; ++mt) acc[ct][mt] *= f;
    }
    if constexpr (TG == 2) {  // the second token group's waves hand over to the first's
      float* o = reinterpret_cast<float*>(lds) + (rg * 16 + c) * (D + 2);
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        __syncthreads();  // the tiles, or what was handed over before, are read
        if (tg == 1) {
#pragma unroll
          for (int mt = 0; mt < G::MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[16 * mt + 4 * g + i] = acc[ct][mt][i];
          if (g == 0) {
            o[D] = m[ct];
            o[D + 1] = l[ct];
          }
        }
        __syncthreads();
        if (tg == 0) {
          const float m1 = o[D], l1 = o[D + 1], M = fmaxf(m[ct], m1);
          const float w0 = m[ct] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[ct] - M);
          const float w1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - M);
          m[ct] = M;
          l[ct] = l[ct] * w0 + l1 * w1;
#pragma unroll
          for (int mt = 0; mt < G::MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[ct][mt][i] = acc[ct][mt][i] * w0 + o[16 * mt + 4 * g + i] * w1;
        }
      }
    }
    // items of 16 rows: ((b Hkv + kvh) nsplit + s) nrp / 16 + row block
    if (tg == 0 && r0 < rows) {
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        const int64_t item = ((int64_t(b) * a.Hkv + kvh) * a.nsplit + s) * (a.nrp / 16) + r0 / 16 + ct;
        float* o = a.part_acc + (item * 16 + c) * D + 4 * g;
#pragma unroll
        for (int mt = 0; mt < G::MT; ++mt) *reinterpret_cast<f32x4*>(o + 16 * mt) = acc[ct][mt];
        if (g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * (item * 16 + c)) = make_float2(m[ct], l[ct]);
      }
    }
    __syncthreads();  // the tiles and what was handed over are read
  }
}

// 16 rows times a D x D matrix on v_mfma_f32_16x16x4f32, a tile of 16 columns a wave: K-step (s, e),
// slot g is column 16 s + 4 g + e of the rows. mat(j, k4) gives rows k4 .. k4 + 3 of column j; the
// operands are loaded ahead of the rows, whose loads they hide behind. Lane 16 g + c ends with
// columns 16 wave + 4 g .. + 3 of row c.
template <int D>
struct TreeProduct {
  f32x4 m[D / 16];
  template <class Mat>
  __device__ __forceinline__ void load(int wave, int lane, Mat&& mat) {
    if (wave >= D / 16) return;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) m[s] = mat(16 * wave + (lane & 15), 16 * s + 4 * (lane >> 4));
  }
  // x: LDS, row c's D floats (16-byte aligned)
  __device__ __forceinline__ f32x4 run(const float* x, int lane) const {
    f32x4 y[2] = {};
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const f32x4 bv = *reinterpret_cast<const f32x4*>(x + 16 * s + 4 * (lane >> 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) y[s & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[s][e], bv[e], y[s & 1], 0, 0, 0);
    }
    return y[0] + y[1];
  }
};

__host__ __device__ constexpr int tree_rotate_threads(int D) { return 4 * D > 256 ? 4 * D : 256; }

// q' of sixteen rows per work-group (rows past n_rep T: zero, up to a multiple of 32), and the nodes' words.
// Products in fp32. Bound by latency and, with many tiles, by the instructions around 32 matrix
// products: 5.5 us for 16 tiles, 14 us for 2,048 (64 heads, 64 nodes, 4 sequences: 12 MB moved).
// WIN: no nodes' words.
template <int D, bool WIN = false>
__global__ __launch_bounds__(tree_rotate_threads(D)) void tree_rotate_kernel(TreeRotArgs a) {
  constexpr int XS = D + 4, NTHR = tree_rotate_threads(D);
  __shared__ __align__(16) float x[16 * XS];
  __shared__ __align__(16) float y[16 * XS];
  __shared__ int par[64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tiles = a.nrp / 16;
  const int64_t unit = blockIdx.x / tiles;  // b Hkv + kvh
  const int r0 = 16 * int(blockIdx.x % tiles), kvh = int(unit % a.Hkv), rows = a.n_rep * a.T;
  const int64_t b = unit / a.Hkv;
  if (r0 >= (rows + 31) / 32 * 32) return;  // of no wave that computes
  const bool words = !WIN && kvh == 0 && r0 == 0;  // one work-group per sequence
  TreeProduct<D> pi;
  pi.load(wave, lane, [&](int j, int k) { return *reinterpret_cast<const f32x4*>(a.pi + j * D + k); });
  if (words && tid < 64) par[tid] = tid < a.T ? a.parents[b * a.psb + tid] : -1;
  // a thread's share of a row by 16 bytes where q is laid out for it (a.vec)
  const auto fetch = [&](auto vec, auto&& load) {
    constexpr int V = decltype(vec)::value, PER = D / V;  // elements a load, loads a row
#pragma unroll
    for (int i0 = 0; i0 < 16 * PER; i0 += NTHR) {
      const int i = i0 + tid, r = r0 + i / PER, d = V * (i % PER);
      if (16 * PER % NTHR != 0 && i >= 16 * PER) break;
      float v[V] = {};
      if (r < rows) load(b * a.qsb + (kvh * a.n_rep + r % a.n_rep) * a.qsh + (r / a.n_rep) * a.qsq + d, v);
#pragma unroll
      for (int e = 0; e < V; ++e) x[(i / PER) * XS + d + e] = v[e];
    }
  };
  const auto words16 = [&](auto vec, auto&& value) {
    fetch(vec, [&](int64_t o, float (&v)[decltype(vec)::value]) {
      constexpr int V = decltype(vec)::value;
      uint16_t h[V];
      __builtin_memcpy(h, __builtin_assume_aligned(static_cast<const uint16_t*>(a.q) + o, 2 * V), 2 * V);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = value(h[e]);
    });
  };
  const auto words32 = [&](auto vec) {
    fetch(vec, [&](int64_t o, float (&v)[decltype(vec)::value]) {
      constexpr int V = decltype(vec)::value;
      __builtin_memcpy(v, __builtin_assume_aligned(static_cast<const float*>(a.q) + o, 4 * V), 4 * V);
    });
  };
  constexpr std::integral_constant<int, 1> one;
  constexpr std::integral_constant<int, 4> four;
  constexpr std::integral_constant<int, 8> eight;
  const auto bf16 = [](uint16_t h) { return bf16_to_f32(h); };
  const auto fp16 = [](uint16_t h) { return f16_to_f32(h); };
  if (a.vec) {
    if (a.q_dtype == WN_F32) words32(four);
    else if (a.q_dtype == WN_BF16) words16(eight, bf16);
    else words16(eight, fp16);
  } else {
    if (a.q_dtype == WN_F32) words32(one);
    else if (a.q_dtype == WN_BF16) words16(one, bf16);
    else words16(one, fp16);
  }
  __syncthreads();
  if (words && tid < a.T) {
    // a parent comes before its child: any other value ends the walk, as -1 does
    uint64_t w = uint64_t(1) << tid;
    for (int n = tid, p = par[n]; p >= 0 && p < n; n = p, p = par[n]) w |= uint64_t(1) << p;
    a.vis[b * a.T + tid] = w;
  }
  const int g = lane >> 4, c = lane & 15;
  if (wave < D / 16) *reinterpret_cast<f32x4*>(y + c * XS + 16 * wave + 4 * g) = pi.run(x + c * XS, lane);
  __syncthreads();
  if (a.qf) {
#pragma unroll
    for (int i = 4 * tid; i < 16 * D; i += 4 * NTHR) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(y + (i / D) * XS + i % D) * a.scale;
      *reinterpret_cast<f32x4*>(a.qf + (unit * a.nrp + r0 + i / D) * D + i % D) = v;
    }
    return;
  }
  // sixteen threads a row: its largest magnitude, then the fp16 terms of q' 2^e (below 2^15)
  if (tid >= 256) return;
  constexpr int DPT = D / 16;
  const int r = tid >> 4, k = tid & 15;
  float v[DPT], top = 0.f;
  __builtin_memcpy(v, __builtin_assume_aligned(y + r * XS + DPT * k, DPT < 4 ? 4 * DPT : 16), 4 * DPT);
#pragma unroll
  for (int d = 0; d < DPT; ++d) top = fmaxf(top, fabsf(v[d]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 16));
  int qe;
  frexpf(fminf(top, 3.0e38f), &qe);
  const int e = min(15 - qe, 120);
  const float up = ldexpf(1.f, e);
  const int64_t row = unit * a.nrp + r0 + r;
  if (k == 0) a.qs[row] = ldexpf(a.scale, -(e + 8));
  _Float16 h[DPT], l[DPT];
#pragma unroll
  for (int d = 0; d < DPT; ++d) {
    const float t = v[d] * up;
    h[d] = _Float16(t);
    l[d] = _Float16(t - float(h[d]));
  }
  constexpr int AL = 2 * DPT < 16 ? 2 * DPT : 16;
  __builtin_memcpy(__builtin_assume_aligned(a.qh + row * D + DPT * k, AL), h, 2 * DPT);
  if (a.exact) __builtin_memcpy(__builtin_assume_aligned(a.ql + row * D + DPT * k, AL), l, 2 * DPT);
}

// R rows per work-group of 16 waves, 16 / R waves a row: the splits' partials merged (weights
// 2^(m_s - max m)), divided by the sum, times Pi_V, cast. A row that saw no key is 0. The statistics
// come a split to a lane, the accumulators a split to a load, eight (R = 4) or four in flight; the first of
// both, and Pi_V's operands, are asked for before anything is known of the sequence: what bounds
// these few rows is one round trip after another: 6 us for 256 rows, 18 us for 16,384 of three
// splits (two round trips and the product for each of 1,024 work-groups, of which 512 run at a time).
template <int D, int R, bool WIN = false>
__global__ __launch_bounds__(1024) void tree_merge_kernel(std::conditional_t<WIN, WindowMergeArgs, TreeMergeArgs> a) {
  constexpr int XS = D + 4, LD = D < 64 ? D : 64, VEC = D / LD;  // lanes a split, dims a lane
  constexpr int SUB = 64 / LD, PARTS = 16 / R * SUB;              // splits are taken in PARTS residue classes
  constexpr int U = R == 4 ? 8 : 4;
  __shared__ __align__(16) float x[PARTS][R][XS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = a.n_rep * a.T, blocks = (rows + R - 1) / R;
  const int64_t unit = blockIdx.x / blocks;
  const int blk = int(blockIdx.x % blocks);
  const int r = wave % R, part = wave / R * SUB + lane / LD, d0 = VEC * (lane % LD);
  const int64_t first = unit * a.nsplit * a.nrp + min(blk * R + r, rows - 1);
  const auto stats = [&](int s) { return *reinterpret_cast<const float2*>(a.part_ml + 2 * (first + int64_t(min(s, a.nsplit - 1)) * a.nrp)); };
  float v[U][VEC];
  const auto fetch = [&](int s0) {  // splits s0 + part, s0 + PARTS + part, ...
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const float* p = a.part_acc + (first + int64_t(min(s0 + PARTS * j + part, a.nsplit - 1)) * a.nrp) * D + d0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j][e] = p[e];
    }
  };
  const float2 ml0 = stats(lane);
  fetch(0);
  TreeProduct<D> pi;
  pi.load(wave, lane, [&](int j, int kk) {
    return f32x4{a.pi_v[kk * D + j], a.pi_v[(kk + 1) * D + j], a.pi_v[(kk + 2) * D + j], a.pi_v[(kk + 3) * D + j]};
  });
  const int L = min(max(a.seq_lens[unit / a.Hkv], 0), a.max_len);
  int live;  // splits that the sequence has: the others' partials are not its own
  if constexpr (WIN) {
    const WindowSpan ws = window_span(L, a.T, a.n_rep, blk * R / a.rows_block * a.rows_block, a.rows_block, a.chunk, a.window, a.sinks,
                                      a.nsplit, a.span);
    live = ws.span ? (ws.total + ws.span - 1) / ws.span : 0;
  } else {
    live = tree_count(L, tree_span(L, a.nsplit, a.span));
  }
  float M = lane < live ? ml0.x : -INFINITY;
  for (int s = 64 + lane; s < live; s += 64) M = fmaxf(M, stats(s).x);
  M = wave_max(M);
  if (M == -INFINITY) M = 0.f;  // no split saw a key: every weight is 0
  float den = 0.f, num[VEC] = {};
  for (int s0 = 0; s0 < live; s0 += 64) {
    const float2 ml = s0 ? stats(s0 + lane) : ml0;
    const bool own = s0 + lane < live;
    const float w = own ? __builtin_amdgcn_exp2f(ml.x - M) : 0.f;  // split s0 + lane's; 0 for one that saw no key
    den = own ? fmaf(w, ml.y, den) : den;
    const int n = min(64, live - s0);
    for (int i = 0; i < n; i += U * PARTS) {
      if (s0 + i) fetch(s0 + i);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int s = i + PARTS * j + part;
        const float ws = __shfl(w, s & 63, 64);
#pragma unroll
        for (int e = 0; e < VEC; ++e) num[e] = s < n ? fmaf(ws, v[j][e], num[e]) : num[e];
      }
    }
  }
  den = wave_sum(den);
  const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
  for (int e = 0; e < VEC; ++e) x[part][r][d0 + e] = num[e] * inv;
  __syncthreads();
  if constexpr (PARTS > 1) {
    for (int i = tid; i < R * D; i += 1024) {
      float t = 0.f;
#pragma unroll
      for (int q = 0; q < PARTS; ++q) t += x[q][i / D][i % D];
      x[0][i / D][i % D] = t;
    }
    __syncthreads();
  }
  const int g = lane >> 4, c = lane & 15, rr = R * blk + c;
  if (wave >= D / 16) return;
  const f32x4 y = pi.run(x[0][c % R], lane);
  if (c >= R || rr >= rows) return;
  const int kvh = int(unit % a.Hkv), Hq = a.Hkv * a.n_rep;
  const int64_t b = unit / a.Hkv;
  const int64_t o = ((b * Hq + kvh * a.n_rep + rr % a.n_rep) * a.T + rr / a.n_rep) * D + 16 * wave + 4 * g;
  if (a.out_dtype == WN_F32) {
    __builtin_memcpy(static_cast<float*>(a.out) + o, &y, 16);
  } else {
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = a.out_dtype == WN_BF16 ? f32_to_bf16(y[i]) : f32_to_f16(y[i]);
    __builtin_memcpy(static_cast<uint16_t*>(a.out) + o, h, 8);
  }
}

template <bool WIN>
using TreeArgsOf = std::conditional_t<WIN, WindowArgs, TreeArgs>;
template <bool WIN>
using TreeKernelSet = std::conditional_t<WIN, TreeKernelsOf<WindowArgs, WindowMergeArgs>, TreeKernels>;

template <int D, bool EX, int NCT, int RG, int TG, int W, bool WIN>
TreeScanOf<TreeArgsOf<WIN>> tree_scan() {
  using C = TreeCfg<D, EX, NCT, RG, TG>;
  return {tree_scan_kernel<D, EX, NCT, RG, TG, W, WIN>, C::ROWS, C::NTHR, C::tab_off, W == 4 && !EX ? 2 * kPairBytes : 0, C::give, 0};
}

template <int D, bool EX, int W, bool WIN>
TreeKernelSet<WIN> tree_kernels() {
  TreeKernelSet<WIN> k;
  if constexpr (D == 256) {
    // 128 accumulator registers per 32 rows: sixteen rows a wave
    k.scan[0] = k.scan[1] = k.scan[2] = k.scan[3] = tree_scan<D, EX, 1, 4, 1, W, WIN>();
  } else {
    k.scan[0] = tree_scan<D, EX, 1, 2, 2, W, WIN>();
    k.scan[1] = tree_scan<D, EX, 2, 2, 2, W, WIN>();
    // More than 64 rows: blocks of 128, which decode a chunk once for all of them. With two terms a
    // factor decoding writes twice the bytes, and eight waves share it (64 query heads, 64 nodes, 4 and
    // 6 bits, in traces: 605 us, two work-groups of four waves and 64 rows 710; a second set of tiles, to decode
    // ahead of the barrier, 600). With single terms four waves take 128 rows, and a second work-group
    // fills their waits (28 heads, 26 nodes: 41 us, eight waves 47).
    if constexpr (EX) k.scan[2] = tree_scan<D, EX, 2, 4, 2, W, WIN>();
    else k.scan[2] = tree_scan<D, EX, 2, 4, 1, W, WIN>();
    if constexpr (WIN) k.scan[3] = tree_scan<D, EX, 2, 8, 1, W, WIN>();
  }
  k.rotate = tree_rotate_kernel<D, WIN>;
  k.merge[0] = tree_merge_kernel<D, 4, WIN>;
  if constexpr (!WIN) k.merge[1] = tree_merge_kernel<D, 16, WIN>;
  k.rotate_threads = tree_rotate_threads(D);
  return k;
}

// Kernels for 4-bit K and V, the width that most caches take, and for any widths.
template <int D, bool WIN = false>
TreeKernelSet<WIN> tree_kernels_for(bool exact, int bw_k, int bw_v) {
  if (bw_k == 4 && bw_v == 4) return exact ? tree_kernels<D, true, 4, WIN>() : tree_kernels<D, false, 4, WIN>();
  return exact ? tree_kernels<D, true, 0, WIN>() : tree_kernels<D, false, 0, WIN>();
}

}  // namespace
}  // namespace wn
