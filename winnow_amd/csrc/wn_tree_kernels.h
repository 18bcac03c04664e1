// The kernels of the tree attention (wn_tree.h), templates on the head dim.
#pragma once

#include "wn_tree.h"

namespace wn {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kTreeCb = 256.0f;      // codebook values are scaled by 2^8
constexpr float kTreeRescale = 8.0f;   // a maximum moves when a score exceeds it by more
constexpr int kTreeNoScale = -64;      // value scale before the first norm

template <int D>
struct TreeGeo {
  static constexpr int DP = D < 32 ? 32 : D;        // K dims, padded to one K-step
  static constexpr int KS = DP / 32, MT = D / 16;   // score K-steps, value M-tiles
  static constexpr int CH = D == 256 ? 32 : 64;     // tokens per chunk
  static constexpr int KROW = 2 * DP + 16;          // bytes of a K tile row: 16 rows in 16 bank quads
  static constexpr int VROW = 2 * CH + 16;          // bytes of a V tile row
  static constexpr int KT = CH * KROW, VT = D * VROW;
};

// Token of row c of score tile t.
__device__ __forceinline__ int tree_tok(int t, int c) { return 32 * (t >> 1) + 8 * (c >> 2) + 4 * (t & 1) + (c & 3); }

// The raw words of one group of eight codes: the up to two 4-byte words that hold bytes
// [o, o + bw) of a block; a word without any of them is not read.
struct TreeRaw {
  uint32_t lo, hi;
};
__device__ __forceinline__ TreeRaw tree_raw(const uint8_t* block, uint32_t o, int bw) {
  const uint32_t a = o & ~3u, b = (o + uint32_t(bw) - 1) & ~3u;
  return TreeRaw{*reinterpret_cast<const uint32_t*>(block + a), *reinterpret_cast<const uint32_t*>(block + b)};
}

// Table entries (high | low << 16) of the eight codes of a group that starts at byte o.
template <int BW>
__device__ __forceinline__ void tree_entries(TreeRaw r, uint32_t o, const char* tab, uint32_t lane, uint32_t (&e)[8]) {
  constexpr int COP = tree_copies(BW);
  const uint32_t own = (lane & uint32_t(COP - 1)) << 2, sh = 8 * (o & 3);
  const uint64_t w = (uint64_t(r.hi) << 32 | r.lo) >> sh;
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

template <class F>
__device__ __forceinline__ void tree_by_width(int bw, F&& f) {
  switch (bw) {  // wave-uniform
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 3: f(std::integral_constant<int, 3>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    case 5: f(std::integral_constant<int, 5>{}); break;
    case 6: f(std::integral_constant<int, 6>{}); break;
    default: f(std::integral_constant<int, 8>{}); break;
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

template <int D, bool EX, int NCT, int RG, int TG>
struct TreeCfg {
  using G = TreeGeo<D>;
  static constexpr int NW = RG * TG, NTHR = 64 * NW, ROWS = 16 * NCT * RG;
  static constexpr int NTW = G::CH / 16 / TG;  // score tiles of a wave
  static constexpr int PL = EX ? 2 : 1;        // planes of a tile
  static constexpr int KI = G::CH * D / 8, VI = KI / 2;                        // dequantization items of a chunk
  static constexpr int NK = (KI + NTHR - 1) / NTHR, NV = (VI + NTHR - 1) / NTHR;
  static constexpr int k_off = 0, v_off = k_off + PL * G::KT, n_off = v_off + PL * G::VT;
  static constexpr int tab_off = n_off + 4 * G::CH;  // norms: K then V, fp16
  // the waves of token group 1 hand over (acc, m, l) in the tiles' place
  static_assert(TG == 1 || RG * NCT * 16 * (D + 2) * 4 <= tab_off, "hand-over of the token groups fits");
  static_assert(NTW % 2 == 0 && tab_off % 16 == 0, "whole value K-steps");
};

template <int D, bool EX, int NCT, int RG, int TG>
__global__ __launch_bounds__(64 * RG * TG) void tree_scan_kernel(TreeArgs a) {
  using C = TreeCfg<D, EX, NCT, RG, TG>;
  using G = TreeGeo<D>;
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int wig = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rg = wig % RG, tg = wig / RG;
  char* tabk = lds + C::tab_off;
  char* tabv = tabk + tree_table_bytes(a.bwk);
  tree_stage_table<C::NTHR>(a.cb_k, a.bwk, tabk, tid);
  tree_stage_table<C::NTHR>(a.cb_v, a.bwv, tabv, tid);
  if constexpr (D < G::DP) {  // the padded dims of the K tile stay zero
    for (int i = tid; i < C::PL * G::KT / 4; i += C::NTHR) reinterpret_cast<uint32_t*>(lds + C::k_off)[i] = 0;
  }

  // unit: ((b Hkv + kvh) nsplit + s) ncg + row block of ROWS
  int u = blockIdx.x;
  const int cg = u % a.ncg;
  u /= a.ncg;
  const int s = u % a.nsplit;
  u /= a.nsplit;
  const int kvh = u % a.Hkv, b = u / a.Hkv;
  const int L = min(max(const_view(a.seq_lens)[b], 0), a.max_pages << a.log2S);
  const int hist = L - a.T;  // position of node 0
  const int nch = (L + G::CH - 1) / G::CH;
  const int ch_lo = int(int64_t(nch) * s / a.nsplit), ch_hi = int(int64_t(nch) * (s + 1) / a.nsplit);
  const int r0 = cg * C::ROWS + rg * 16 * NCT;  // the wave's first row
  const int64_t row0 = (int64_t(b) * a.Hkv + kvh) * a.nrp + r0;

  f32x4 acc[NCT][G::MT];
  float m[NCT], l[NCT], sc[NCT];
  uint64_t vis[NCT];
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
    const int node = (r0 + 16 * ct + c) / a.n_rep;
    vis[ct] = node < a.T ? a.vis[int64_t(b) * a.T + node] : 0;
#pragma unroll
    for (int k = 0; k < G::KS; ++k) {
      const bool pad = D < 32 && g >= D / 8;  // dims past D
      qh[ct][k] = pad ? h8{} : *reinterpret_cast<const h8*>(a.qh + row * D + 32 * k + 8 * g);
      if constexpr (EX) ql[ct][k] = pad ? h8{} : *reinterpret_cast<const h8*>(a.ql + row * D + 32 * k + 8 * g);
    }
  }

  if (ch_lo < ch_hi) {
    const int t_hi = min(G::CH * ch_hi, L), col_hi = (t_hi - 1) >> a.log2S, smask = (1 << a.log2S) - 1;
    const int32_t* trow = a.table + int64_t(b) * a.tsb;
    const uint32_t nbk = uint32_t(D * a.bwk / 8), nbv = uint32_t(D * a.bwv / 8), last_page = uint32_t(a.num_pages - 1);
    // tokens past the range read its last page (and are masked): every address is one of the pool
    auto page_of = [&](int t) { return int64_t(min(uint32_t(trow[min(t >> a.log2S, col_hi)]), last_page)); };

    TreeRaw kr[C::NK], vr[C::NV][2];
    uint16_t nr = 0;
    auto load = [&](int c0) {
#pragma unroll
      for (int j = 0; j < C::NK; ++j) {
        const int it = min(tid + C::NTHR * j, C::KI - 1), tok = it / (D / 8), dg = it % (D / 8);
        const int t = c0 + tok;
        kr[j] = tree_raw(a.k_pages + page_of(t) * a.ksp + kvh * a.ksh, uint32_t(t & smask) * nbk + uint32_t(dg * a.bwk), a.bwk);
      }
#pragma unroll
      for (int j = 0; j < C::NV; ++j) {
        const int it = min(tid + C::NTHR * j, C::VI - 1), tp = it % (G::CH / 2), dg = it / (G::CH / 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = c0 + 2 * tp + h;
          vr[j][h] = tree_raw(a.v_pages + page_of(t) * a.vsp + kvh * a.vsh, uint32_t(t & smask) * nbv + uint32_t(dg * a.bwv), a.bwv);
        }
      }
      if (tid < 2 * G::CH) {
        const int t = c0 + tid % G::CH;
        const int64_t pid = page_of(t);
        const uint16_t* p = tid < G::CH ? a.k_norms + pid * a.knp + kvh * a.knh : a.v_norms + pid * a.vnp + kvh * a.vnh;
        nr = t < t_hi ? p[t & smask] : uint16_t(0);  // what lies past the sequence may hold anything
      }
    };
    auto store = [&](int c0) {
      tree_by_width(a.bwk, [&](auto bw) {
        constexpr int BW = decltype(bw)::value;
#pragma unroll
        for (int j = 0; j < C::NK; ++j) {
          const int it = tid + C::NTHR * j;
          if (C::KI % C::NTHR && it >= C::KI) break;
          const int tok = it / (D / 8), dg = it % (D / 8);
          uint32_t e[8];
          tree_entries<BW>(kr[j], uint32_t((c0 + tok) & smask) * nbk + uint32_t(dg * BW), tabk, lane, e);
          char* dst = lds + C::k_off + tok * G::KROW + 16 * dg;
          *reinterpret_cast<u32x4*>(dst) = u32x4{pack_lo(e[0], e[1]), pack_lo(e[2], e[3]), pack_lo(e[4], e[5]), pack_lo(e[6], e[7])};
          if constexpr (EX)
            *reinterpret_cast<u32x4*>(dst + G::KT) = u32x4{pack_hi(e[0], e[1]), pack_hi(e[2], e[3]), pack_hi(e[4], e[5]), pack_hi(e[6], e[7])};
        }
      });
      tree_by_width(a.bwv, [&](auto bw) {
        constexpr int BW = decltype(bw)::value;
#pragma unroll
        for (int j = 0; j < C::NV; ++j) {
          const int it = tid + C::NTHR * j;
          if (C::VI % C::NTHR && it >= C::VI) break;
          const int tp = it % (G::CH / 2), dg = it / (G::CH / 2);
          uint32_t e0[8], e1[8];
          const int t = c0 + 2 * tp;
          tree_entries<BW>(vr[j][0], uint32_t(t & smask) * nbv + uint32_t(dg * BW), tabv, lane, e0);
          tree_entries<BW>(vr[j][1], uint32_t((t + 1) & smask) * nbv + uint32_t(dg * BW), tabv, lane, e1);
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            char* dst = lds + C::v_off + (8 * dg + d) * G::VROW + 4 * tp;
            *reinterpret_cast<uint32_t*>(dst) = pack_lo(e0[d], e1[d]);
            if constexpr (EX) *reinterpret_cast<uint32_t*>(dst + G::VT) = pack_hi(e0[d], e1[d]);
          }
        }
      });
      if (tid < 2 * G::CH) reinterpret_cast<uint16_t*>(lds + C::n_off)[tid] = nr;
    };

    load(G::CH * ch_lo);
    for (int ch = ch_lo; ch < ch_hi; ++ch) {
      const int c0 = G::CH * ch;
      __syncthreads();  // the last chunk's tiles are read (at first: the tables are staged)
      store(c0);
      if (ch + 1 < ch_hi) load(c0 + G::CH);
      __syncthreads();

      // scores of the wave's tokens: register i of tile t is token w0 + tree_tok(t, 4 g + i)
      const int w0 = 16 * C::NTW * tg;
      f32x4 d[NCT][C::NTW];
#pragma unroll
      for (int t = 0; t < C::NTW; ++t) {
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) d[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        const char* kp = lds + C::k_off + (w0 + tree_tok(t, c)) * G::KROW + 16 * g;
#pragma unroll
        for (int k = 0; k < G::KS; ++k) {
          const h8 kh = *reinterpret_cast<const h8*>(kp + 64 * k);
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) d[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[ct][k], d[ct][t], 0, 0, 0);
          if constexpr (EX) {
            const h8 kl = *reinterpret_cast<const h8*>(kp + G::KT + 64 * k);
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
              d[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[ct][k], d[ct][t], 0, 0, 0);
              d[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[ct][k], d[ct][t], 0, 0, 0);
            }
          }
        }
      }
      // norms of the wave's tokens, eight consecutive ones per K-step of the values
      h8 nk[C::NTW / 2], nv[C::NTW / 2];
      uint32_t nmax = 0;
#pragma unroll
      for (int ks = 0; ks < C::NTW / 2; ++ks) {
        const uint16_t* np = reinterpret_cast<const uint16_t*>(lds + C::n_off) + w0 + 32 * ks + 8 * g;
        nk[ks] = *reinterpret_cast<const h8*>(np);
        nv[ks] = *reinterpret_cast<const h8*>(np + G::CH);
#pragma unroll
        for (int j = 0; j < 8; ++j) nmax = max(nmax, min(uint32_t(__builtin_bit_cast(uint16_t, nv[ks][j])) & 0x7fffu, 0x7bffu));
      }
      // value scale: every n_V < 2^(7 + gs), so 2^kTreeRescale n_V 2^-gs < 2^15 in fp16; it
      // follows the norms' magnitude (n_V = 2^-20 keeps its bits)
      {
        int ge;
        const float top = wave_max(f16_to_f32(uint16_t(nmax)));
        frexpf(top, &ge);
        if (top > 0.f && ge - 7 > gs) {  // wave-uniform, rare after the first chunk
          const float f = ldexpf(1.f, max(gs - (ge - 7), -126));
          gs = ge - 7;
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
            for (int mt = 0; mt < G::MT; ++mt) acc[ct][mt] *= f;
        }
      }
      const float vsc = ldexpf(1.f, -gs);
      const bool full = c0 + G::CH <= hist;  // no node among the chunk's tokens

      h8 ph[NCT][C::NTW / 2], pl[EX ? NCT : 1][EX ? C::NTW / 2 : 1];
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        // the chunk's visible tokens: bit j for token c0 + j (positions before the tree, and
        // the node's own word of nodes, shifted to where the tree starts)
        uint32_t seen[C::NTW / 2];
        if (!full) {
          const int at = hist - c0;  // the tree's first position in the chunk (or before it)
          const uint64_t word = at >= 0 ? (vis[ct] << at | ((uint64_t(1) << at) - 1)) : at > -64 ? vis[ct] >> -at : 0;
#pragma unroll
          for (int ks = 0; ks < C::NTW / 2; ++ks) seen[ks] = uint32_t(word >> (w0 + 32 * ks + 8 * g)) & 0xffu;
        }
        const bool fresh = m[ct] == -INFINITY;
        const float m0 = fresh ? 0.f : m[ct];
        float x[C::NTW / 2][8], top = -INFINITY;
#pragma unroll
        for (int ks = 0; ks < C::NTW / 2; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float y = fmaf(d[ct][2 * ks + (j >> 2)][j & 3] * sc[ct], float(nk[ks][j]), -m0);
            if (!full && !(seen[ks] >> j & 1)) y = -INFINITY;
            x[ks][j] = y;
            top = fmaxf(top, y);
          }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const bool move = top > kTreeRescale || (fresh && top > -INFINITY);
        if (__any(move)) {
          const float shift = move ? top : 0.f;
          const float alpha = move ? (fresh ? 0.f : __builtin_amdgcn_exp2f(-top)) : 1.f;
          m[ct] = move ? m0 + top : m[ct];
          l[ct] *= alpha;
#pragma unroll
          for (int mt = 0; mt < G::MT; ++mt) acc[ct][mt] *= alpha;
#pragma unroll
          for (int ks = 0; ks < C::NTW / 2; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[ks][j] -= shift;
        }
#pragma unroll
        for (int ks = 0; ks < C::NTW / 2; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float p = __builtin_amdgcn_exp2f(x[ks][j]);
            l[ct] += p;
            float w = p * (float(nv[ks][j]) * vsc);
            if (!full && !(seen[ks] >> j & 1)) w = 0.f;  // a norm that is not finite reaches no row that does not see it
            const _Float16 h = _Float16(w);
            ph[ct][ks][j] = h;
            if constexpr (EX) pl[ct][ks][j] = _Float16(w - float(h));
          }
      }
      // values: A row c of M-tile mt = dim 16 mt + c, k-slots of lane group g = tokens 32 ks + 8 g .. + 7
#pragma unroll
      for (int mt = 0; mt < G::MT; ++mt) {
        const char* vp = lds + C::v_off + (16 * mt + c) * G::VROW + 2 * (w0 + 8 * g);
#pragma unroll
        for (int ks = 0; ks < C::NTW / 2; ++ks) {
          const h8 vh = *reinterpret_cast<const h8*>(vp + 64 * ks);
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct) acc[ct][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[ct][ks], acc[ct][mt], 0, 0, 0);
          if constexpr (EX) {
            const h8 vl = *reinterpret_cast<const h8*>(vp + G::VT + 64 * ks);
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct) {
              acc[ct][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[ct][ks], acc[ct][mt], 0, 0, 0);
              acc[ct][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[ct][ks], acc[ct][mt], 0, 0, 0);
            }
          }
        }
      }
    }
  }

  const float f = ldexpf(1.f, max(gs, -60) - 8);
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16, 64);
    l[ct] += __shfl_xor(l[ct], 32, 64);
#pragma unroll
    for (int mt = 0; mt < G::MT; ++mt) acc[ct][mt] *= f;
  }
  if constexpr (TG == 2) {  // the second token group's waves hand over to the first's
    __syncthreads();  // the tiles are read
    float* give = reinterpret_cast<float*>(lds) + (rg * NCT * 16) * (D + 2);
    if (tg == 1) {
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        float* o = give + (16 * ct + c) * (D + 2);
#pragma unroll
        for (int mt = 0; mt < G::MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[16 * mt + 4 * g + i] = acc[ct][mt][i];
        if (g == 0) {
          o[D] = m[ct];
          o[D + 1] = l[ct];
        }
      }
    }
    __syncthreads();
    if (tg == 1) return;
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      const float* o = give + (16 * ct + c) * (D + 2);
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
  // items of 16 rows: ((b Hkv + kvh) nsplit + s) nrp / 16 + row block
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    const int64_t item = ((int64_t(b) * a.Hkv + kvh) * a.nsplit + s) * (a.nrp / 16) + r0 / 16 + ct;
    float* o = a.part_acc + (item * 16 + c) * D + 4 * g;
#pragma unroll
    for (int mt = 0; mt < G::MT; ++mt) *reinterpret_cast<f32x4*>(o + 16 * mt) = acc[ct][mt];
    if (g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * (item * 16 + c)) = make_float2(m[ct], l[ct]);
  }
}

// Columns j of 16 rows of x (LDS rows of D + 4 floats) times a D x D matrix on
// v_mfma_f32_16x16x4f32: wave w takes column tiles w, w + 4, ...; K-step (s, e), slot g is
// column 16 s + 4 g + e of x. mat(j, k4) gives rows k4 .. k4 + 3 of column j. Lane 16 g + c
// ends with columns 16 t + 4 g .. + 3 of row c.
template <int D, class Mat, class Out>
__device__ __forceinline__ void tree_rows_product(const float* x, int wave, int lane, Mat&& mat, Out&& out) {
  const int g = lane >> 4, c = lane & 15;
  for (int t = wave; t < D / 16; t += 4) {
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      const f32x4 av = mat(16 * t + c, 16 * s + 4 * g), bv = *reinterpret_cast<const f32x4*>(x + c * (D + 4) + 16 * s + 4 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) y = __builtin_amdgcn_mfma_f32_16x16x4f32(av[e], bv[e], y, 0, 0, 0);
    }
    out(t, y);
  }
}

// q' of sixteen rows per work-group (rows past n_rep T: zero), and the nodes' words.
template <int D>
__global__ __launch_bounds__(256) void tree_rotate_kernel(TreeRotArgs a) {
  constexpr int XS = D + 4;
  __shared__ __align__(16) float x[16 * XS];
  __shared__ __align__(16) float y[16 * XS];
  __shared__ int par[64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tiles = a.nrp / 16;
  const int64_t unit = blockIdx.x / tiles;  // b Hkv + kvh
  const int r0 = 16 * int(blockIdx.x % tiles), kvh = int(unit % a.Hkv), rows = a.n_rep * a.T;
  const int64_t b = unit / a.Hkv;
  const bool words = kvh == 0 && r0 == 0;  // one work-group per sequence
  if (words && tid < 64) par[tid] = tid < a.T ? a.parents[b * a.psb + tid] : -1;
  for (int i = tid; i < 16 * D; i += 256) {
    const int r = r0 + i / D, d = i % D;
    float v = 0.f;
    if (r < rows) v = load_elem(a.q, b * a.qsb + (kvh * a.n_rep + r % a.n_rep) * a.qsh + (r / a.n_rep) * a.qsq + d, a.q_dtype);
    x[(i / D) * XS + d] = v;
  }
  __syncthreads();
  if (words && tid < a.T) {
    // a parent comes before its child: any other value ends the walk, as -1 does
    uint64_t w = uint64_t(1) << tid;
    for (int n = tid, p = par[n]; p >= 0 && p < n; n = p, p = par[n]) w |= uint64_t(1) << p;
    a.vis[b * a.T + tid] = w;
  }
  const int g = lane >> 4, c = lane & 15;
  tree_rows_product<D>(
      x, wave, lane, [&](int j, int k) { return *reinterpret_cast<const f32x4*>(a.pi + j * D + k); },
      [&](int t, f32x4 v) { *reinterpret_cast<f32x4*>(y + c * XS + 16 * t + 4 * g) = v; });
  __syncthreads();
  // sixteen threads a row: its largest magnitude, then the fp16 terms of q' 2^e (below 2^15)
  const int r = tid >> 4, k = tid & 15;
  float top = 0.f;
#pragma unroll
  for (int d = k; d < D; d += 16) top = fmaxf(top, fabsf(y[r * XS + d]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 16));
  int qe;
  frexpf(fminf(top, 3.0e38f), &qe);
  const int e = min(15 - qe, 120);
  const float up = ldexpf(1.f, e);
  const int64_t row = unit * a.nrp + r0 + r;
  if (k == 0) a.qs[row] = ldexpf(a.scale, -(e + 8));
#pragma unroll
  for (int d = k; d < D; d += 16) {
    const float v = y[r * XS + d] * up;
    const _Float16 h = _Float16(v);
    a.qh[row * D + d] = h;
    if (a.exact) a.ql[row * D + d] = _Float16(v - float(h));
  }
}

// Sixteen rows per work-group: the splits' partials merged (weights 2^(m_s - max m)),
// divided by the sum, times Pi_V, cast. A row that saw no key is 0.
template <int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeMergeArgs a) {
  constexpr int XS = D + 4, DPT = D / 16;  // dims per thread
  __shared__ __align__(16) float x[16 * XS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tiles = a.nrp / 16;
  const int64_t unit = blockIdx.x / tiles;
  const int blk = int(blockIdx.x % tiles), rows = a.n_rep * a.T;
  const int r = tid >> 4, k = tid & 15;
  const int64_t first = (unit * a.nsplit * tiles + blk) * 16 + r, step = int64_t(tiles) * 16;
  float M = -INFINITY;
  for (int s = 0; s < a.nsplit; ++s) M = fmaxf(M, a.part_ml[2 * (first + s * step)]);
  float den = 0.f, num[DPT];
#pragma unroll
  for (int i = 0; i < DPT; ++i) num[i] = 0.f;
  if (M != -INFINITY) {
    for (int s = 0; s < a.nsplit; ++s) {
      const int64_t p = first + s * step;
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * p);
      const float w = __builtin_amdgcn_exp2f(ml.x - M);  // 0 for a split that saw no key
      den = fmaf(w, ml.y, den);
#pragma unroll
      for (int i = 0; i < DPT; ++i) num[i] = fmaf(w, a.part_acc[p * D + k + 16 * i], num[i]);
    }
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
  for (int i = 0; i < DPT; ++i) x[r * XS + k + 16 * i] = num[i] * inv;
  __syncthreads();
  const int g = lane >> 4, c = lane & 15, rr = 16 * blk + c;
  const int kvh = int(unit % a.Hkv), Hq = a.Hkv * a.n_rep;
  const int64_t b = unit / a.Hkv;
  const int64_t o = ((b * Hq + kvh * a.n_rep + rr % a.n_rep) * a.T + rr / a.n_rep) * D + 4 * g;
  tree_rows_product<D>(
      x, wave, lane,
      [&](int j, int kk) {
        return f32x4{a.pi_v[kk * D + j], a.pi_v[(kk + 1) * D + j], a.pi_v[(kk + 2) * D + j], a.pi_v[(kk + 3) * D + j]};
      },
      [&](int t, f32x4 v) {
        if (rr >= rows) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) store_elem(a.out, o + 16 * t + i, a.out_dtype, v[i]);
      });
}

template <int D, bool EX, int NCT, int RG, int TG>
TreeScan tree_scan() {
  using C = TreeCfg<D, EX, NCT, RG, TG>;
  return TreeScan{tree_scan_kernel<D, EX, NCT, RG, TG>, C::ROWS, C::NTHR, C::tab_off};
}

template <int D, bool EX>
TreeKernels tree_kernels() {
  TreeKernels k;
  if constexpr (D == 256) {
    // 128 accumulator registers per 32 rows: sixteen rows a wave
    k.scan[0] = k.scan[1] = k.scan[2] = tree_scan<D, EX, 1, 4, 1>();
  } else {
    k.scan[0] = tree_scan<D, EX, 1, 2, 2>();
    k.scan[1] = tree_scan<D, EX, 2, 2, 2>();
    k.scan[2] = tree_scan<D, EX, 2, 4, 1>();
  }
  k.rotate = tree_rotate_kernel<D>;
  k.merge = tree_merge_kernel<D>;
  return k;
}

}  // namespace
}  // namespace wn
