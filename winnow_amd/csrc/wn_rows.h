// What the per-wave scans over packed pages share (prefill.hip: the fused prefill; tree_rows.hip:
// trees of drafted tokens): one wave takes 16 NCT query rows against 64-token chunks at head_dim
// 128, K and V codes of 4 or 6 bits going through LDS codebook tables straight into MFMA operands.
// Args: the kernel's arguments (k_pages, v_pages, k_norms, v_norms, the strides ksp .. vnh, log2S,
// part_acc, part_ml).
#pragma once

#include "wn_common.h"
#include "wn_tables.h"

namespace wn {
namespace {

// The four 16-token tiles of chunk [c0, c0+64): page ids (wave-uniform) and in-page
// slots. A tile's 16 tokens share a page (16 | c0 and S >= 16); its page-table column
// is clamped to col_hi, the range's last page (tokens past the range are read from
// real pages and masked).
struct PfTiles {
  uint32_t pid[4];
  uint32_t slot[4];
};

template <class Args>
__device__ __forceinline__ PfTiles pf_tiles(const Args& a, const int32_t* trow, int c0, int col_hi) {
  PfTiles o;
  const int smask = (1 << a.log2S) - 1;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int t0 = c0 + 16 * t;
    // the page table is not written while the scan runs: const_view keeps these
    // wave-uniform reads scalar loads (the pacing word's LDS store would otherwise
    // make the compiler read them with vector loads and wait on them)
    o.pid[t] = uint32_t(__builtin_amdgcn_readfirstlane(const_view(trow)[min(t0 >> a.log2S, col_hi)]));
    o.slot[t] = uint32_t(t0 & smask);
  }
  return o;
}

// K rows: tile t, quarter g of token c0 + 16t + c (words [t BWK, t BWK + BWK)).
template <int BWK>
struct PfK {
  uint32_t w[4 * BWK];
};
// V rows: token (t, i) = c0 + 16t + 4g + i, codes of dims 8c .. 8c+7 (6-bit: the raw
// 8-byte window from 6c rounded down to 4), VW words each.
template <int BWV>
struct PfV {
  static constexpr int VW = BWV == 4 ? 1 : 2;
  uint32_t w[16 * VW];
};
// fp16 norms of tokens (t, i): half i & 1 of word 2t + (i >> 1).
struct PfN {
  uint32_t nk[8], nv[8];
};

template <int BWK, class Args>
__device__ __forceinline__ void pf_load_k(const Args& a, const PfTiles& tl, int kvh, int lane, PfK<BWK>& o) {
  constexpr int NBK = 16 * BWK;
  const int g = lane >> 4, c = lane & 15;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint8_t* kp = a.k_pages + uint64_t(tl.pid[t]) * uint64_t(a.ksp) + uint64_t(kvh) * uint64_t(a.ksh) +
                        (tl.slot[t] + uint32_t(c)) * uint32_t(NBK) + uint32_t(4 * BWK * g);
    if constexpr (BWK == 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(kp);
      o.w[4 * t] = x.x;
      o.w[4 * t + 1] = x.y;
      o.w[4 * t + 2] = x.z;
      o.w[4 * t + 3] = x.w;
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint2 x = reinterpret_cast<const uint2*>(kp)[j];
        o.w[6 * t + 2 * j] = x.x;
        o.w[6 * t + 2 * j + 1] = x.y;
      }
    }
  }
}

template <int BWV, class Args>
__device__ __forceinline__ void pf_load_v(const Args& a, const PfTiles& tl, int kvh, int lane, PfV<BWV>& o) {
  constexpr int NBV = 16 * BWV, VW = PfV<BWV>::VW;
  const int g = lane >> 4, c = lane & 15;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint8_t* vb = a.v_pages + uint64_t(tl.pid[t]) * uint64_t(a.vsp) + uint64_t(kvh) * uint64_t(a.vsh) +
                        (tl.slot[t] + uint32_t(4 * g)) * uint32_t(NBV);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (BWV == 4) {
        o.w[4 * t + i] = *reinterpret_cast<const uint32_t*>(vb + i * NBV + 4 * c);
      } else {
        uint2 x;
        __builtin_memcpy(&x, __builtin_assume_aligned(vb + i * NBV + ((6 * c) & ~3), 4), 8);
        o.w[VW * (4 * t + i)] = x.x;
        o.w[VW * (4 * t + i) + 1] = x.y;
      }
    }
  }
}

template <class Args>
__device__ __forceinline__ void pf_load_n(const Args& a, const PfTiles& tl, int kvh, int lane, PfN& o) {
  const int g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t ns = tl.slot[t] + uint32_t(4 * g);
    const uint2 nk = *reinterpret_cast<const uint2*>(a.k_norms + uint64_t(tl.pid[t]) * uint64_t(a.knp) +
                                                     uint64_t(kvh) * uint64_t(a.knh) + ns);
    const uint2 nv = *reinterpret_cast<const uint2*>(a.v_norms + uint64_t(tl.pid[t]) * uint64_t(a.vnp) +
                                                     uint64_t(kvh) * uint64_t(a.vnh) + ns);
    o.nk[2 * t] = nk.x;
    o.nk[2 * t + 1] = nk.y;
    o.nv[2 * t] = nv.x;
    o.nv[2 * t + 1] = nv.y;
  }
}

__device__ __forceinline__ float half_at(const uint32_t* w, int k) {
  return f16_to_f32(uint16_t(w[k >> 1] >> (16 * (k & 1))));
}

// The V rows' token pairs (2p, 2p+1) rewritten in place so that one word per (pair,
// dim parity) holds the pair indices: 4-bit, the byte of dims (2j, 2j+1) becomes
// (first token's code of dim 2j, second's) in the first word and the same for dim
// 2j+1 in the second; 6-bit, the raw windows are moved down to the codes and the pair
// becomes (Ce, Co), Ce holding the first token's even-numbered codes with the second's
// shifted up one field into the gaps, Co the same for the odd ones (pair index of dim
// m: the 12 bits of Ce (m even) or Co (m odd) from bit 6 m).
template <int BWV>
__device__ __forceinline__ void pf_merge_pairs(PfV<BWV>& o, int lane) {
  if constexpr (BWV == 4) {
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const uint32_t wa = o.w[2 * p], wb = o.w[2 * p + 1];
      o.w[2 * p] = bitsel(0x0F0F0F0Fu, wa, wb << 4);
      o.w[2 * p + 1] = bitsel(0x0F0F0F0Fu, wa >> 4, wb);
    }
  } else {
    constexpr uint64_t E = 0x03F03F03F03Full;    // fields 0, 2, 4, 6 of 6 bits
    constexpr uint64_t O = ~E & 0xFFFFFFFFFFFFull;  // fields 1, 3, 5, 7
    const uint32_t sh = 16u * uint32_t(lane & 1);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      uint32_t* x = o.w + 2 * (2 * p);
      uint32_t* y = o.w + 2 * (2 * p + 1);
      const uint64_t a = (uint64_t(x[1]) << 32 | x[0]) >> sh;
      const uint64_t b = (uint64_t(y[1]) << 32 | y[0]) >> sh;
      const uint64_t bs = b << 6;
      const uint64_t ce = (a & E) | (bs & ~E);
      const uint64_t co = (a & O) | (bs & ~O);
      x[0] = uint32_t(ce);
      x[1] = uint32_t(ce >> 32);
      y[0] = uint32_t(co);
      y[1] = uint32_t(co >> 32);
    }
  }
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

template <int NCT>
struct PfState {
  f32x4 acc[NCT][8];  // acc[ct][mt] register i: dim 32g + 8i + mt of column c, scaled by 2^(8-gs)
  float m[NCT];       // reference maximum of column c (log2 units; -inf before its first key)
  float l[NCT];       // sum of 2^(s - m) over this lane's tokens
  int lim[NCT];       // last visible token of column c (padding rows: no limit)
  int gs;             // value scale shift (wave-uniform)
};

constexpr int kPfLookahead = 4;  // K-steps of table reads in flight ahead of their MFMA

// Scores of the chunk: d[ct][t] register i = token 16t + 4g + i of column c, before
// the n_K 2^-(e+8) scale. Step k = 4s + t (K-step s of tile t); one A operand (four
// pair lookups) feeds NCT MFMAs.
template <int BWK, int NCT>
__device__ __forceinline__ void pf_scores(const PfK<BWK>& K, TabTf<BWK>& cbk, const h8 (&qb)[NCT][4],
                                          f32x4 (&d)[NCT][4]) {
  constexpr int LA = kPfLookahead;
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
    for (int t = 0; t < 4; ++t) d[ct][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // the four entries of a step land in one 4-register operand (no moves to assemble it)
  u32x4 e[LA + 1];
  auto look = [&](auto kc, u32x4& o) {
    constexpr int k = decltype(kc)::value, s = k >> 2, t = k & 3;
    o[0] = piece_pair_tf<BWK, 4 * s>(K.w + t * BWK, cbk);
    o[1] = piece_pair_tf<BWK, 4 * s + 1>(K.w + t * BWK, cbk);
    o[2] = piece_pair_tf<BWK, 4 * s + 2>(K.w + t * BWK, cbk);
    o[3] = piece_pair_tf<BWK, 4 * s + 3>(K.w + t * BWK, cbk);
  };
  // the schedule is pinned step by step (sched_barrier): left free, the compiler
  // hoists every table read to the top and runs out of registers
  static_for<0, LA>([&](auto kc) { look(kc, e[decltype(kc)::value]); });
  __builtin_amdgcn_sched_barrier(0);
  static_for<0, 16>([&](auto kc) {
    constexpr int k = decltype(kc)::value, s = k >> 2, t = k & 3, j = k % (LA + 1);
    if constexpr (k + LA < 16) {
      look(std::integral_constant<int, k + LA>{}, e[(k + LA) % (LA + 1)]);
      __builtin_amdgcn_sched_barrier(0);
    }
    const h8 av = __builtin_bit_cast(h8, e[j]);
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) d[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, qb[ct][s], d[ct][t], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// Entry of the 4-bit pair in byte J of x: the address 4 lane | byte << 8 | slot << 16
// formed by one byte permute of x and the table register (a fresh register per read,
// where entry_tf rewrites the shared one in place).
template <int J>
__device__ __forceinline__ uint32_t entry_perm(const TabTf<4>& tab, uint32_t x) {
  const uint32_t addr = __builtin_amdgcn_perm(x, tab.r[0], 0x03020000u | uint32_t(4 + J) << 8);
  return *reinterpret_cast<const uint32_t*>(tab.lds + addr);
}

// Values of the chunk: step k = 8ks + mt; pair q of K-step ks = tokens (8ks + 2q,
// 8ks + 2q + 1) of the V rows, merged by pf_merge_pairs.
template <int BWV, int NCT>
__device__ __forceinline__ void pf_values(const PfV<BWV>& V, TabTf<BWV>& cbv, const h8 (&pb)[NCT][2],
                                          PfState<NCT>& st) {
  constexpr int LA = kPfLookahead, VW = PfV<BWV>::VW;
  u32x4 e[LA + 1];
  auto look = [&](auto kc, u32x4& o) {
    constexpr int k = decltype(kc)::value, ks = k >> 3, mt = k & 7;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t* w = V.w + VW * (8 * ks + 2 * q + (mt & 1));
      if constexpr (BWV == 4) o[q] = entry_perm<(mt >> 1)>(cbv, w[0]);
      else o[q] = pair_entry_tf(cbv, pair_offset<6, 6 * mt, 2>(w));
    }
  };
  static_for<0, LA>([&](auto kc) { look(kc, e[decltype(kc)::value]); });
  __builtin_amdgcn_sched_barrier(0);
  static_for<0, 16>([&](auto kc) {
    constexpr int k = decltype(kc)::value, ks = k >> 3, mt = k & 7, j = k % (LA + 1);
    if constexpr (k + LA < 16) {
      look(std::integral_constant<int, k + LA>{}, e[(k + LA) % (LA + 1)]);
      __builtin_amdgcn_sched_barrier(0);
    }
    const h8 av = __builtin_bit_cast(h8, e[j]);
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct)
      st.acc[ct][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pb[ct][ks], st.acc[ct][mt], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// Writes the (acc, m, l) partial of each column (query row) of the block: lane (g, c)
// writes dims 32g .. 32g+31 of row 16 ct + c.
template <int NCT, class Args>
__device__ __forceinline__ void pf_write(const Args& a, PfState<NCT>& st, int64_t row0, int lane) {
  const int g = lane >> 4, c = lane & 15;
  const float f = ldexpf(1.f, st.gs - 8);
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    float l = st.l[ct];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const int64_t row = row0 + 16 * ct + c;
    float* dst = a.part_acc + row * 128 + 32 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<float4*>(dst + 8 * i) = make_float4(st.acc[ct][0][i] * f, st.acc[ct][1][i] * f,
                                                            st.acc[ct][2][i] * f, st.acc[ct][3][i] * f);
      *reinterpret_cast<float4*>(dst + 8 * i + 4) = make_float4(st.acc[ct][4][i] * f, st.acc[ct][5][i] * f,
                                                                st.acc[ct][6][i] * f, st.acc[ct][7][i] * f);
    }
    if (g == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * row) = make_float2(st.m[ct], l);
  }
}

// Logical index of work-group p of n when groups go to the 8 XCDs round robin: XCD x
// holds groups x, x+8, ...; they become a contiguous run of logical indices, so the
// waves of neighbouring items (the column blocks of one split) share an XCD's L2.
__device__ __forceinline__ int pf_xcd_major(int p, int n) {
  const int q = n >> 3, r = n & 7, x = p & 7, s = p >> 3;
  return x * q + min(x, r) + s;
}

template <int BWK, int BWV>
struct PfLds {
  static constexpr bool k4 = BWK == 4, v4 = BWV == 4;
  static constexpr int k_off = k4 && !v4 ? kTfTableBytes : 0;
  static constexpr int v_off = v4 ? kTfTableBytes : k4 ? 0 : tf_table_bytes<BWK>();
  static constexpr int pace = k_off + tf_table_bytes<BWK>() > v_off + tf_table_bytes<BWV>()
                                  ? k_off + tf_table_bytes<BWK>()
                                  : v_off + tf_table_bytes<BWV>();  // one word per wave (Pace)
  static constexpr int total = pace + 4 * 8;
  static_assert(total <= 160 * 1024, "LDS of a work-group exceeds 160 KB");
};

}  // namespace
}  // namespace wn
