// Rotation and merge of the windowed attention's rows by work-groups that stay (the rotation: below).
//
// The merge: each keeps its part of the rotation in registers and takes tile after tile of sixteen rows, the
// next tile's partials on their way while one is multiplied. tree_merge_kernel<D, 4> reads the 4 D^2 bytes of
// the rotation once for every four rows, but joins the splits of a row by a whole wave. us in traces, it and this, by head_dim, tiles and splits:
//   128    8 tiles   2 splits  6.4   4.8     8 splits  6.1   5.3     32 splits  6.0   9.4
//   128  128 tiles   2 splits 12.5   5.1     8 splits 12.6   6.1     32 splits 14.6  12.8
//   128  384 tiles   2 splits 34     8.0     8 splits 34    10.4     32 splits 37    26
//    64  128 tiles   2 splits  8.8   4.7     8 splits  8.2   4.0     32 splits  8.4   8.4
//   256  128 tiles   2 splits 22    11       8 splits 24    14       32 splits 27    26
// Against sixteen rows a work-group (tree_merge_kernel<D, 16>), head_dim 128, one or two splits: 512 tiles
// 10.2 and 8.5, 1,024 18.5 and 13.8, 4,000 64 and 40; head_dim 64 and 4,000 47 and 17. The bytes of
// 4,000 tiles (partials read, a bf16 result written) take 10 us at 4.8 TB/s; what is left is the tile's
// chain of load, barrier and products.
#pragma once

#include "wn_tree_kernels.h"

namespace wn {
namespace {

// q' of every row, as tree_rotate_kernel writes it, for many tiles of sixteen rows: a work-group keeps its
// part of Pi_K and takes tile after tile, the next one's rows on their way while one is multiplied.
// us in traces, a work-group a tile and this: head_dim 256, 504 tiles 25.8 and 21.3, 7,104 297 and 158 (fp32 matrix cores: 93); head_dim
// 128, 512 tiles 8.1 and 8.5, 1,024 13.8 and 13.6, 4,000 39 and 34, 7,700 62 and 54. At head_dim 64 a rotation is 16 KB, and 4,000 tiles
// take 15.9 and 16.3.
template <int D>
__global__ __launch_bounds__(window_row_threads(D)) void window_rotate_kernel(TreeRotArgs a, int tiles) {
  constexpr int XS = D + 4, EPT = 16 * D / window_row_threads(D), DPT = D / 16;
  static_assert(EPT == 4 && DPT >= 8, "16 or 8 bytes a load, 16 a store");
  __shared__ __align__(16) float x[16 * XS];
  __shared__ __align__(16) float y[16 * XS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, per = a.nrp / 16, rows = a.n_rep * a.T;
  TreeProduct<D> pi;
  pi.load(wave, lane, [&](int j, int k) { return *reinterpret_cast<const f32x4*>(a.pi + j * D + k); });
  const int rr = tid * EPT / D, d0 = tid * EPT % D;  // the thread's elements of a tile
  f32x4 v;
  const auto fetch = [&](int tile) {
    const int unit = tile / per, r = 16 * (tile % per) + rr, kvh = unit % a.Hkv;
    v = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r >= rows) return;  // padding
    const int64_t o = int64_t(unit / a.Hkv) * a.qsb + (kvh * a.n_rep + r % a.n_rep) * a.qsh + (r / a.n_rep) * a.qsq + d0;
    if (a.vec && a.q_dtype == WN_F32) {
      v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + o);
    } else if (a.vec) {
      const uint2 h = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + o);
      const uint32_t w[4] = {h.x & 0xffffu, h.x >> 16, h.y & 0xffffu, h.y >> 16};
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a.q_dtype == WN_BF16 ? bf16_to_f32(uint16_t(w[e])) : f16_to_f32(uint16_t(w[e]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = load_elem(a.q, o + e, a.q_dtype);
    }
  };
  fetch(blockIdx.x);
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    *reinterpret_cast<f32x4*>(x + rr * XS + d0) = v;
    __syncthreads();  // x; and y of the tile before is read
    if (tile + int(gridDim.x) < tiles) fetch(tile + gridDim.x);
    const int g = lane >> 4, c = lane & 15;
    *reinterpret_cast<f32x4*>(y + c * XS + 16 * wave + 4 * g) = pi.run(x + c * XS, lane);
    __syncthreads();  // y; and x is read
    if (tid < 256) {
      // sixteen threads a row: its largest magnitude, then the fp16 terms of q' 2^e (below 2^15)
      const int r = tid >> 4, k = tid & 15;
      float w[DPT], top = 0.f;
      __builtin_memcpy(w, __builtin_assume_aligned(y + r * XS + DPT * k, 16), 4 * DPT);
#pragma unroll
      for (int d = 0; d < DPT; ++d) top = fmaxf(top, fabsf(w[d]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 16));
      int qe;
      frexpf(fminf(top, 3.0e38f), &qe);
      const int e = min(15 - qe, 120);
      const float up = ldexpf(1.f, e);
      const int64_t row = int64_t(tile) * 16 + r;  // a unit's rows are nrp, a multiple of sixteen
      if (k == 0) a.qs[row] = ldexpf(a.scale, -(e + 8));
      _Float16 h[DPT], l[DPT];
#pragma unroll
      for (int d = 0; d < DPT; ++d) {
        const float t = w[d] * up;
        h[d] = _Float16(t);
        l[d] = _Float16(t - float(h[d]));
      }
      __builtin_memcpy(__builtin_assume_aligned(a.qh + row * D + DPT * k, 16), h, 2 * DPT);
      if (a.exact) __builtin_memcpy(__builtin_assume_aligned(a.ql + row * D + DPT * k, 16), l, 2 * DPT);
    }
  }
}

// A lane takes EPT elements of one row, its splits one after the other.
template <int D>
__global__ __launch_bounds__(window_row_threads(D)) void window_merge_kernel(WindowMergeArgs a) {
  constexpr int XS = D + 4, EPT = 16 * D / window_row_threads(D);
  constexpr int U = D == 256 ? 1 : 8;  // splits loaded at once (at 256 the rotation takes half of the 128 registers)
  __shared__ __align__(16) float x[2][16 * XS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rows = a.n_rep * a.T, blocks = (rows + 15) / 16, Hq = a.Hkv * a.n_rep;
  TreeProduct<D> pi;
  if (wave < D / 16)
    pi.load(wave, lane, [&](int j, int k) {
      return f32x4{a.pi_v[k * D + j], a.pi_v[(k + 1) * D + j], a.pi_v[(k + 2) * D + j], a.pi_v[(k + 3) * D + j]};
    });
  const int rr = tid * EPT / D, d0 = tid * EPT % D;
  float v[U][EPT];
  float2 ml[U];
  // A tile's row (past the last row: that again) in U splits from s.
  const auto fetch = [&](int tile, int s) {
    const int64_t row = (int64_t(tile / blocks) * a.nsplit + s) * a.nrp + min(16 * (tile % blocks) + rr, rows - 1);
    const float* acc = a.part_acc + row * D + d0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= a.nsplit) break;
      ml[u] = *reinterpret_cast<const float2*>(a.part_ml + 2 * (row + int64_t(u) * a.nrp));
      __builtin_memcpy(v[u], __builtin_assume_aligned(acc + int64_t(u) * a.nrp * D, 4 * EPT), 4 * EPT);
    }
  };
  fetch(blockIdx.x, 0);
  for (int tile = blockIdx.x, buf = 0; tile < a.tiles; tile += gridDim.x, buf ^= 1) {
    const int unit = tile / blocks, blk = tile % blocks, b = unit / a.Hkv;
    const int L = min(max(a.seq_lens[b], 0), a.max_len);
    const WindowSpan ws = window_span(L, a.T, a.n_rep, 16 * blk / a.rows_block * a.rows_block, a.rows_block, a.chunk, a.window, a.sinks,
                                      a.nsplit, a.span);
    const int live = ws.span ? (ws.total + ws.span - 1) / ws.span : 0;
    float M = -INFINITY, den = 0.f, num[EPT] = {};
    for (int s = 0; s < live; s += U) {
      if (s) fetch(tile, s);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s + u >= live) break;
        // a split that saw no key has weight 0, and so has one whose every score is NaN: its sums are NaN, and stay so
        const float up = fmaxf(M, ml[u].x), top = up == -INFINITY ? 0.f : up;
        const float old = __builtin_amdgcn_exp2f(M - top), w = __builtin_amdgcn_exp2f(ml[u].x - top);
        den = den * old + w * ml[u].y;
#pragma unroll
        for (int e = 0; e < EPT; ++e) num[e] = num[e] * old + w * v[u][e];
        M = up;
      }
    }
    const float inv = den != 0.f ? 1.f / den : 0.f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[buf][rr * XS + d0 + e] = num[e] * inv;
    __syncthreads();  // x[buf]; its last readers are a barrier behind
    if (tile + int(gridDim.x) < a.tiles) fetch(tile + gridDim.x, 0);
    const int g = lane >> 4, c = lane & 15, row = 16 * blk + c;
    if (wave < D / 16) {
      const f32x4 y = pi.run(x[buf] + c * XS, lane);
      if (row < rows) {
        const int64_t o = ((int64_t(b) * Hq + unit % a.Hkv * a.n_rep + row % a.n_rep) * a.T + row / a.n_rep) * D + 16 * wave + 4 * g;
        if (a.out_dtype == WN_F32) {
          __builtin_memcpy(static_cast<float*>(a.out) + o, &y, 16);
        } else {
          uint16_t h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = a.out_dtype == WN_BF16 ? f32_to_bf16(y[i]) : f32_to_f16(y[i]);
          __builtin_memcpy(static_cast<uint16_t*>(a.out) + o, h, 8);
        }
      }
    }
  }
}

template <int D>
WindowKernels window_kernels_for(bool exact, int bw_k, int bw_v) {
  WindowKernels k;
  static_cast<TreeKernelsOf<WindowArgs, WindowMergeArgs>&>(k) = tree_kernels_for<D, true>(exact, bw_k, bw_v);
  k.merge[1] = window_merge_kernel<D>;
  if constexpr (D >= 128) k.rotate_many = window_rotate_kernel<D>;
  return k;
}

}  // namespace
}  // namespace wn
