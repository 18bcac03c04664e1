// Operands and device helpers that the quantize kernels share (quant.hip: sixteen
// vectors per work-group, float64 rotation; quant_tile.hip: many vectors per wave).
#pragma once

#include <type_traits>

#include "wn_common.h"

namespace wn {

struct QuantSide {
  const void* x;
  int64_t sb, sh, sn;  // element strides of (B, H, n, D)
  const float* pi;
  const float* bnd;
  int bw;
  uint8_t* pages;  // scatter mode
  int64_t psp, psh;
  uint16_t* norms;
  int64_t nsp, nsh;
  uint8_t* codes_out;  // flat mode
  float* norms_out;
};

template <class Side>
struct QuantArgsOf {
  Side side[2];  // K, V
  const int32_t* table;
  const int32_t* start_pos;
  int64_t tsb;
  int64_t total;  // vectors per side = B*H*n
  int H, n, log2S, num_pages, max_pages, x_dtype, scatter;
};
using QuantArgs = QuantArgsOf<QuantSide>;

// Outlier channels (launch_quantize_split): boundaries, width, rows and norms of the second group.
struct QuantGroup2 {
  const float* bnd;
  int bw;
  uint8_t* pages;
  uint16_t* norms;
};

struct QuantSplitSide : QuantSide {
  QuantGroup2 second;
};

struct QuantSplitArgs : QuantArgsOf<QuantSplitSide> {
  const uint8_t* chan;    // group of each channel
  int split, pos0;        // codes of group 0, first position
  int64_t cap;            // rows per (sequence, head)
};

// The position rotation of an append (wn_append_rotated_kv): K is rotated on its way into the
// quantizer, and q beside it, by work-groups of its own.
struct QuantRotary {
  const void* cos;  // (B, n, R), a row per token, of rot_dtype
  const void* sin;
  int64_t csb, csn, ssb, ssn;  // element strides; of the batch 0 where it shares one table
  const void* q;               // (B, Hq, n, D), or null
  int64_t qsb, qsh, qsn;
  void* q_out;                 // contiguous, q's type
  int rot_dtype, R, q_dtype, Hq, B;
  int q_vec;  // q, its output and the tables can be read by 16 bytes, eight channels and their partners at once
  int k_vec;  // K and the tables can
};

struct QuantRotArgs : QuantArgs {
  QuantRotary rot;
  int split[2];  // of the tile kernel: first work-group of V, and of q
};

// Channel d of a rotated row, from the row's channels and its token's cos and sin:
//   x_d cos_d - x_(d + R/2) sin_d   (d < R/2),   x_d cos_d + x_(d - R/2) sin_d   (d < R),   x_d
// The products of fp32 values are exact in float64, so the sum is rounded once there and once to
// fp32: the same bits whoever computes it.
__device__ __forceinline__ float turn(float x, float partner, float c, float s) {
  return float(fma(double(partner), double(s), double(x) * double(c)));
}
__device__ __forceinline__ float rotated_elem(const QuantRotary& r, const void* x, int64_t row, int x_dtype, int64_t co, int64_t so, int d) {
  const float v = load_elem(x, row + d, x_dtype);
  if (d >= r.R) return v;
  const int half = r.R / 2;
  const float p = load_elem(x, row + (d < half ? d + half : d - half), x_dtype);
  return turn(v, d < half ? -p : p, load_elem(r.cos, co + d, r.rot_dtype), load_elem(r.sin, so + d, r.rot_dtype));
}

// Eight elements of a row as they are stored.
template <int DT>
struct Raw8 {
  uint4 w[DT == WN_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* x, int64_t i) {
  Raw8<DT> r;
  if constexpr (DT == WN_F32) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(x) + i);
    r.w[0] = p[0];
    r.w[1] = p[1];
  } else {
    r.w[0] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + i);
  }
  return r;
}
template <int DT>
__device__ __forceinline__ float elem(const Raw8<DT>& r, int k) {
  const uint4 a = r.w[DT == WN_F32 ? k >> 2 : 0];
  if constexpr (DT == WN_F32) {
    const int j = k & 3;
    return __builtin_bit_cast(float, j == 0 ? a.x : j == 1 ? a.y : j == 2 ? a.z : a.w);
  } else {
    const int j = k >> 1;
    const uint32_t w = j == 0 ? a.x : j == 1 ? a.y : j == 2 ? a.z : a.w;
    if constexpr (DT == WN_BF16) return __builtin_bit_cast(float, k & 1 ? w & 0xffff0000u : w << 16);
    else return f16_to_f32(uint16_t(k & 1 ? w >> 16 : w));
  }
}

// Channels d .. d + 7 of a rotated row (R and R / 2 multiples of 8: they and their partners are
// eight in a row each). Of two 16-bit factors the products are exact in fp32 already, and the fused
// sum there is the same value.
template <int DT, int CT>
__device__ __forceinline__ void rotated8(const QuantRotary& r, const void* x, int64_t row, int64_t co, int64_t so, int d, float (&y)[8]) {
  const Raw8<DT> v = load8<DT>(x, row + d);
  if (d >= r.R) {
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = elem<DT>(v, k);
    return;
  }
  const int half = r.R / 2;
  const Raw8<DT> p = load8<DT>(x, row + (d < half ? d + half : d - half));
  const Raw8<CT> c = load8<CT>(r.cos, co + d), s = load8<CT>(r.sin, so + d);
  const uint32_t flip = d < half ? 0x80000000u : 0u;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float q = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, elem<DT>(p, k)) ^ flip);
    if constexpr (DT != WN_F32 && CT != WN_F32) y[k] = fmaf(q, elem<CT>(s, k), elem<DT>(v, k) * elem<CT>(c, k));
    else y[k] = turn(elem<DT>(v, k), q, elem<CT>(c, k), elem<CT>(s, k));
  }
}

// Channels d .. d + 7 (lo) and d + R / 2 .. d + R / 2 + 7 (hi) at once: each is the other's partner.
template <int DT, int CT>
__device__ __forceinline__ void rotated8_pair(const Raw8<DT>& lo, const Raw8<DT>& hi, const Raw8<CT>& c0, const Raw8<CT>& s0, const Raw8<CT>& c1,
                                              const Raw8<CT>& s1, float (&y0)[8], float (&y1)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = elem<DT>(lo, k), b = elem<DT>(hi, k);
    if constexpr (DT != WN_F32 && CT != WN_F32) {
      y0[k] = fmaf(-b, elem<CT>(s0, k), a * elem<CT>(c0, k));
      y1[k] = fmaf(a, elem<CT>(s1, k), b * elem<CT>(c1, k));
    } else {
      y0[k] = turn(a, -b, elem<CT>(c0, k), elem<CT>(s0, k));
      y1[k] = turn(b, a, elem<CT>(c1, k), elem<CT>(s1, k));
    }
  }
}

// Eight values as the rotated q's type, 16-byte aligned.
template <int DT>
__device__ __forceinline__ void store_rotated8(void* out, int64_t i, const float (&y)[8]) {
  if constexpr (DT == WN_F32) {
    __builtin_memcpy(__builtin_assume_aligned(static_cast<float*>(out) + i, 16), y, 32);
  } else {
    uint16_t o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = DT == WN_BF16 ? f32_to_bf16(y[k]) : f32_to_f16(y[k]);
    __builtin_memcpy(__builtin_assume_aligned(static_cast<uint16_t*>(out) + i, 16), o, 16);
  }
}

// q by 16 bytes: an item is sixteen channels of a token, eight and their partners or sixteen behind the
// rotated ones, for HEADS heads, whose cos and sin are one; a head's rows are read and written once,
// all in flight together.
template <int D, int NTHR, int DT, int CT>
__device__ __forceinline__ void rotate_heads(const QuantRotary& r, int n, uint32_t block, uint32_t blocks, int tid) {
  constexpr int HEADS = DT == WN_F32 ? 2 : 4;
  constexpr uint32_t PARTS = D / 16;
  const uint32_t groups = (uint32_t(r.Hq) + HEADS - 1) / HEADS, items = uint32_t(r.B) * groups * uint32_t(n) * PARTS, turned = uint32_t(r.R) / 16;
  for (uint32_t it = block * NTHR + tid; it < items; it += blocks * NTHR) {
    const uint32_t row = it / PARTS, part = it % PARTS, i = row % uint32_t(n), bg = row / uint32_t(n), h0 = bg % groups * HEADS, b = bg / groups;
    const bool turns = part < turned;
    const uint32_t d = turns ? 8 * part : r.R + 16 * (part - turned), step = turns ? r.R / 2 : 8;
    const int64_t qo = b * r.qsb + i * r.qsn + d;
    Raw8<DT> lo[HEADS], hi[HEADS];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      const int64_t at = qo + min(h0 + h, uint32_t(r.Hq) - 1) * r.qsh;  // past the last: it again
      lo[h] = load8<DT>(r.q, at);
      hi[h] = load8<DT>(r.q, at + step);
    }
    const uint32_t cd = turns ? d : 0;  // some row's: not used
    const int64_t co = b * r.csb + i * r.csn + cd, so = b * r.ssb + i * r.ssn + cd;
    const Raw8<CT> c0 = load8<CT>(r.cos, co), s0 = load8<CT>(r.sin, so), c1 = load8<CT>(r.cos, co + r.R / 2), s1 = load8<CT>(r.sin, so + r.R / 2);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      if (h0 + h >= uint32_t(r.Hq)) break;
      float y0[8], y1[8];
      if (turns) {
        rotated8_pair<DT, CT>(lo[h], hi[h], c0, s0, c1, s1, y0, y1);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          y0[k] = elem<DT>(lo[h], k);
          y1[k] = elem<DT>(hi[h], k);
        }
      }
      const int64_t to = ((int64_t(b) * r.Hq + h0 + h) * n + i) * D + d;
      store_rotated8<DT>(r.q_out, to, y0);
      store_rotated8<DT>(r.q_out, to + step, y1);
    }
  }
}

// f(x_dtype, type of the tables), as constants
template <class F>
__device__ __forceinline__ void rotary_types(const QuantRotary& r, int x_dtype, F&& f) {
  const auto by = [&](auto dt) {
    if (r.rot_dtype == WN_F32) f(dt, std::integral_constant<int, WN_F32>{});
    else if (r.rot_dtype == WN_BF16) f(dt, std::integral_constant<int, WN_BF16>{});
    else f(dt, std::integral_constant<int, WN_F16>{});
  };
  if (x_dtype == WN_F32) by(std::integral_constant<int, WN_F32>{});
  else if (x_dtype == WN_BF16) by(std::integral_constant<int, WN_BF16>{});
  else by(std::integral_constant<int, WN_F16>{});
}

// rotated8 of rows whose type is a run-time value.
__device__ __forceinline__ void rotated8_of(const QuantRotary& r, const void* x, int x_dtype, int64_t row, int64_t co, int64_t so, int d, float (&y)[8]) {
  rotary_types(r, x_dtype, [&](auto dt, auto ct) { rotated8<decltype(dt)::value, decltype(ct)::value>(r, x, row, co, so, d, y); });
}

// q's rows rotated, by the threads of `blocks` work-groups of NTHR: by rotate_heads, or eight channels of
// a row (b, h, i) an item, element by element.
template <int D, int NTHR>
__device__ __forceinline__ void rotate_queries(const QuantRotary& r, int n, uint32_t block, uint32_t blocks, int tid) {
  if (r.q_vec) {
    rotary_types(r, r.q_dtype, [&](auto dt, auto ct) { rotate_heads<D, NTHR, decltype(dt)::value, decltype(ct)::value>(r, n, block, blocks, tid); });
    return;
  }
  constexpr uint32_t EIGHTS = D / 8;
  const uint32_t items = uint32_t(r.B) * uint32_t(r.Hq) * uint32_t(n) * EIGHTS;  // below 2^30 (the host's check)
  for (uint32_t it = block * NTHR + tid; it < items; it += blocks * NTHR) {
    const uint32_t row = it / EIGHTS, d = 8 * (it % EIGHTS), i = row % uint32_t(n), bh = row / uint32_t(n), h = bh % uint32_t(r.Hq),
                   b = bh / uint32_t(r.Hq);
    const int64_t qo = b * r.qsb + h * r.qsh + i * r.qsn, co = b * r.csb + i * r.csn, so = b * r.ssb + i * r.ssn;
    const int64_t to = int64_t(row) * D + d;
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = rotated_elem(r, r.q, qo, r.q_dtype, co, so, d + k);
    if (r.q_dtype == WN_F32) store_rotated8<WN_F32>(r.q_out, to, y);
    else if (r.q_dtype == WN_BF16) store_rotated8<WN_BF16>(r.q_out, to, y);
    else store_rotated8<WN_F16>(r.q_out, to, y);
  }
}

// pos[k] = #{b < y[k]} over the 2^bw - 1 ascending boundaries (torch.bucketize,
// right=False), for N values at once: the N binary searches advance in lockstep, so
// each level issues N independent LDS reads instead of one dependent read per value.
template <int N>
__device__ __forceinline__ void bucketize_n(const float* bnd, int bw, const float (&y)[N], uint32_t (&pos)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) pos[k] = 0;
  for (int step = 1 << (bw - 1); step > 0; step >>= 1) {
    float b[N];
#pragma unroll
    for (int k = 0; k < N; ++k) b[k] = bnd[pos[k] + step - 1];
#pragma unroll
    for (int k = 0; k < N; ++k) pos[k] += b[k] < y[k] ? step : 0;
  }
}

// The bw bytes of eight bw-bit codes packed LSB-first, stored at p (p is aligned to
// the largest power of two dividing bw).
__device__ __forceinline__ void store_packed8(uint8_t* p, uint64_t v, int bw) {
  if (bw == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(uint32_t(v), uint32_t(v >> 32));
  } else if (bw == 4) {
    *reinterpret_cast<uint32_t*>(p) = uint32_t(v);
  } else if (bw == 2) {
    *reinterpret_cast<uint16_t*>(p) = uint16_t(v);
  } else if (bw == 6) {
    reinterpret_cast<uint16_t*>(p)[0] = uint16_t(v);
    reinterpret_cast<uint16_t*>(p)[1] = uint16_t(v >> 16);
    reinterpret_cast<uint16_t*>(p)[2] = uint16_t(v >> 32);
  } else {
    for (int k = 0; k < bw; ++k) p[k] = uint8_t(v >> (8 * k));
  }
}

// quant_tile.hip: whether its kernel serves these operands, and its launch (0: launched).
bool quantize_tiles_ok(const QuantArgs& a, int sides, int D);
int launch_quantize_tiles(const QuantArgs& a, int sides, int D, hipStream_t st);
int launch_quantize_tiles(const QuantRotArgs& a, int sides, int D, hipStream_t st);
// The same kernel with two groups of channels, rows of a contiguous cache (quant.hip's
// wn_append_split).
bool quantize_split_ok(const QuantSplitArgs& a, int sides, int D);
int launch_quantize_split(const QuantSplitArgs& a, int sides, int D, hipStream_t st);

}  // namespace wn
