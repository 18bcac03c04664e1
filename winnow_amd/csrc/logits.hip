// Logits as a sampler or a greedy choice is to see them: penalties for tokens of a row's
// history, biases of single tokens, and a bit mask of the tokens that are allowed.
//
//   seen    the token is in history[0, length)
//   c       how often it is in history[prompt_length, length)
//   x <- seen ? (x > 0 ? x / repetition : x repetition) : x
//   x <- x - frequency c - (c > 0 ? presence : 0)
//   x <- x + (the row's biases of the token, in the order of the list)
//   x <- allowed ? x : -inf
//
// in fp32, rounded once to the logits' type; a logit that nothing applies to keeps its bits.
//
// Bound: HBM, one read and one write of the logits; latency at few rows. A work-group of four
// waves takes a segment of a row. Its logits and mask bytes are asked for first and travel while
// it reads the whole history (16 KB of 4,096 tokens, from L2 for all segments but the first) and
// counts, in a word of LDS per token of the segment, what the history says of it. The counters
// are whole numbers, so the order of the atomics does not show; biases are found by a walk
// over the segment's part of the list, which keeps the list's order.
#include <algorithm>

#include "wn_common.h"

namespace wn {
namespace {

constexpr int kLgThreads = 256;
constexpr int kLgBiases = 1024;   // most entries of a row's list

struct LogitsArgs {
  const void* x;
  void* out;
  int64_t xs, os;  // row strides, elements
  const int32_t* history;
  int64_t hs;
  const int32_t* lengths;         // null: H
  const int32_t* prompt_lengths;  // null: 0
  const float* repetition;        // null: the scalars below
  const float* presence;
  const float* frequency;
  float rep, pres, freq;
  const int32_t* bias_ids;
  const float* bias;
  int64_t bis, bs;
  const uint8_t* allowed;  // bytes of little-endian words
  int64_t as;              // row stride, bytes
  int V, H, J, nseg;
};

// A token's word: bit 0 seen, bit 1 on the bias list, then its count.
constexpr uint32_t kSeen = 1, kBiased = 2, kOne = 4;

// PIECES: 16-byte pieces of a thread.
template <int DT, int PIECES>
__global__ __launch_bounds__(kLgThreads) void logits_kernel(LogitsArgs a) {
  constexpr int ES = DT == WN_F32 ? 4 : 2, PE = 16 / ES;       // elements of a piece
  constexpr int SEG = kLgThreads * PIECES * PE;
  typedef uint32_t Words __attribute__((ext_vector_type(4)));
  extern __shared__ __align__(16) uint32_t tab[];               // SEG words, then the biases in reach
  __shared__ int n_bias;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x / a.nseg;
  const int base = int(blockIdx.x % a.nseg) * SEG, n = min(SEG, a.V - base);
  const char* x = static_cast<const char*>(a.x) + (row * a.xs + base) * ES;
  char* out = static_cast<char*>(a.out) + (row * a.os + base) * ES;

  Words w[PIECES];
  uint32_t ok[PIECES];  // the mask's byte of a piece's first element
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int i = (p * kLgThreads + tid) * PE;
    w[p] = Words{0, 0, 0, 0};
    if (i + PE <= n) {
      __builtin_memcpy(&w[p], __builtin_assume_aligned(x + i * ES, ES), 16);
    } else {
#pragma unroll
      for (int e = 0; e < PE; ++e)
        if (i + e < n) {
          if constexpr (ES == 4) w[p][e] = *reinterpret_cast<const uint32_t*>(x + (i + e) * 4);
          else w[p][e >> 1] |= uint32_t(*reinterpret_cast<const uint16_t*>(x + (i + e) * 2)) << (16 * (e & 1));
        }
    }
    ok[p] = a.allowed && i < n ? a.allowed[row * a.as + ((base + i) >> 3)] >> (i & 7) : 0xffu;  // base: a multiple of 8
  }

  const bool counted = a.history || a.J;  // uniform
  float rep = a.rep, pres = a.pres, freq = a.freq;
  int32_t* bid = reinterpret_cast<int32_t*>(tab + SEG);
  float* bval = reinterpret_cast<float*>(bid + a.J);
  if (counted) {
    if (a.repetition) rep = a.repetition[row];
    if (a.presence) pres = a.presence[row];
    if (a.frequency) freq = a.frequency[row];
#pragma unroll
    for (int i = 0; i < SEG / 4; i += kLgThreads) reinterpret_cast<Words*>(tab)[i + tid] = Words{0, 0, 0, 0};
    __syncthreads();
    if (a.history) {
      const int32_t* hist = a.history + row * a.hs;
      const int len = a.lengths ? min(max(a.lengths[row], 0), a.H) : a.H;
      const int made = a.prompt_lengths ? a.prompt_lengths[row] : 0;
      constexpr int U = 8;  // in flight together
      for (int h0 = 0; h0 < len; h0 += U * kLgThreads) {
        uint32_t t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = h0 + u * kLgThreads + tid;
          t[u] = h < len ? uint32_t(hist[h]) - uint32_t(base) : ~0u;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (t[u] < uint32_t(n)) {
            atomicOr(&tab[t[u]], kSeen);
            if (h0 + u * kLgThreads + tid >= made) atomicAdd(&tab[t[u]], kOne);
          }
      }
    }
    if (a.J && tid < 64) {  // one wave keeps the list's order
      int at = 0;
      for (int j0 = 0; j0 < a.J; j0 += 64) {
        const int j = j0 + lane;
        const uint32_t t = j < a.J ? uint32_t(a.bias_ids[row * a.bis + j]) - uint32_t(base) : ~0u;
        const bool mine = t < uint32_t(n);
        const uint64_t all = __ballot(mine);
        if (mine) {
          const int to = at + int(__builtin_amdgcn_mbcnt_hi(uint32_t(all >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(all), 0)));
          bid[to] = int32_t(t);
          bval[to] = a.bias[row * a.bs + j];
          atomicOr(&tab[t], kBiased);
        }
        at += __builtin_popcountll(all);
      }
      if (lane == 0) n_bias = at;
    }
    __syncthreads();
  }

  const auto value = [](Words v, int e) {
    if constexpr (DT == WN_F32) return __builtin_bit_cast(float, uint32_t(v[e]));
    const uint16_t h = uint16_t(v[e >> 1] >> (16 * (e & 1)));
    return DT == WN_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
  };
  const auto put = [](Words& v, int e, uint32_t bits) {
    if constexpr (ES == 4) v[e] = bits;
    else v[e >> 1] = e & 1 ? (v[e >> 1] & 0xffffu) | bits << 16 : (v[e >> 1] & 0xffff0000u) | bits;
  };
  constexpr uint32_t kMinusInf = DT == WN_F32 ? 0xff800000u : DT == WN_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int i = (p * kLgThreads + tid) * PE;
    if (counted) {
      Words t[PE / 4];
#pragma unroll
      for (int q = 0; q < PE / 4; ++q) t[q] = reinterpret_cast<const Words*>(tab + i)[q];
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < PE; ++e) any |= t[e >> 2][e & 3];
      if (any) {
#pragma unroll
        for (int e = 0; e < PE; ++e) {
          const uint32_t f = t[e >> 2][e & 3];
          if (!f) continue;
          float v = value(w[p], e);
          if (f & kSeen) v = v > 0.f ? v / rep : v * rep;
          const uint32_t c = f / kOne;
          if (c) v = v - freq * float(c) - pres;
          if (f & kBiased)
            for (int j = 0; j < n_bias; ++j)
              if (bid[j] == i + e) v += bval[j];
          put(w[p], e, DT == WN_F32 ? __builtin_bit_cast(uint32_t, v) : DT == WN_BF16 ? f32_to_bf16(v) : f32_to_f16(v));
        }
      }
    }
    const uint32_t all = PE == 8 ? 0xffu : 0xfu;
    if ((ok[p] & all) != all) {
#pragma unroll
      for (int e = 0; e < PE; ++e)
        if (!(ok[p] >> e & 1)) put(w[p], e, kMinusInf);
    }
    if (i + PE <= n) {
      __builtin_memcpy(__builtin_assume_aligned(out + i * ES, ES), &w[p], 16);
    } else {
#pragma unroll
      for (int e = 0; e < PE; ++e)
        if (i + e < n) {
          if constexpr (ES == 4) *reinterpret_cast<uint32_t*>(out + (i + e) * 4) = w[p][e];
          else *reinterpret_cast<uint16_t*>(out + (i + e) * 2) = uint16_t(w[p][e >> 1] >> (16 * (e & 1)));
        }
    }
  }
}

struct LogitsPlan {
  void (*fn)(LogitsArgs);
  int seg;  // elements of a segment
};

template <int PIECES>
LogitsPlan logits_plan(int dtype) {
  const int seg = kLgThreads * PIECES * (dtype == WN_F32 ? 4 : 8);
  return {dtype == WN_F32 ? logits_kernel<WN_F32, PIECES> : dtype == WN_F16 ? logits_kernel<WN_F16, PIECES> : logits_kernel<WN_BF16, PIECES>, seg};
}

}  // namespace
}  // namespace wn

extern "C" int wn_adjust_logits(const void* logits, int dtype, int64_t stride, void* out, int64_t out_stride, int64_t N, int V,
                                const int32_t* history, int64_t history_stride, int H, const int32_t* lengths,
                                const int32_t* prompt_lengths, const float* repetition, const float* presence,
                                const float* frequency, float repetition_all, float presence_all, float frequency_all,
                                const int32_t* bias_ids, int64_t bias_ids_stride, const float* bias, int64_t bias_stride, int J,
                                const uint32_t* allowed, int64_t allowed_stride, void* stream) {
  using namespace wn;
  clear_error();
  WN_REQUIRE(N >= 0 && V > 0 && H >= 0 && H < (1 << 30) && J >= 0, WN_E_INVALID, "adjust_logits: bad sizes N=%lld V=%d H=%d J=%d",
             (long long)N, V, H, J);
  WN_REQUIRE(V <= INT32_MAX - 65536, WN_E_INVALID, "adjust_logits: V=%d", V);
  WN_REQUIRE(J <= kLgBiases, WN_E_INVALID, "adjust_logits: %d biases a row (at most %d)", J, kLgBiases);
  WN_REQUIRE(dtype >= WN_F32 && dtype <= WN_BF16, WN_E_INVALID, "adjust_logits: dtype code %d", dtype);
  if (N == 0) return WN_OK;
  const int es = dtype == WN_F32 ? 4 : 2;
  WN_REQUIRE(logits && out && (!H || history) && (!J || (bias_ids && bias)), WN_E_INVALID, "adjust_logits: null operand");
  WN_REQUIRE(stride >= 0 && history_stride >= 0 && bias_ids_stride >= 0 && bias_stride >= 0 && allowed_stride >= 0 &&
                 (out_stride >= V || N == 1),
             WN_E_INVALID, "adjust_logits: negative stride, or rows of out that overlap");
  WN_REQUIRE(aligned(logits, es) && aligned(out, es) && aligned(history, 4) && aligned(bias_ids, 4) && aligned(bias, 4) &&
                 aligned(allowed, 4) && aligned(lengths, 4) && aligned(prompt_lengths, 4) && aligned(repetition, 4) &&
                 aligned(presence, 4) && aligned(frequency, 4),
             WN_E_INVALID, "adjust_logits: operands aligned to their type");
  const LogitsPlan plan = logits_plan<4>(dtype);
  const int nseg = (V - 1) / plan.seg + 1;
  WN_REQUIRE(N <= INT32_MAX / nseg, WN_E_INVALID, "adjust_logits: grid too large");
  LogitsArgs a;
  a.x = logits;
  a.out = out;
  a.xs = stride;
  a.os = out_stride;
  a.history = H ? history : nullptr;
  a.hs = history_stride;
  a.lengths = lengths;
  a.prompt_lengths = prompt_lengths;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.rep = repetition_all;
  a.pres = presence_all;
  a.freq = frequency_all;
  a.bias_ids = bias_ids;
  a.bis = bias_ids_stride;
  a.bias = bias;
  a.bs = bias_stride;
  a.allowed = reinterpret_cast<const uint8_t*>(allowed);
  a.as = 4 * allowed_stride;
  a.V = V;
  a.H = H;
  a.J = J;
  a.nseg = nseg;
  const size_t lds = a.history || J ? size_t(plan.seg) * 4 + size_t(J) * 8 : 0;
  hipLaunchKernelGGL(plan.fn, dim3(unsigned(N * nseg)), dim3(kLgThreads), lds, static_cast<hipStream_t>(stream), a);
  return check_launch("wn_adjust_logits");
}
