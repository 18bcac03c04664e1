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
// Bound: HBM, one read and one write of the logits; latency at few rows. A work-group takes a
// segment of a row, as long as there are work-groups enough: every one reads the whole history (from
// L2, but for the first). It marks the segment's touched tokens in a bitmap in LDS, counts the bits
// before each of the bitmap's words, and keeps one word per touched token, found by its rank among
// them: what the history says of it. The segment then streams through, four pieces of 16 bytes a
// thread in flight; a piece with a bit set has its touched logits adjusted one after the other.
// Counters are whole numbers, so no order of the atomics shows; biases are found by a walk over the
// segment's part of their list, which keeps its order.
// 1,024 rows of 128,256 bf16, a mask, 32 biases and histories of 2,048 to 4,096 tokens: 119 us, 4.7 TB/s
// (a copy of them 97 us, an arithmetic per element by a dense table of counts 245: some lane of a
// wave had work at each of a piece's elements); 208 rows of 50,257 fp16 14 us, one row of 128,256 fp32 6.5.
#include <algorithm>

#include "wn_common.h"

namespace wn {
namespace {

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
  int V, H, J, nseg, seg;  // seg: tokens of a segment, a multiple of 32
  int words;               // touched tokens that a segment may have
};

// A touched token's word: bit 0 seen, bit 1 on the bias list, then its count.
constexpr uint32_t kSeen = 1, kBiased = 2, kOne = 4;

// LDS of a work-group: the bitmap, the bits before each of its words, the touched tokens' words, the
// biases in reach.
constexpr int64_t logits_lds(int64_t seg, int64_t words, int64_t J) { return seg / 8 + seg / 8 + 4 * words + 8 * J; }

template <int DT, int NTHR>
__global__ __launch_bounds__(NTHR) void logits_kernel(LogitsArgs a) {
  constexpr int ES = DT == WN_F32 ? 4 : 2, PE = 16 / ES;  // elements of a piece
  constexpr int U = 4;                                    // pieces of a thread in flight
  typedef uint32_t Words __attribute__((ext_vector_type(4)));
  extern __shared__ __align__(16) uint32_t lds[];
  __shared__ int n_bias, sums[NTHR / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x / a.nseg;
  const int base = int(blockIdx.x % a.nseg) * a.seg, n = min(a.seg, a.V - base);
  const char* x = static_cast<const char*>(a.x) + (row * a.xs + base) * ES;
  char* out = static_cast<char*>(a.out) + (row * a.os + base) * ES;
  uint32_t* bits = lds;
  uint32_t* before = bits + a.seg / 32;
  uint32_t* word = before + a.seg / 32;
  int32_t* bid = reinterpret_cast<int32_t*>(word + a.words);
  float* bval = reinterpret_cast<float*>(bid + a.J);

  Words w[U];
  uint32_t ok[U];  // the mask's byte of a piece's first element
  const auto load = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = ((k0 + u) * NTHR + tid) * PE;
      w[u] = Words{0, 0, 0, 0};
      if (i + PE <= n) {
        __builtin_memcpy(&w[u], __builtin_assume_aligned(x + int64_t(i) * ES, ES), 16);
      } else {
#pragma unroll
        for (int e = 0; e < PE; ++e)
          if (i + e < n) {
            if constexpr (ES == 4) w[u][e] = reinterpret_cast<const uint32_t*>(x)[i + e];
            else w[u][e >> 1] |= uint32_t(reinterpret_cast<const uint16_t*>(x)[i + e]) << (16 * (e & 1));
          }
      }
      ok[u] = a.allowed && i < n ? a.allowed[row * a.as + ((base + i) >> 3)] >> (i & 7) : 0xffu;  // base: a multiple of 8
    }
  };
  load(0);

  const bool counted = a.history || a.J;  // uniform
  const float rep = a.repetition ? a.repetition[row] : a.rep, pres = a.presence ? a.presence[row] : a.pres,
              freq = a.frequency ? a.frequency[row] : a.freq;
  if (counted) {
    for (int i = tid; i < a.seg / 32; i += NTHR) bits[i] = 0;
    for (int i = tid; i < a.words; i += NTHR) word[i] = 0;
    __syncthreads();
    const int32_t* hist = a.history + row * a.hs;
    const int len = !a.history ? 0 : a.lengths ? min(max(a.lengths[row], 0), a.H) : a.H;
    const int made = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    // f(place, token of the segment) for the history's tokens that lie in it, a thread's F in flight
    // together; of a history of F NTHR tokens or fewer the second call has them still
    constexpr int F = 8;
    uint32_t t[F];
    const auto each = [&](bool again, auto&& f) {
      for (int h0 = 0; h0 < len; h0 += F * NTHR) {
        if (!again || len > F * NTHR) {
#pragma unroll
          for (int u = 0; u < F; ++u) {
            const int h = h0 + u * NTHR + tid;
            t[u] = h < len ? uint32_t(hist[h]) - uint32_t(base) : ~0u;
          }
        }
#pragma unroll
        for (int u = 0; u < F; ++u)
          if (t[u] < uint32_t(n)) f(h0 + u * NTHR + tid, t[u]);
      }
    };
    each(false, [&](int, uint32_t t) { atomicOr(&bits[t >> 5], 1u << (t & 31)); });
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
          atomicOr(&bits[t >> 5], 1u << (t & 31));
        }
        at += __builtin_popcountll(all);
      }
      if (lane == 0) n_bias = at;
    }
    __syncthreads();
    // the bits before each word: a thread's words one after the other, the threads' sums by waves
    const int each_of = (a.seg / 32 + NTHR - 1) / NTHR, first = tid * each_of, last = min(first + each_of, a.seg / 32);
    int mine = 0;
    for (int i = first; i < last; ++i) mine += __builtin_popcount(bits[i]);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(upto, o, 64);
      upto += lane >= o ? y : 0;
    }
    if (lane == 63) sums[tid >> 6] = upto;
    __syncthreads();
    int at = upto - mine;
    for (int i = 0; i < (tid >> 6); ++i) at += sums[i];
    for (int i = first; i < last; ++i) {
      before[i] = uint32_t(at);
      at += __builtin_popcount(bits[i]);
    }
    __syncthreads();
    const auto rank = [&](uint32_t t) { return before[t >> 5] + uint32_t(__builtin_popcount(bits[t >> 5] & ((1u << (t & 31)) - 1))); };
    each(true, [&](int h, uint32_t t) {
      uint32_t* to = &word[rank(t)];
      atomicOr(to, kSeen);
      if (h >= made) atomicAdd(to, kOne);
    });
    if (a.J)
      for (int j = tid; j < n_bias; j += NTHR) atomicOr(&word[rank(uint32_t(bid[j]))], kBiased);
    __syncthreads();
  }

  constexpr uint32_t kMinusInf = DT == WN_F32 ? 0xff800000u : DT == WN_BF16 ? 0xff80u : 0xfc00u;
  const auto put = [](Words& v, int e, uint32_t b) {
    if constexpr (ES == 4) v[e] = b;
    else v[e >> 1] = e & 1 ? (v[e >> 1] & 0xffffu) | b << 16 : (v[e >> 1] & 0xffff0000u) | b;
  };
  const int pieces = (n + PE - 1) / PE;
  for (int k0 = 0; k0 * NTHR < pieces; k0 += U) {
    Words v[U];
    uint32_t allow[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = w[u];
      allow[u] = ok[u];
    }
    if ((k0 + U) * NTHR < pieces) load(k0 + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = ((k0 + u) * NTHR + tid) * PE;
      if (i >= n) continue;
      if (counted) {
        const uint32_t mask = bits[i >> 5], in = mask >> (i & 31) & ((1u << PE) - 1);
        if (in) {
          uint32_t r = before[i >> 5] + uint32_t(__builtin_popcount(mask & ((1u << (i & 31)) - 1)));
          for (uint32_t left = in; left; left &= left - 1, ++r) {
            const int e = __builtin_ctz(left);
            const uint32_t f = word[r], c = f / kOne;
            // element e, chosen by value: an index into registers would send them through memory
            uint32_t raw = v[u][0];
#pragma unroll
            for (int q = 1; q < 4; ++q) raw = (e * ES) >> 2 == q ? v[u][q] : raw;
            float y;
            if constexpr (DT == WN_F32) y = __builtin_bit_cast(float, raw);
            else y = DT == WN_BF16 ? bf16_to_f32(uint16_t(raw >> (16 * (e & 1)))) : f16_to_f32(uint16_t(raw >> (16 * (e & 1))));
            if (f & kSeen) y = y > 0.f ? y / rep : y * rep;
            if (c) y = y - freq * float(c) - pres;
            if (f & kBiased)
              for (int j = 0; j < n_bias; ++j)
                if (bid[j] == i + e) y += bval[j];
            uint32_t b;
            if constexpr (DT == WN_F32) {
              b = __builtin_bit_cast(uint32_t, y);
            } else {
              b = DT == WN_BF16 ? f32_to_bf16(y) : f32_to_f16(y);
              b = e & 1 ? (raw & 0xffffu) | b << 16 : (raw & 0xffff0000u) | b;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) v[u][q] = (e * ES) >> 2 == q ? b : v[u][q];
          }
        }
      }
      constexpr uint32_t kAll = (1u << PE) - 1;
      if ((allow[u] & kAll) != kAll) {
#pragma unroll
        for (int e = 0; e < PE; ++e)
          if (!(allow[u] >> e & 1)) put(v[u], e, kMinusInf);
      }
      if (i + PE <= n) {
        __builtin_memcpy(__builtin_assume_aligned(out + int64_t(i) * ES, ES), &v[u], 16);
      } else {
#pragma unroll
        for (int e = 0; e < PE; ++e)
          if (i + e < n) {
            if constexpr (ES == 4) reinterpret_cast<uint32_t*>(out)[i + e] = v[u][e];
            else reinterpret_cast<uint16_t*>(out)[i + e] = uint16_t(v[u][e >> 1] >> (16 * (e & 1)));
          }
      }
    }
  }
}

struct LogitsPlan {
  void (*fn)(LogitsArgs);
  int threads;
  int seg;  // tokens of a segment
};

// Touched tokens that a segment may have.
int logits_words(int seg, int H, int J) { return int(std::min<int64_t>(seg, int64_t(H) + J)); }

// Two work-groups a CU where segments of 4,096 tokens and more give them; longer ones, which read the
// history less often, up to 45,056 and what 64 KB of LDS hold. V = 128,256, bf16, H = 4,096, by segment, us:
// 1 row 4,096: 6.7, 16,384: 9.8; 64 rows 8,192: 16.4, 16,384: 16.0, 32,768: 17.6; 1,024 rows 16,384: 161,
// 32,768: 128, 43,000: 127, 65,536: 129. With four waves or sixteen in a work-group: 9 and 11% more at 1,024 rows.
LogitsPlan pick_logits(int dtype, int64_t N, int V, int H, int J) {
  const int64_t most = (int64_t(V) + 4095) / 4096, wanted = (2 * std::max(1, device_cus()) + N - 1) / N;
  int64_t nseg = std::max<int64_t>((int64_t(V) + 45055) / 45056, std::min(wanted, most));
  int seg;
  do {
    seg = int(((V + nseg - 1) / nseg + 63) / 64 * 64);
    ++nseg;
  } while ((H || J) && logits_lds(seg, logits_words(seg, H, J), J) > 65536 - 256);
  constexpr int NTHR = 512;
  return {dtype == WN_F32 ? logits_kernel<WN_F32, NTHR> : dtype == WN_F16 ? logits_kernel<WN_F16, NTHR> : logits_kernel<WN_BF16, NTHR>, NTHR, seg};
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
  const LogitsPlan plan = pick_logits(dtype, N, V, H, J);
  const int nseg = (V - 1) / plan.seg + 1;
  WN_REQUIRE(N <= INT32_MAX / nseg && grid_fits(N * nseg, plan.threads), WN_E_INVALID, "adjust_logits: grid too large");
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
  a.seg = plan.seg;
  a.words = logits_words(plan.seg, H, J);
  const size_t lds = H || J ? size_t(logits_lds(plan.seg, a.words, J)) : 0;
  hipLaunchKernelGGL(plan.fn, dim3(unsigned(N * nseg)), dim3(plan.threads), lds, static_cast<hipStream_t>(stream), a);
  return check_launch("wn_adjust_logits");
}
