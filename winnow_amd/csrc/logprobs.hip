// Log probabilities of given tokens, with the entropy and the most likely alternatives of
// every row of logits, in one pass over them.
//
//   m = max x,  l = sum e^(x - m),  t = sum (x - m) e^(x - m)
//   logprob(i) = x_i - m - log l,   entropy = log l - t / l
//   alternatives: the `top` largest logits, equal ones by the lowest index first.
//
// Both terms of the entropy are positive, so nothing cancels. Sums are fp32, per lane
// first, so a sum over 2^17 tokens adds some 500 terms in a row and then a tree.
//
// Bound: HBM, one read of the logits. A work-group of four waves takes a row, or a segment
// of it where there are few rows (a second launch then joins the segments): each lane keeps
// its own running (m, l, t), rescaled once per 16-byte piece.
//
// The alternatives of a wave are a sorted list across its lanes (lane i: the i-th best),
// as 64-bit keys (value in the order of unsigned numbers, then ~index), so that one
// comparison orders equal logits too and the result does not depend on who came first. A
// piece whose largest logit cannot beat the list's last is skipped with one comparison per
// lane; the waves of a work-group share the best of their last keys, each of which is a
// lower bound of the row's.
#include <algorithm>

#include "wn_common.h"

namespace wn {
namespace {

constexpr int kTopMost = 64;     // alternatives: a list is one wave's lanes
constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;

struct LpArgs {
  const void* x;
  int64_t row_stride;   // elements
  int64_t outer_stride; // of a block of `inner` rows
  int inner;
  const int64_t* tokens;  // null: no given tokens
  float* logprob;
  float* entropy;
  float* top_lp;   // (N, top)
  int64_t* top_id;
  float4* part;    // (N, nseg): m, l, t, -
  uint64_t* keys;  // (N, nseg, top)
  int64_t N;
  int V, top, nseg, seg;  // seg: elements of a segment
};

// A logit as an unsigned number in its order; -0 and 0 alike, NaN above everything.
__device__ __forceinline__ uint32_t lp_order(float x) {
  uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t i) { return uint64_t(lp_order(x)) << 32 | ~i; }

__device__ __forceinline__ uint64_t lp_read(uint64_t v, int lane) {
  return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(v >> 32), lane))) << 32 |
         uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), lane));
}

// The best keys a wave has met: lane i holds the i-th best (0: none yet).
struct LpList {
  uint64_t mine = 0, last = 0;  // last: the least key worth taking is above this (wave-uniform)
  int top;
  // takes every lane's key that belongs in the list
  __device__ __forceinline__ void offer(uint64_t key, int lane) {
    uint64_t hit = __ballot(key > last);
    while (hit) {
      const uint64_t k = lp_read(key, __builtin_ctzll(hit));
      hit &= hit - 1;
      if (k <= last) continue;  // wave-uniform: the list has moved on
      const int pos = __popcll(__ballot(mine > k));
      const uint64_t up = __shfl_up(mine, 1, 64);
      mine = lane < pos ? mine : lane == pos ? k : up;
      last = max(last, lp_read(mine, top - 1));
    }
  }
};

struct LpSum {
  float m = -INFINITY, l = 0.f, t = 0.f;
  // joins o: both relative to the larger maximum
  __device__ __forceinline__ void join(float om, float ol, float ot) {
    const float M = fmaxf(m, om);
    const float da = m == -INFINITY ? 0.f : m - M, db = om == -INFINITY ? 0.f : om - M;
    const float wa = __builtin_amdgcn_exp2f(da * kLog2e), wb = __builtin_amdgcn_exp2f(db * kLog2e);
    // a difference that overflowed has weight 0: its share is left out, not 0 times infinity
    const float ta = wa > 0.f ? wa * (t + da * l) : 0.f, tb = wb > 0.f ? wb * (ot + db * ol) : 0.f;
    l = wa * l + wb * ol;
    t = ta + tb;
    m = M;
  }
};

template <int DT>
struct LpType {
  using T = uint16_t;
  static constexpr int VEC = 8;
};
template <>
struct LpType<WN_F32> {
  using T = float;
  static constexpr int VEC = 4;
};
template <int DT>
__device__ __forceinline__ float lp_elem(uint32_t w, int half) {
  if constexpr (DT == WN_F32) return __builtin_bit_cast(float, w);
  else if constexpr (DT == WN_BF16) return __builtin_bit_cast(float, half ? w & 0xffff0000u : w << 16);
  else return f16_to_f32(uint16_t(half ? w >> 16 : w));
}

// N values (those of x at index i0 ..) into a lane's sums and the wave's list.
template <int N>
__device__ __forceinline__ void lp_take(const float (&x)[N], uint32_t i0, int n, LpSum& s, LpList& list, int lane) {
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < N; ++j) top = fmaxf(top, x[j]);  // what lies past n is -inf
  const float mn = fmaxf(s.m, top);
  const float mz = mn == -INFINITY ? 0.f : mn;
  const float d0 = s.m == -INFINITY ? 0.f : s.m - mz;
  const float f = __builtin_amdgcn_exp2f(d0 * kLog2e);
  s.t = f > 0.f ? f * (s.t + d0 * s.l) : 0.f;
  s.l *= f;
  s.m = mn;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float d = x[j] - mz, p = __builtin_amdgcn_exp2f(d * kLog2e);
    s.l += p;
    s.t = fmaf(p, fmaxf(d, -1000.f), s.t);  // e^-1000 is 0: -inf and overflows add nothing
  }
  if (list.top) {
    if (__any(n > 0 && lp_key(top, i0) > list.last)) {  // no element of the piece has a better key
#pragma unroll
      for (int j = 0; j < N; ++j) list.offer(j < n ? lp_key(x[j], i0 + j) : 0, lane);
    }
  }
}

__device__ __forceinline__ float lp_nan() { return __builtin_bit_cast(float, 0x7fc00000u); }

// The row's answers from its sums (wave 0 of a work-group; every lane has them) and list.
__device__ __forceinline__ void lp_finish(const LpArgs& a, int64_t row, const LpSum& s, uint64_t key, int lane, float given) {
  const float ll = logf(s.l);
  if (lane == 0) {
    if (a.tokens) a.logprob[row] = (given - s.m) - ll;
    if (a.entropy) a.entropy[row] = ll - s.t / s.l;
  }
  if (lane < a.top) {
    a.top_lp[row * a.top + lane] = (lp_value(uint32_t(key >> 32)) - s.m) - ll;
    a.top_id[row * a.top + lane] = int64_t(~uint32_t(key));
  }
}

template <int DT>
__device__ __forceinline__ float lp_given(const LpArgs& a, int64_t row, const typename LpType<DT>::T* x) {
  if (!a.tokens) return 0.f;
  const int64_t tok = a.tokens[row];
  if (tok < 0 || tok >= a.V) return lp_nan();  // no token of the row: nothing is read
  if constexpr (DT == WN_F32) return x[tok];
  else return lp_elem<DT>(x[tok], 0);
}

template <int DT>
__global__ __launch_bounds__(kLpThreads) void logprobs_kernel(LpArgs a) {
  using T = typename LpType<DT>::T;
  constexpr int VEC = LpType<DT>::VEC;
  __shared__ uint64_t lists[kLpWaves * kTopMost];
  __shared__ float sums[kLpWaves * 3];
  __shared__ uint64_t floor_key;  // the largest `last` of the work-group's waves
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.nseg;
  const int seg = int(blockIdx.x % a.nseg);
  const T* x = static_cast<const T*>(a.x) + (row / a.inner) * a.outer_stride + (row % a.inner) * a.row_stride;
  if (tid == 0) floor_key = 0;
  __syncthreads();

  // segments are cut where the row's memory is 16-byte aligned: element head + k seg
  const int head = min(a.V, int((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const int lo = seg == 0 ? 0 : int(min(int64_t(a.V), head + int64_t(seg) * a.seg));
  const int hi = seg == a.nseg - 1 ? a.V : int(min(int64_t(a.V), head + int64_t(seg + 1) * a.seg));
  const int body = min(hi, max(lo, head));           // first aligned element
  const int whole = body + (hi - body) / VEC * VEC;  // end of the aligned pieces

  LpSum s;
  LpList list;
  list.top = a.top;
  auto share = [&]() {
    if (!a.top) return;
    const uint64_t f = lp_read(__hip_atomic_load(&floor_key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP), 0);
    if (f < list.last) {
      if (lane == 0) atomicMax(reinterpret_cast<unsigned long long*>(&floor_key), (unsigned long long)list.last);
    } else {
      list.last = f;
    }
  };
  // the ends, at most 2 VEC - 2 elements: one per lane of wave 0
  if (wave == 0) {
    const int before = body - lo, after = hi - whole;
    const int i = lane < before ? lo + lane : whole + (lane - before);
    const bool live = lane < before + after;
    float v[1] = {-INFINITY};
    if (live) {
      if constexpr (DT == WN_F32) v[0] = x[i];
      else v[0] = lp_elem<DT>(x[i], 0);
    }
    lp_take<1>(v, uint32_t(i), live ? 1 : 0, s, list, lane);
  }
  constexpr int STEP = 64 * VEC;  // a wave's piece of the row
  for (int p = body + wave * STEP; p < whole; p += kLpWaves * STEP) {
    const int i = p + lane * VEC;
    float v[VEC];
    const bool live = i < whole;
    if (live) {
      const uint4 w = *reinterpret_cast<const uint4*>(x + i);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = DT == WN_F32 ? lp_elem<DT>(ws[j], 0) : lp_elem<DT>(ws[j / 2], j & 1);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = -INFINITY;
    }
    lp_take<VEC>(v, uint32_t(i), live ? VEC : 0, s, list, lane);
    share();
  }

  // the lanes' sums, then the waves'
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s.join(__shfl_xor(s.m, o, 64), __shfl_xor(s.l, o, 64), __shfl_xor(s.t, o, 64));
  if (lane == 0) {
    sums[3 * wave] = s.m;
    sums[3 * wave + 1] = s.l;
    sums[3 * wave + 2] = s.t;
  }
  lists[wave * kTopMost + lane] = list.mine;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) s.join(sums[3 * w], sums[3 * w + 1], sums[3 * w + 2]);
  if (a.top) {
    list.last = lp_read(list.mine, a.top - 1);
    for (int w = 1; w < kLpWaves; ++w) list.offer(lane < a.top ? lists[w * kTopMost + lane] : 0, lane);
  }
  if (a.nseg == 1) {
    lp_finish(a, row, s, list.mine, lane, lane == 0 ? lp_given<DT>(a, row, x) : 0.f);
    return;
  }
  const int64_t part = row * a.nseg + seg;
  if (lane == 0) a.part[part] = make_float4(s.m, s.l, s.t, 0.f);
  if (lane < a.top) a.keys[part * a.top + lane] = list.mine;
}

// Joins the segments of a row: one wave per row.
template <int DT>
__global__ __launch_bounds__(64) void logprobs_join_kernel(LpArgs a) {
  using T = typename LpType<DT>::T;
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + (row / a.inner) * a.outer_stride + (row % a.inner) * a.row_stride;
  const float given = lane == 0 ? lp_given<DT>(a, row, x) : 0.f;
  LpSum s;
  for (int g = lane; g < a.nseg; g += 64) {
    const float4 p = a.part[row * a.nseg + g];
    s.join(p.x, p.y, p.z);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s.join(__shfl_xor(s.m, o, 64), __shfl_xor(s.l, o, 64), __shfl_xor(s.t, o, 64));
  LpList list;
  list.top = a.top;
  const int n = a.nseg * a.top;
  for (int i0 = 0; i0 < n; i0 += 64) list.offer(i0 + lane < n ? a.keys[row * n + i0 + lane] : 0, lane);
  lp_finish(a, row, s, list.mine, lane, given);
}

// Segments of a row: one for as many rows as fill the device with a few work-groups per
// CU, else as many as that takes, of 2,048 elements at least.
int lp_segments(int64_t N, int V) {
  const int64_t want = (1024 + N - 1) / std::max<int64_t>(N, 1);
  return int(std::max<int64_t>(1, std::min<int64_t>(want, (int64_t(V) + 2047) / 2048)));
}

int64_t align256(int64_t x) { return (x + 255) & ~int64_t(255); }

}  // namespace
}  // namespace wn

extern "C" int64_t wn_token_logprobs_workspace_bytes(int64_t N, int V, int top) {
  using namespace wn;
  if (N < 0 || V <= 0 || top < 0 || top > kTopMost || top > V) return -1;
  const int nseg = lp_segments(N, V);
  return nseg == 1 ? 0 : align256(N * nseg * 16) + N * nseg * top * 8;
}

extern "C" int wn_token_logprobs(const void* logits, int dtype, int64_t stride_outer, int64_t stride_inner, int64_t inner,
                                 const int64_t* tokens, float* logprob, float* entropy, float* top_logprobs,
                                 int64_t* top_ids, int64_t N, int V, int top, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  using namespace wn;
  clear_error();
  WN_REQUIRE(N >= 0 && V > 0 && inner > 0 && inner <= INT32_MAX, WN_E_INVALID, "logprobs: bad sizes N=%lld V=%d inner=%lld",
             (long long)N, V, (long long)inner);
  WN_REQUIRE(dtype >= WN_F32 && dtype <= WN_BF16, WN_E_INVALID, "logprobs: dtype code %d", dtype);
  WN_REQUIRE(top >= 0 && top <= kTopMost && top <= V, WN_E_INVALID, "logprobs: top %d (0 .. %d, at most V)", top, kTopMost);
  if (N == 0) return WN_OK;
  WN_REQUIRE(logits && !tokens == !logprob && (!top || (top_logprobs && top_ids)), WN_E_INVALID, "logprobs: null operand");
  WN_REQUIRE(aligned(logits, dtype == WN_F32 ? 4 : 2), WN_E_INVALID, "logprobs: logits are not aligned to their type");
  const int nseg = lp_segments(N, V);
  const int64_t need = wn_token_logprobs_workspace_bytes(N, V, top);
  WN_REQUIRE(nseg == 1 || (workspace && workspace_bytes >= need && aligned(workspace, 256)), WN_E_WORKSPACE,
             "logprobs: workspace needs %lld bytes, 256-aligned (got %lld)", (long long)need, (long long)workspace_bytes);
  WN_REQUIRE(N * nseg < (int64_t(1) << 31), WN_E_INVALID, "logprobs: grid too large");
  LpArgs a;
  a.x = logits;
  a.row_stride = stride_inner;
  a.outer_stride = stride_outer;
  a.inner = int(inner);
  a.tokens = tokens;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_lp = top_logprobs;
  a.top_id = top_ids;
  a.part = static_cast<float4*>(workspace);
  a.keys = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + align256(N * nseg * 16));
  a.N = N;
  a.V = V;
  a.top = top;
  a.nseg = nseg;
  a.seg = int(((int64_t(V) + nseg - 1) / nseg + 63) / 64 * 64);  // whole 16-byte pieces
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(unsigned(N * nseg)), join(static_cast<unsigned>(N));
  auto run = [&](auto scan, auto joined) {
    hipLaunchKernelGGL(scan, grid, dim3(kLpThreads), 0, st, a);
    if (nseg > 1) hipLaunchKernelGGL(joined, join, dim3(64), 0, st, a);
  };
  if (dtype == WN_F32) run(logprobs_kernel<WN_F32>, logprobs_join_kernel<WN_F32>);
  else if (dtype == WN_F16) run(logprobs_kernel<WN_F16>, logprobs_join_kernel<WN_F16>);
  else run(logprobs_kernel<WN_BF16>, logprobs_join_kernel<WN_BF16>);
  return check_launch("wn_token_logprobs");
}
