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
// its own running (m, l, t), rescaled once per batch of four 16-byte pieces, while the next
// batch travels.
//
// The alternatives of a wave are a sorted list across its lanes (lane i: the i-th best),
// as 64-bit keys (value in the order of unsigned numbers, then ~index), so that one
// comparison orders equal logits too and the result does not depend on who came first. A
// batch whose largest logit cannot beat the list's bound is skipped with one comparison per
// lane; of a piece that can, only the lanes that do are looked at. An insertion costs 36
// instructions, so what counts is how few there are, and the bound is what keeps them few:
//   - it starts from the first batch: a wave's ceil(top / 4)-th largest of its lanes' maxima, the
//     least of the four waves' (at least `top` logits are no smaller);
//   - later the waves publish their ceil(top / 4)-th best: again the least of the four;
//   - where many lanes of a batch have a hit all the same (rising logits) it goes up to the
//     top-th largest of the lanes' maxima before any is inserted.
// 1,024 rows of 128,256 bf16: 46 us without alternatives (5.8 TB/s; 37 us of them are the vector
// instructions, nine an element with an exponential), 78 us with 20, whose insertions add to the
// instructions; 208 rows of 50,257 fp16, one alternative: 13.6 us and 4 for the second launch; one
// row of 128,256 fp32, five: 8.5 and 4, latency.
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

// x of the lane before (lane 0 keeps its own).
__device__ __forceinline__ uint32_t lp_before(uint32_t x) {
  return uint32_t(__builtin_amdgcn_update_dpp(int(x), int(x), 0x138, 0xf, 0xf, false));  // wave_shr:1
}

// The best keys a wave has met: lane i holds the i-th best (0: none yet).
struct LpList {
  uint64_t mine = 0, last = 0;  // last: a key must be above this to be worth taking (wave-uniform)
  int top;
  // takes every lane's key that belongs in the list
  __device__ __forceinline__ void offer(uint64_t key, int lane) {
    uint64_t hit = __ballot(key > last);
    while (hit) {
      const uint64_t k = lp_read(key, __builtin_ctzll(hit));
      const int pos = __popcll(__ballot(mine > k));
      const uint64_t up = uint64_t(lp_before(uint32_t(mine >> 32))) << 32 | lp_before(uint32_t(mine));
      mine = lane < pos ? mine : lane == pos ? k : up;
      last = max(last, lp_read(mine, top - 1));
      hit &= __ballot(key > last) & ~(hit & -hit);
    }
  }
  // at least `top` keys are known to be `bound` or above (0: nothing is known)
  __device__ __forceinline__ void raise(uint64_t bound) { last = bound ? max(last, bound - 1) : last; }
};

// The largest b, its low 44 bits 0, such that `rank` lanes have keys of b or above (0: fewer have any).
__device__ __forceinline__ uint64_t lp_bound(uint64_t key, int rank) {
  const uint32_t k = uint32_t(key >> 32);
  uint32_t b = 0;
#pragma unroll
  for (uint32_t bit = 1u << 31; bit >= 1u << 12; bit >>= 1) b = __popcll(__ballot(k >= (b | bit))) >= rank ? b | bit : b;
  return uint64_t(b) << 32;
}

// The work-group's waves agree on a bound: the least of what each has published (a rank of
// ceil(top / 4) in its own).
__device__ __forceinline__ uint64_t lp_least(const uint64_t* best) {
  uint64_t least = best[0];
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) least = min(least, best[w]);
  return lp_read(least, 0);
}

// The waves' sorted lists merged: a key's place is its place in its own list plus the keys above it
// in the others'. lists: kLpWaves of 64, out: 64, zero. Every wave calls.
__device__ __forceinline__ void lp_merge(uint64_t mine, int top, int wave, int lane, uint64_t* lists, uint64_t* out) {
  lists[wave * 64 + lane] = mine;
  __syncthreads();
  int place = lane;
#pragma unroll
  for (int o = 1; o < kLpWaves; ++o) {
    const uint64_t* l = lists + (wave + o) % kLpWaves * 64;
    int n = 0;
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) n += l[n + step - 1] > mine ? step : 0;
    place += n + (l[n] > mine);
  }
  if (mine && place < top) out[place] = mine;
  __syncthreads();
}

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

// N values into a lane's sums; their maximum `top`.
template <int N>
__device__ __forceinline__ void lp_add(const float (&x)[N], float top, LpSum& s) {
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
  __shared__ uint64_t lists[kLpWaves * 64], merged[64];
  __shared__ float sums[kLpWaves * 3];
  __shared__ uint64_t best[kLpWaves], agreed;  // of each wave, its ceil(top / 4)-th best; the bound from them
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x / a.nseg;
  const int seg = int(blockIdx.x % a.nseg);
  const T* x = static_cast<const T*>(a.x) + (row / a.inner) * a.outer_stride + (row % a.inner) * a.row_stride;
  if (wave == 0) merged[lane] = 0;

  // segments are cut where the row's memory is 16-byte aligned: element head + k seg
  const int head = min(a.V, int((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const int lo = seg == 0 ? 0 : int(min(int64_t(a.V), head + int64_t(seg) * a.seg));
  const int hi = seg == a.nseg - 1 ? a.V : int(min(int64_t(a.V), head + int64_t(seg + 1) * a.seg));
  const int body = min(hi, max(lo, head));           // first aligned element
  const int whole = body + (hi - body) / VEC * VEC;  // end of the aligned pieces

  LpSum s;
  LpList list;
  list.top = a.top;
  // batches of U pieces a wave; piece u of the batch at p starts at p + u kLpWaves STEP
  constexpr int STEP = 64 * VEC, U = 4, BATCH = U * kLpWaves * STEP;
  uint4 w[U];
  // unsigned: a position past the end may pass 2^31
  const uint32_t end = uint32_t(whole);
  auto load = [&](uint32_t p) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = p + u * kLpWaves * STEP + lane * VEC;
      if (i < end) w[u] = *reinterpret_cast<const uint4*>(x + i);
    }
  };
  auto values = [&](const uint4& q, float (&v)[VEC]) {
    const uint32_t ws[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = DT == WN_F32 ? lp_elem<DT>(ws[j], 0) : lp_elem<DT>(ws[j / 2], j & 1);
  };
  // lanes whose largest value, in a piece or batch from i on, can be among the best: no element of
  // the lane has a key above the first index's with that value
  auto hits = [&](float top, uint32_t i, bool live) {
    uint64_t hit = __ballot(live && lp_key(top, i) > list.last);
    if (__popcll(hit) > max(a.top, 8)) {
      list.raise(lp_bound(live ? lp_key(top, 0) : 0, a.top));
      hit = __ballot(live && lp_key(top, i) > list.last);
    }
    return hit;
  };
  // takes those of a piece at i0 (of lane 0), top: each lane's largest value in it
  auto collect = [&](const uint4& q, float top, uint32_t i0) {
    const uint32_t i = i0 + lane * VEC;
    const bool live = i < end;
    uint64_t hit = hits(top, i, live);
    while (hit) {
      const int from = __builtin_ctzll(hit);
      const uint32_t ws[4] = {uint32_t(__builtin_amdgcn_readlane(int(q.x), from)), uint32_t(__builtin_amdgcn_readlane(int(q.y), from)),
                              uint32_t(__builtin_amdgcn_readlane(int(q.z), from)), uint32_t(__builtin_amdgcn_readlane(int(q.w), from))};
      const int word = lane / (VEC / 4);  // lane j: element j of the piece
      const uint32_t mine = word == 0 ? ws[0] : word == 1 ? ws[1] : word == 2 ? ws[2] : ws[3];
      list.offer(lane < VEC ? lp_key(lp_elem<DT>(mine, lane & 1), i0 + from * VEC + lane) : 0, lane);
      hit &= __ballot(live && lp_key(top, i) > list.last) & ~(hit & -hit);
    }
  };
  uint32_t p = uint32_t(body) + uint32_t(wave) * STEP;
  load(p);
  const int rank = (a.top + kLpWaves - 1) / kLpWaves;
  uint64_t told = 0;
  if (a.top) {
    uint64_t first = 0;  // a bound of the lane's largest key in its first batch
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[VEC], top = -INFINITY;
      values(w[u], v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) top = fmaxf(top, v[j]);
      if (p + u * kLpWaves * STEP + lane * VEC < end) first = max(first, lp_key(top, 0xffffffffu));
    }
    told = lp_bound(first, rank);
    if (lane == 0) best[wave] = told;
    if (tid == 0) agreed = 0;
    __syncthreads();
    list.raise(lp_least(best));
  }
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
    lp_add<1>(v, v[0], s);
    if (a.top) list.offer(live ? lp_key(v[0], uint32_t(i)) : 0, lane);
  }
  for (; p < end; p += BATCH) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = w[u];
    load(p + BATCH);
    const uint64_t bound = a.top ? __hip_atomic_load(&agreed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) : 0;
    float tops[U];
    if (p + (U - 1) * kLpWaves * STEP + STEP <= end) {  // every piece is whole
      float v[U][VEC], all[U * VEC], top = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        values(q[u], v[u]);
        tops[u] = -INFINITY;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          tops[u] = fmaxf(tops[u], v[u][j]);
          all[u * VEC + j] = v[u][j];
        }
        top = fmaxf(top, tops[u]);
      }
      lp_add<U * VEC>(all, top, s);
      if (!a.top) continue;
      list.raise(lp_read(bound, 0));
      if (!hits(top, p + lane * VEC, true)) continue;
#pragma unroll
      for (int u = 0; u < U; ++u) collect(q[u], tops[u], p + u * kLpWaves * STEP);
    } else {
      if (a.top) list.raise(lp_read(bound, 0));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t i0 = p + u * kLpWaves * STEP;
        if (i0 >= end) break;
        float v[VEC], top = -INFINITY;
        values(q[u], v);
        const bool live = i0 + lane * VEC < end;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[j] = live ? v[j] : -INFINITY;
          top = fmaxf(top, v[j]);
        }
        lp_add<VEC>(v, top, s);
        if (a.top) collect(q[u], top, i0);
      }
    }
    if (a.top) {
      const uint64_t own = lp_read(list.mine, rank - 1);
      if (own > told) {
        told = own;
        if (lane == 0) __hip_atomic_store(&best[wave], own, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        uint64_t least = own;
#pragma unroll
        for (int o = 0; o < kLpWaves; ++o)
          least = min(least, o == wave ? own : __hip_atomic_load(&best[o], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
        if (lane == 0) atomicMax(reinterpret_cast<unsigned long long*>(&agreed), (unsigned long long)least);
      }
    }
  }

  // the lanes' sums, then the waves'
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s.join(__shfl_xor(s.m, o, 64), __shfl_xor(s.l, o, 64), __shfl_xor(s.t, o, 64));
  if (lane == 0) {
    sums[3 * wave] = s.m;
    sums[3 * wave + 1] = s.l;
    sums[3 * wave + 2] = s.t;
  }
  if (a.top) lp_merge(list.mine, a.top, wave, lane, lists, merged);
  else __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) s.join(sums[3 * w], sums[3 * w + 1], sums[3 * w + 2]);
  const uint64_t key = merged[lane];
  if (a.nseg == 1) {
    lp_finish(a, row, s, key, lane, lane == 0 ? lp_given<DT>(a, row, x) : 0.f);
    return;
  }
  const int64_t part = row * a.nseg + seg;
  if (lane == 0) a.part[part] = make_float4(s.m, s.l, s.t, 0.f);
  if (lane < a.top) a.keys[part * a.top + lane] = key;
}

// Joins the segments of a row: a work-group per row, a quarter of the segments' keys to a wave, with
// the bound of the waves' lanes' maxima as above.
template <int DT>
__global__ __launch_bounds__(kLpThreads) void logprobs_join_kernel(LpArgs a) {
  using T = typename LpType<DT>::T;
  __shared__ uint64_t lists[kLpWaves * 64], merged[64], best[kLpWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + (row / a.inner) * a.outer_stride + (row % a.inner) * a.row_stride;
  const int n = a.nseg * a.top;
  const uint64_t* keys = a.keys + row * n;
  constexpr int U = 4;  // kept in registers, 1,024 keys of the row; the rest is read again
  uint64_t key[U], first = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) key[u] = kLpThreads * u + tid < n ? keys[kLpThreads * u + tid] : 0;
  LpSum s;
  float given = 0.f;
  if (wave == 0) {
    if (lane == 0) given = lp_given<DT>(a, row, x);
    for (int g = lane; g < a.nseg; g += 64) {
      const float4 p = a.part[row * a.nseg + g];
      s.join(p.x, p.y, p.z);
    }
    merged[lane] = 0;
  }
  if (a.top) {
#pragma unroll
    for (int u = 0; u < U; ++u) first = max(first, key[u]);
    for (int i = kLpThreads * U + tid; i < n; i += kLpThreads) first = max(first, keys[i]);
    const uint64_t own = lp_bound(first, (a.top + kLpWaves - 1) / kLpWaves);
    if (lane == 0) best[wave] = own;
    __syncthreads();
    LpList list;
    list.top = a.top;
    list.raise(lp_least(best));
#pragma unroll
    for (int u = 0; u < U; ++u) list.offer(key[u], lane);
    for (int i = kLpThreads * U; i < n; i += kLpThreads) list.offer(i + tid < n ? keys[i + tid] : 0, lane);
    lp_merge(list.mine, a.top, wave, lane, lists, merged);
  }
  if (wave != 0) return;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s.join(__shfl_xor(s.m, o, 64), __shfl_xor(s.l, o, 64), __shfl_xor(s.t, o, 64));
  lp_finish(a, row, s, merged[lane], lane, given);
}

// Segments of a row, of 2,048 elements at least: the count that takes the least time for 1,024
// work-groups at a time (four per CU), a work-group taking the time of its elements and 2,000
// more, the second launch that of 10,000 (5 us): one, or as many as fill one to four rounds.
int lp_segments(int64_t N, int V) {
  const int64_t most = std::min<int64_t>(1024, (int64_t(V) + 2047) / 2048);
  int64_t best = 1, least = (N + 1023) / 1024 * (int64_t(V) + 2000);
  for (int64_t rounds = 1; rounds <= 4; ++rounds) {
    const int64_t n = std::min(most, 1024 * rounds / std::max<int64_t>(N, 1));
    if (n <= best) continue;
    const int64_t cost = (N * n + 1023) / 1024 * ((V + n - 1) / n + 2000) + 10000;
    if (cost < least) {
      best = n;
      least = cost;
    }
    if (n == most) break;
  }
  return int(best);
}

int64_t align256(int64_t x) { return (x + 255) & ~int64_t(255); }
int64_t lp_bytes(int64_t N, int64_t nseg, int top) { return nseg == 1 ? 0 : align256(N * nseg * 16) + N * nseg * top * 8; }

}  // namespace
}  // namespace wn

extern "C" int64_t wn_token_logprobs_workspace_bytes(int64_t N, int V, int top) {
  using namespace wn;
  if (N < 0 || V <= 0 || top < 0 || top > kTopMost || top > V) return -1;
  return lp_bytes(N, lp_segments(N, V), top);
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
  const int64_t need = lp_bytes(N, nseg, top);
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
    if (nseg > 1) hipLaunchKernelGGL(joined, join, dim3(kLpThreads), 0, st, a);
  };
  if (dtype == WN_F32) run(logprobs_kernel<WN_F32>, logprobs_join_kernel<WN_F32>);
  else if (dtype == WN_F16) run(logprobs_kernel<WN_F16>, logprobs_join_kernel<WN_F16>);
  else run(logprobs_kernel<WN_BF16>, logprobs_join_kernel<WN_BF16>);
  return check_launch("wn_token_logprobs");
}
