// Routing of tokens to experts: scores, group-limited top-k and weights from router logits, the gradient of the weights
// with respect to the logits, and the tables of the grouped GEMM's layouts that follow from the routing.
//
// Callers of the reference do these steps with torch softmax / topk / sort / bincount
// (asym_gemm/unified_moe/runtime.py:1422-1476).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <cstdint>

#include "../../include/asymgemm_b200.h"

int agb_fail(int code, const char* message);
int agb_device_sm_count(int* out);

namespace agb {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kRouteMaxTopK = 32;       // one lane of the token's warp per chosen expert
constexpr int kRouteMaxPerLane = 32;    // experts held by one lane
constexpr int kLayoutMaxExperts = 1024;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float warp_max_f(float v) {
  float r;   // sm_100a reduces floats across the warp in one instruction
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ float reciprocal(float x) {      // 1 ulp, 0 for infinity
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A logit as the router counts it: NaN and -inf switch the expert off, +inf is the largest finite number.
__device__ __forceinline__ float clean(float l) { return fminf(fmaxf(l, -INFINITY), FLT_MAX); }   // max(NaN, x) = x

// Where a row's experts lie: every group on 1 << shift neighbouring lanes, per_lane consecutive experts on each.
struct LaneMap {
  int shift, per_lane;
  int vector_rows, vector_bias;      // every lane's experts are full and 16-byte aligned in the logits / the bias:
  int lane_shift;                    // then per_lane = 1 << lane_shift
};

struct RouteParams {
  const void* logits;
  const float* bias;
  const int* rows_used;
  long long* ids;
  float* weights;
  long long tokens, ld;
  int experts, top_k, groups, top_groups, group_size;
  int sigmoid, group_max, renormalize;
  LaneMap warp;       // one row on the 32 lanes of a warp
  LaneMap part;       // route_top8_kernel: one row on row_lanes lanes
  int row_lanes, index_bits;
  float scale;
};

// ------------------------------------------------------------------------------------------------ forward
// Two kernels. route_topk_kernel (top_k above 8): one warp per token (route_row). The lane order is the expert order, a group's two
// best scores are a short shuffle reduction, and "lowest index among equals" is "lowest lane, then lowest slot". Each lane sorts its experts once (lists of 8, as 32-bit keys that carry the slot in
// their lowest bits); the k best are then taken off the heads of the lists, one warp-wide integer maximum and one predicated
// shift each. route_top8_kernel, below, has several tokens per warp. Both are bound by the instructions they issue, not by
// memory (figures at launch_route).
//
// Order. Keys are scores in fp32, cut off at the slot bits; `tol` bounds what they are off by. A token with two neighbours in
// the order, or two groups at the border, closer than that -- one in a few hundred -- is decided once more in 64 bits
// (route_exact), unless the two have equal logits and biases, whose order is by index in any arithmetic. The result is that of
// the formulas whatever the last bits of the exponentials are.
struct Slots {
  int first, count;      // this lane holds the experts first .. first + count - 1
  __device__ __forceinline__ Slots(const RouteParams& p, const LaneMap& map, int lane) {
    const int g = lane >> map.shift, in = (lane & ((1 << map.shift) - 1)) * map.per_lane;
    first = g * p.group_size + in;
    count = g < p.groups ? max(0, min(map.per_lane, p.group_size - in)) : 0;
  }
};

// The same selection in 64 bits: returns the expert chosen i-th on lane i (-1: none left). Every loop is rolled: it runs for a few
// rows per million, and its size is all that the others see of it (65536 x 256: 53 us inlined so, 57 as a called function, whose
// calling convention the whole kernel pays for). Where every row comes here -- logits that are all equal, as before training, or
// sigmoids that are saturated -- the same call takes 264 to 293 us.
template <typename T>
__device__ __forceinline__ int route_exact(const RouteParams& p, const T* row, int lane) {
  const Slots at(p, p.warp, lane);
  double c[kRouteMaxPerLane], mx = -INFINITY, sum = 0;
  auto logit = [&](int j) { return static_cast<double>(clean(to_float(row[at.first + j]))); };
  auto everyone = [&](double v, auto join) {
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(kAll, v, o));
    return v;
  };
  auto larger = [](double a, double b) { return fmax(a, b); };
#pragma unroll 1
  for (int j = 0; j < at.count; ++j) mx = fmax(mx, logit(j));
  if (!p.sigmoid) mx = everyone(mx, larger);
#pragma unroll 1
  for (int j = 0; j < at.count; ++j) {
    const double l = logit(j), e = exp(p.sigmoid ? -l : l - mx);
    c[j] = l == -INFINITY ? -INFINITY : p.sigmoid ? 1 / (1 + e) : e;
    if (l > -INFINITY) sum += e;
  }
  if (!p.sigmoid) sum = everyone(sum, [](double a, double b) { return a + b; });
  double a1 = -INFINITY, a2 = -INFINITY;
#pragma unroll 1
  for (int j = 0; j < at.count; ++j) {
    if (!p.sigmoid) c[j] /= sum;
    if (p.bias != nullptr) c[j] += static_cast<double>(clean(p.bias[at.first + j]));      // -inf on either side: off
    a2 = fmax(a2, fmin(a1, c[j]));
    a1 = fmax(a1, c[j]);
  }
  bool kept = true;
  if (p.groups > 1) {
#pragma unroll 1
    for (int o = 1; o < (1 << p.warp.shift); o <<= 1) {
      const double b1 = __shfl_xor_sync(kAll, a1, o), b2 = __shfl_xor_sync(kAll, a2, o);
      a2 = fmax(fmax(a2, b2), fmin(a1, b1));
      a1 = fmax(a1, b1);
    }
    const double mine = p.group_max || a2 == -INFINITY ? a1 : a1 + a2;
    const int g = lane >> p.warp.shift;
    int rank = 0;
#pragma unroll 1
    for (int o = 0; o < p.groups; ++o) {
      const double other = __shfl_sync(kAll, mine, o << p.warp.shift);
      rank += other > mine || (other == mine && o < g);
    }
    kept = rank < p.top_groups;
  }
  // without a bias the scores rise with the logits: among the groups kept, the logits themselves are the exact order
#pragma unroll 1
  for (int j = 0; j < at.count; ++j) c[j] = !kept ? -INFINITY : p.bias == nullptr && c[j] > -INFINITY ? logit(j) : c[j];
  int chosen = -1;
#pragma unroll 1
  for (int i = 0; i < p.top_k; ++i) {
    double m = -INFINITY;
    int slot = 0;
#pragma unroll 1
    for (int j = 0; j < at.count; ++j) {
      if (c[j] > m) {
        m = c[j];
        slot = j;
      }
    }
    const double best = everyone(m, larger);
    if (best == -INFINITY) break;
    const int w = __ffs(__ballot_sync(kAll, m == best)) - 1, e = __shfl_sync(kAll, at.first + slot, w);
    if (lane == w) c[slot] = -INFINITY;
    if (lane == i) chosen = e;
  }
  return chosen;
}

// Slots of one lane from a row of logits or the bias. `vector`: every lane's slots are full and 16-byte aligned.
template <typename T, int VPL>
__device__ __forceinline__ void load_slots(bool vector, const T* row, const Slots& at, float (&l)[VPL]) {
  constexpr int kBytes = VPL * static_cast<int>(sizeof(T));
  if constexpr (kBytes >= 16) {
    if (vector) {
#pragma unroll
      for (int q = 0; q < kBytes / 16; ++q) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (at.count > 0) v = __ldg(reinterpret_cast<const uint4*>(row + at.first) + q);
        const T* t = reinterpret_cast<const T*>(&v);
        constexpr int kPer = 16 / static_cast<int>(sizeof(T));
#pragma unroll
        for (int i = 0; i < kPer; ++i) l[q * kPer + i] = at.count > 0 ? clean(to_float(t[i])) : -INFINITY;
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < VPL; ++j) l[j] = j < at.count ? clean(to_float(row[at.first + j])) : -INFINITY;
}

// Order-preserving map of floats to signed integers (its own inverse). -inf, "off", maps below every live key.
__device__ __forceinline__ int32_t key_of(float v) {
  const int32_t u = __float_as_int(v + 0.f);        // -0 and 0 are equal
  return u ^ ((u >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float value_of(int32_t key) { return __int_as_float(key ^ ((key >> 31) & 0x7fffffff)); }
constexpr int32_t kOffKeys = static_cast<int32_t>(0x807fffffu);      // keys of -inf with any slot bits are not above this

__device__ __forceinline__ void order(int32_t& a, int32_t& b) {
  const int32_t hi = max(a, b);
  b = min(a, b);
  a = hi;
}
// Batcher's odd-even merge sort, largest first.
template <int N>
__device__ __forceinline__ void sort_list(int32_t (&s)[N]) {
  if constexpr (N >= 2) {
#pragma unroll
    for (int i = 0; i < N; i += 2) order(s[i], s[i + 1]);
  }
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      order(s[i], s[i + 2]);
      order(s[i + 1], s[i + 3]);
      order(s[i + 1], s[i + 2]);
    }
  }
  if constexpr (N == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) order(s[i], s[i + 4]);
    order(s[2], s[4]);
    order(s[3], s[5]);
    order(s[1], s[2]);
    order(s[3], s[4]);
    order(s[5], s[6]);
  }
}

// The selection for one row on a whole warp: returns the expert chosen i-th on lane i (-1: none left), and, where a softmax over
// the whole row was taken, its maximum and sum.
template <typename T, int VPL>
__device__ __forceinline__ int route_row(const RouteParams& p, const T* row, int lane, float& row_max, float& sum) {
  constexpr int kLen = VPL < 8 ? VPL : 8, kLists = VPL / kLen;
  constexpr int32_t kSlotMask = VPL - 1;      // key bits that hold VPL - 1 - slot
  const bool scored = p.bias != nullptr || p.groups > 1;      // the order needs the scores, not just the logits
  const Slots at(p, p.warp, lane);
  float c[VPL];      // what the experts are ordered by; -inf = off
  load_slots<T, VPL>(p.warp.vector_rows, row, at, c);
  row_max = sum = 0.f;
  if (!p.sigmoid && (scored || !p.renormalize)) {
    float mx = c[0];
#pragma unroll
    for (int j = 1; j < VPL; ++j) mx = fmaxf(mx, c[j]);
    row_max = warp_max_f(mx);
#pragma unroll
    for (int j = 0; j < VPL; ++j) sum += c[j] > -INFINITY ? __expf(c[j] - row_max) : 0.f;
    sum = warp_sum_f(sum);
  }
  bool unsure = false;
  float tol = 0.f;
  if (scored) {
    float s[VPL];
    const float inv = 1.f / sum;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      s[j] = p.sigmoid ? __fdividef(1.f, 1.f + __expf(-c[j])) : __expf(c[j] - row_max) * inv;
    }
    bool any_off = false;      // rare, so the common row has no select per expert
#pragma unroll
    for (int j = 0; j < VPL; ++j) any_off = any_off || c[j] == -INFINITY;
    // Error of a score. Sigmoid: s (1 - s) |l| 2^-23 from the exponential's argument, a few roundings of a number <= 1.
    // Softmax, of numbers <= 1 / sum: d e^-d 2^-23 for l = max - d, and up to 37 additions in the sum.
    tol = p.sigmoid ? 0x1p-20f : 0x1p-18f * inv;
    if (p.bias != nullptr) {
      float bias[VPL];
      load_slots<float, VPL>(p.warp.vector_bias, p.bias, at, bias);
#pragma unroll
      for (int j = 0; j < VPL; ++j) s[j] += bias[j];      // a bias of -inf switches the expert off by itself
    }
    if (any_off) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) s[j] = c[j] == -INFINITY ? -INFINITY : s[j];
    }
    if (p.groups > 1) {
      float a1 = -INFINITY, a2 = -INFINITY;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        a2 = fmaxf(a2, fminf(a1, s[j]));
        a1 = fmaxf(a1, s[j]);
      }
      for (int o = 1; o < (1 << p.warp.shift); o <<= 1) {
        const float b1 = __shfl_xor_sync(kAll, a1, o), b2 = __shfl_xor_sync(kAll, a2, o);
        a2 = fmaxf(fmaxf(a2, b2), fminf(a1, b1));
        a1 = fmaxf(a1, b1);
      }
      const float mine = p.group_max || a2 == -INFINITY ? a1 : a1 + a2;
      const int g = lane >> p.warp.shift;
      int rank = 0;
      for (int o = 0; o < p.groups; ++o) {
        const float other = __shfl_sync(kAll, mine, o << p.warp.shift);
        rank += other > mine || (other == mine && o < g);
      }
      const bool kept = rank < p.top_groups, real = g < p.groups;
      // the weakest group kept against the strongest one left out
      const float low = -warp_max_f(real && kept ? -mine : -INFINITY), high = warp_max_f(real && !kept ? mine : -INFINITY);
      if (high > -INFINITY) unsure = !(low - high > 4.f * tol + 0x1p-20f * (fabsf(low) + fabsf(high)));
      if (!kept) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) s[j] = c[j] = -INFINITY;
      }
    }
    if (p.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < VPL; ++j) c[j] = s[j];
    }
  }

  int32_t list[kLists][kLen];
#pragma unroll
  for (int j = 0; j < VPL; ++j) list[j / kLen][j % kLen] = (key_of(c[j]) & ~kSlotMask) | (VPL - 1 - j);
#pragma unroll
  for (int q = 0; q < kLists; ++q) sort_list<kLen>(list[q]);

  int32_t my_key = kOffKeys;      // lane i: the key and lane of the expert taken i-th
  int my_lane = 0;
  auto head = [&] {
    int32_t h = list[0][0];
#pragma unroll
    for (int q = 1; q < kLists; ++q) h = max(h, list[q][0]);
    return h;
  };
  // The best head by value, of equal ones the lowest lane's (the slot bits order experts within a lane only).
  auto take_best = [&](int32_t h, int& w) {
    const int32_t value = __reduce_max_sync(kAll, h & ~kSlotMask);
    w = __ffs(__ballot_sync(kAll, (h & ~kSlotMask) == value)) - 1;
    return __shfl_sync(kAll, h, w);
  };
  for (int i = 0; i < p.top_k; ++i) {
    int w;
    const int32_t best = take_best(head(), w);
    if (best <= kOffKeys) break;
#pragma unroll
    for (int q = 0; q < kLists; ++q) {
      const bool pop = lane == w && list[q][0] == best;
#pragma unroll
      for (int j = 0; j + 1 < kLen; ++j) list[q][j] = pop ? list[q][j + 1] : list[q][j];
      list[q][kLen - 1] = pop ? INT32_MIN : list[q][kLen - 1];
    }
    if (lane == i) {
      my_key = best;
      my_lane = w;
    }
  }
  auto expert_of = [&](int32_t key, int owner) {
    const int g = owner >> p.warp.shift, in = (owner & ((1 << p.warp.shift) - 1)) * p.warp.per_lane;
    return key <= kOffKeys ? -1 : g * p.group_size + in + kSlotMask - (key & kSlotMask);
  };
  int chosen = expert_of(my_key, my_lane);
  {
    // each expert taken against the next in the order: lane top_k - 1's next is the first one left out
    int out_lane;
    const int32_t out = take_best(head(), out_lane);
    int32_t next_key = __shfl_down_sync(kAll, my_key, 1);
    int next_e = __shfl_down_sync(kAll, chosen, 1);
    if (lane == p.top_k - 1) {
      next_key = out;
      next_e = expert_of(out, out_lane);
    }
    const float v = value_of(my_key & ~kSlotMask), u = value_of(next_key & ~kSlotMask);
    constexpr float kCut = VPL * 0x1p-23f + 0x1p-22f;      // the slot bits cut off, half a step of the sum with the bias
    const float off = p.bias != nullptr ? tol : 0.f;
    bool close = lane < p.top_k && my_key > kOffKeys && next_key > kOffKeys && !(v - u > 2.f * off + kCut * (fabsf(v) + fabsf(u)));
    if (__any_sync(kAll, close)) {
      if (close) {
        close = clean(to_float(row[chosen])) != clean(to_float(row[next_e])) ||
                (p.bias != nullptr && clean(p.bias[chosen]) != clean(p.bias[next_e]));
      }
      unsure = unsure || __any_sync(kAll, close);
    }
  }
  if (unsure) chosen = route_exact<T>(p, row, lane);
  return lane < p.top_k ? chosen : -1;
}

template <typename T, int VPL>
__global__ void __launch_bounds__(128) route_topk_kernel(const RouteParams p) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  const long long used = p.rows_used != nullptr ? *p.rows_used : p.tokens;
  for (long long token = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); token < p.tokens; token += warps) {
    long long* ids = p.ids + token * p.top_k;
    float* weights = p.weights + token * p.top_k;
    if (token >= used) {      // a padding token is routed nowhere
      if (lane < p.top_k) {
        ids[lane] = -1;
        weights[lane] = 0.f;
      }
      continue;
    }
    const T* row = static_cast<const T*>(p.logits) + token * p.ld;
    float row_max, sum;
    const int chosen = route_row<T, VPL>(p, row, lane, row_max, sum);
    // Weights, lane i for the expert chosen i-th. Sums over at most 32 chosen experts, in fp32.
    const float l = chosen >= 0 ? clean(to_float(row[chosen])) : -INFINITY;
    float w = 0.f;
    if (p.renormalize) {
      // scores up to a common factor: shifting by the largest chosen logit (sigmoid: only where all are negative) keeps
      // rows of very small scores away from 0 / 0
      float top = warp_max_f(l);
      if (p.sigmoid) {
        top = fminf(top, 0.f);
        const float t = __expf(-fabsf(l));
        w = __fdividef(l >= 0.f ? 1.f : __expf(l - top), 1.f + t);
      } else {
        w = __expf(l - top);
      }
      if (chosen < 0) w = 0.f;
      const float total = warp_sum_f(w);
      w = chosen >= 0 ? __fdividef(w, total) : 0.f;
    } else if (chosen >= 0) {
      w = __fdividef(p.sigmoid ? 1.f : __expf(l - row_max), p.sigmoid ? 1.f + __expf(-l) : sum);
    }
    if (lane < p.top_k) {
      ids[lane] = chosen;
      weights[lane] = w * p.scale;
    }
  }
}

// top_k up to 8: a row on `row_lanes` lanes, 32 / row_lanes rows per warp, so that what is done once per row -- ranking the groups,
// joining the lanes' lists, the weights -- is done for several rows at once. Keys carry the expert's index in their lowest bits.
// A lane sorts its experts in lists of 8 and merges them into its 8 best; the lanes' lists are merged by xor-shuffles (the
// larger of a[i] and b[7 - i] are the 8 best of both, in bitonic order), after which every lane of the row has the answer
// without a serial step per expert. The best key that a merge leaves out is kept: it says whether the eighth is clear of the rest.
// Experts too close for their keys (the index takes 8 of 24 bits with 256 experts, so one token in twenty) are put in order by
// their fp32 values, one per lane, and where those are too close by 64-bit ones; only where several more than eight are close at
// the border, or two groups are, does route_exact decide the row.
__device__ __forceinline__ void bitonic8(int32_t (&a)[8]) {
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((i & d) == 0) order(a[i], a[i + d]);
  }
}
// a = the 8 largest of a and b (both sorted), sorted; `left` = the largest of those left out and what it was.
__device__ __forceinline__ void merge8(int32_t (&a)[8], const int32_t (&b)[8], int32_t& left) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    left = max(left, min(a[i], b[7 - i]));
    a[i] = max(a[i], b[7 - i]);
  }
  bitonic8(a);
}

// Experts 8 q .. of a lane whose `count` experts start at `mine`, -inf past the last one. RAW: without clean(), where the caller
// looks at all eight itself.
template <typename T, bool RAW = false>
__device__ __forceinline__ void load8(bool vector, const T* mine, int count, int q, float (&l)[8]) {
  const T* src = mine + 8 * q;
  if (vector && count > 0) {
    constexpr int kWords = static_cast<int>(sizeof(T)) / 2;      // 16-byte words
    uint4 u[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) u[i] = reinterpret_cast<const uint4*>(src)[i];
#pragma unroll
    for (int j = 0; j < 8; ++j) l[j] = RAW ? to_float(reinterpret_cast<const T*>(u)[j]) : clean(to_float(reinterpret_cast<const T*>(u)[j]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) l[j] = 8 * q + j >= count ? -INFINITY : RAW ? to_float(src[j]) : clean(to_float(src[j]));
  }
}

// Rolled over a lane's pieces of 8 experts: straight-line code for 32 of them did not fit the instruction cache (65536 x 256: 108 us
// against 60). STAGED: the warp's rows come through shared memory by 16-byte asynchronous copies, each lane's experts 16 bytes
// further apart there; read straight from memory, lanes 64 bytes or more apart take a cache line each for 16 bytes.
template <typename T, bool STAGED>
__global__ void __launch_bounds__(128, 8) route_top8_kernel(const RouteParams p) {
  const int lane = threadIdx.x & 31, width = p.row_lanes, in_row = lane & (width - 1), row0 = lane & ~(width - 1);
  const int rows_per_warp = 32 / width;
  const long long token0 = (static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5)) * rows_per_warp;
  if (token0 >= p.tokens) return;
  const long long token = token0 + lane / width;
  const bool exists = token < p.tokens, live = exists && (p.rows_used == nullptr || token < *p.rows_used);
  const T* row = static_cast<const T*>(p.logits) + token * p.ld;
  Slots at(p, p.part, in_row);
  if (!live) at.count = 0;
  extern __shared__ uint4 route_smem[];
  const int lane_bytes = p.part.per_lane * static_cast<int>(sizeof(T));      // STAGED: a multiple of 64
  char* stage = reinterpret_cast<char*>(route_smem) + (threadIdx.x >> 5) * 32 * (lane_bytes + 16);
  const T* mine = row + at.first;
  if constexpr (STAGED) {
    const int row_bytes = p.experts * static_cast<int>(sizeof(T));
    const long long limit = p.rows_used == nullptr ? p.tokens : min(p.tokens, static_cast<long long>(*p.rows_used));
    for (int r = 0; r < rows_per_warp && token0 + r < limit; ++r) {
      const char* src = reinterpret_cast<const char*>(static_cast<const T*>(p.logits) + (token0 + r) * p.ld);
      const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(stage + r * width * (lane_bytes + 16)));
      for (int byte = lane * 16; byte < row_bytes; byte += 512)      // 16 bytes of padding per lane before this one
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + byte + (byte / static_cast<int>(sizeof(T)) >> p.part.lane_shift) * 16), "l"(src + byte) : "memory");
    }
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    mine = reinterpret_cast<const T*>(stage + lane * (lane_bytes + 16));
  }
  // logit of an expert of this lane's row
  auto logit = [&](int e) {
    if constexpr (STAGED) {
      const int owner = e >> p.part.lane_shift;
      return clean(to_float(reinterpret_cast<const T*>(stage + (row0 + owner) * (lane_bytes + 16))[e - (owner << p.part.lane_shift)]));
    } else {
      return clean(to_float(row[e]));
    }
  };
  auto row_max_of = [&](float v) {
    for (int o = width >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
  };
  auto row_sum_of = [&](float v) {
    for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
  };
  const bool scored = p.bias != nullptr || p.groups > 1, softmax_all = !p.sigmoid && (scored || !p.renormalize);
  const int pieces = (p.part.per_lane + 7) >> 3;
  float row_max = 0.f, sum = 0.f, inv = 0.f;
  if (softmax_all) {      // two more walks over the row, out of L1 after the first
    float mx = -INFINITY, l[8];
    for (int q = 0; q < pieces; ++q) {
      load8(p.part.vector_rows, mine, at.count, q, l);
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, l[j]);
    }
    row_max = row_max_of(mx);
    for (int q = 0; q < pieces; ++q) {
      load8(p.part.vector_rows, mine, at.count, q, l);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += l[j] > -INFINITY ? __expf(l[j] - row_max) : 0.f;
    }
    sum = row_sum_of(sum);
    inv = 1.f / sum;
  }
  const float tol = !scored ? 0.f : p.sigmoid ? 0x1p-20f : 0x1p-18f * inv;      // as in route_topk_kernel

  // the 8 best keys of this lane, the best one left out, and the two largest scores
  const int32_t index_mask = (1 << p.index_bits) - 1;
  int32_t top[8], left = INT32_MIN;
  float a1 = -INFINITY, a2 = -INFINITY;
  // One piece: c raw logits in, cleaned ones out, s the scores with their bias (where scores are needed).
  auto score = [&](int q, float (&c)[8], float (&s)[8]) {
    // NaN, infinities and missing experts are rare: one look at the sum spares the common piece two operations per expert
    float size = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) size += fabsf(c[j]);
    float b[8];
    if (p.bias != nullptr) {
      load8<float, true>(p.part.vector_bias, p.bias + at.first, at.count, q, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) size += fabsf(b[j]);
    }
    const bool special = !(size < INFINITY);
    if (special) {
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = clean(c[j]);
    }
    if (!scored) return;
    if (p.sigmoid) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = reciprocal(1.f + __expf(-c[j]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = __expf(c[j] - row_max) * inv;
    }
    if (special) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[j] = c[j] == -INFINITY ? -INFINITY : s[j];
        if (p.bias != nullptr) b[j] = clean(b[j]);
      }
    }
    if (p.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += b[j];      // a bias of -inf switches the expert off by itself
    }
  };
  float c[8];
  load8<T, true>(p.part.vector_rows, mine, at.count, 0, c);
#pragma unroll 1
  for (int q = 0; q < pieces; ++q) {
    float s[8], next[8];
    if (q + 1 < pieces) load8<T, true>(p.part.vector_rows, mine, at.count, q + 1, next);
    score(q, c, s);
    if (scored) {
      if (p.groups > 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a2 = fmaxf(a2, fminf(a1, s[j]));
          a1 = fmaxf(a1, s[j]);
        }
      }
      if (p.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = s[j];
      }
    }
    int32_t list[8];
    if (p.part.vector_rows) {      // the first expert is a multiple of 8: its index is or'ed in with the slot's
      const int32_t index = (index_mask - 7) - (at.first + 8 * q);
#pragma unroll
      for (int j = 0; j < 8; ++j) list[j] = ((key_of(c[j]) & ~index_mask) | index) | (7 - j);
    } else {
      const int32_t index0 = index_mask - (at.first + 8 * q);
#pragma unroll
      for (int j = 0; j < 8; ++j) list[j] = (key_of(c[j]) & ~index_mask) | ((index0 - j) & index_mask);
    }
    sort_list<8>(list);
    if (q == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) top[j] = list[j];
    } else {
      merge8(top, list, left);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = next[j];
  }

  bool unsure = false, kept = true;
  if (p.groups > 1) {
    for (int o = 1; o < (1 << p.part.shift); o <<= 1) {
      const float b1 = __shfl_xor_sync(kAll, a1, o), b2 = __shfl_xor_sync(kAll, a2, o);
      a2 = fmaxf(fmaxf(a2, b2), fminf(a1, b1));
      a1 = fmaxf(a1, b1);
    }
    const float mine = p.group_max || a2 == -INFINITY ? a1 : a1 + a2;
    const int g = in_row >> p.part.shift;
    int rank = 0;
    for (int o = 0; o < p.groups; ++o) {
      const float other = __shfl_sync(kAll, mine, row0 + (o << p.part.shift));
      rank += other > mine || (other == mine && o < g);
    }
    const bool real = g < p.groups;
    kept = rank < p.top_groups;
    // the weakest group kept against the strongest one left out
    const float low = -row_max_of(real && kept ? -mine : -INFINITY), high = row_max_of(real && !kept ? mine : -INFINITY);
    if (high > -INFINITY) unsure = !(low - high > 4.f * tol + 0x1p-20f * (fabsf(low) + fabsf(high)));
    if (!kept) {
      left = INT32_MIN;
#pragma unroll
      for (int j = 0; j < 8; ++j) top[j] = INT32_MIN;
    }
  }
  // the 8 best keys of the row, on every lane of it
  for (int o = 1; o < width; o <<= 1) {
    int32_t other[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) other[j] = __shfl_xor_sync(kAll, top[j], o);
    left = max(left, __shfl_xor_sync(kAll, left, o));
    merge8(top, other, left);
  }
  // lane i of the row has the i-th best
  int32_t key = kOffKeys;
#pragma unroll
  for (int j = 0; j < 8; ++j) key = in_row == j ? top[j] : key;
  auto expert_of = [&](int32_t k) { return k <= kOffKeys ? -1 : index_mask - (k & index_mask); };
  int chosen = expert_of(key);

  if (p.bias != nullptr || sizeof(T) == 4) {      // keys of 16-bit logits are exact: 13 bits above the index at least
    int32_t next = __shfl_down_sync(kAll, key, 1);
    if (in_row == 7) next = left;
    const float v = value_of(key & ~index_mask), u = value_of(next & ~index_mask), off = p.bias != nullptr ? tol : 0.f;
    const float cut = __int2float_rn(index_mask + 1) * 0x1p-23f + 0x1p-22f;
    const bool close = in_row < 8 && key > kOffKeys && next > kOffKeys && !(v - u > 2.f * off + cut * (fabsf(v) + fabsf(u)));
    const unsigned all_close = __ballot_sync(kAll, close);
    if (all_close != 0u) {
      const unsigned here = (all_close >> row0) & 0xffu;
      // what was left out may belong among the first top_k only if nothing separates it from them; then the best one left out
      // takes part below, and if the row has more that close, route_exact decides it
      const unsigned chain = 0xffu & ~((1u << (p.top_k - 1)) - 1u);
      bool border = (here & chain) == chain;
      if (__any_sync(kAll, border)) {
        const float last = value_of(__shfl_sync(kAll, key, row0 + 7) & ~index_mask), least = last - 2.f * off - cut * 2.f * fabsf(last);
        int near = 0;
#pragma unroll 1
        for (int q = 0; q < pieces; ++q) {
          float s[8];
          load8<T, true>(p.part.vector_rows, mine, at.count, q, c);
          score(q, c, s);
#pragma unroll
          for (int j = 0; j < 8; ++j) near += kept && (p.bias != nullptr ? s[j] : c[j]) >= least;
        }
        for (int o = width >> 1; o > 0; o >>= 1) near += __shfl_xor_sync(kAll, near, o);
        if (border && near > 9) {
          unsure = true;
          border = false;
        }
      }
      const int ninth = border ? expert_of(left) : -1;
      // in order by the whole fp32 value, then, where even that is within its error of the next, by the exact one
      const float l = chosen >= 0 ? logit(chosen) : -INFINITY, b = p.bias != nullptr && chosen >= 0 ? clean(p.bias[chosen]) : 0.f;
      const float l9 = ninth >= 0 ? logit(ninth) : -INFINITY, b9 = p.bias != nullptr && ninth >= 0 ? clean(p.bias[ninth]) : 0.f;
      auto value32 = [&](float l, float b) {
        return p.bias == nullptr || l == -INFINITY ? l : (p.sigmoid ? reciprocal(1.f + __expf(-l)) : __expf(l - row_max) * inv) + b;
      };
      const float f = value32(l, b), f9 = value32(l9, b9);
      // the eight, and the ninth where there is one, by value and then by index; lane i gets the i-th
      auto sort_by = [&](auto value, auto value9) {
        int rank = ninth >= 0 && (value9 > value || (value9 == value && ninth < chosen)), rank9 = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const auto v = __shfl_sync(kAll, value, row0 + j);
          const int e = __shfl_sync(kAll, chosen, row0 + j);
          rank += v > value || (v == value && e < chosen);
          rank9 += v > value9 || (v == value9 && e < ninth);
        }
        int sorted = ninth >= 0 && rank9 == in_row ? ninth : -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = __shfl_sync(kAll, rank, row0 + j), e = __shfl_sync(kAll, chosen, row0 + j);
          if (e >= 0 && r == in_row) sorted = e;
        }
        return sorted;
      };
      // two with the same logit and bias are in the right order already, by index, and need no more
      bool alike = false;
      auto compare = [&](float fj, float lj, float bj) {
        alike = alike || (in_row < 8 && chosen >= 0 && lj > -INFINITY && (lj != l || bj != b) && !(fabsf(fj - f) > 2.f * off + 0x1p-22f * (fabsf(fj) + fabsf(f))));
      };
#pragma unroll
      for (int j = 0; j < 8; ++j) compare(__shfl_sync(kAll, f, row0 + j), __shfl_sync(kAll, l, row0 + j), __shfl_sync(kAll, b, row0 + j));
      compare(f9, l9, b9);
      alike = alike && p.bias != nullptr;      // logits alone are exact
      int sorted = sort_by(f, f9);
      const unsigned all_alike = __ballot_sync(kAll, alike);
      if (all_alike != 0u) {
        if (p.sigmoid) {
          auto value64 = [&](float l, float b) { return l > -INFINITY ? 1 / (1 + exp(-static_cast<double>(l))) + static_cast<double>(b) : -INFINITY; };
          sorted = sort_by(value64(l, b), value64(l9, b9));
        } else if (((all_alike >> row0) & 0xffu) != 0u) {
          unsure = true;      // a softmax score needs its sum in 64 bits too
        }
      }
      if (here != 0u) chosen = sorted;
    }
  }
  unsigned exact = __ballot_sync(kAll, unsure && live && in_row == 0);
  while (exact != 0u) {
    const int first = __ffs(exact) - 1;
    exact &= exact - 1;
    const int e = route_exact<T>(p, static_cast<const T*>(p.logits) + (token0 + first / width) * p.ld, lane);
    const int theirs = __shfl_sync(kAll, e, in_row);
    if (row0 == first) chosen = theirs;
  }
  if (in_row >= p.top_k) chosen = -1;

  const float l = chosen >= 0 ? logit(chosen) : -INFINITY;
  float w = 0.f;
  if (p.renormalize) {      // as in route_topk_kernel
    float best = row_max_of(l);
    if (p.sigmoid) {
      best = fminf(best, 0.f);
      const float t = __expf(-fabsf(l));
      w = __fdividef(l >= 0.f ? 1.f : __expf(l - best), 1.f + t);
    } else {
      w = __expf(l - best);
    }
    if (chosen < 0) w = 0.f;
    const float total = row_sum_of(w);
    w = chosen >= 0 ? __fdividef(w, total) : 0.f;
  } else if (chosen >= 0) {
    w = __fdividef(p.sigmoid ? 1.f : __expf(l - row_max), p.sigmoid ? 1.f + __expf(-l) : sum);
  }
  if (exists && in_row < p.top_k) {
    p.ids[token * p.top_k + in_row] = chosen;
    p.weights[token * p.top_k + in_row] = w * p.scale;
  }
}

// ------------------------------------------------------------------------------------------------ backward
// dlogits of one token per warp. Weights w_i = scale * s_i (/ S, S = sum of the chosen scores), gradients g_i:
//   renormalised:  dl_i = scale * q_i * d_i * (g_i - sum_j q_j g_j),  q = s / S,  d = 1 (softmax) or 1 - s_i (sigmoid);
//   sigmoid:       dl_i = scale * g_i * s_i * (1 - s_i);
//   softmax:       dl_j = scale * s_j * ([j chosen] g_j - sum_i s_i g_i), for every expert j.
// Experts that do not appear get 0, so only the last form reads the whole row; all write it in 16-byte pieces and the few chosen
// entries over it (65536 x 256 fp32, top 8: 42 us with the entries merged into the pieces before the store, 21 to 26 so: 67 MB written,
// and of the logits a cache line per chosen expert read; the softmax that is not renormalised 42, reading the row three times).
struct RouteGradParams {
  const void* logits;
  const float* dweights;
  const long long* ids;
  void* dlogits;
  long long tokens, ld;
  int experts, top_k, sigmoid, renormalize;
  float scale;
};

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(128) route_topk_backward_kernel(const RouteGradParams p) {
  const long long token = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (token >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + token * p.ld;
  T* out = static_cast<T*>(p.dlogits) + token * p.experts;
  const bool dense = !p.sigmoid && !p.renormalize;
  int id = -1;
  float g = 0.f;
  if (lane < p.top_k) {
    const long long e = p.ids[token * p.top_k + lane];
    if (e >= 0 && e < p.experts) {
      id = static_cast<int>(e);
      g = p.dweights[token * p.top_k + lane] * p.scale;
    }
  }
  const float l = id >= 0 ? clean(to_float(row[id])) : -INFINITY;
  if (l == -INFINITY) {      // switched off: its weight is 0 whatever the gradient asks for
    id = -1;
    g = 0.f;
  }
  float v = 0.f, row_max = 0.f, inv = 0.f, dot = 0.f;
  if (p.renormalize) {
    float top = warp_max_f(l), s = 0.f, rest = 1.f;
    if (p.sigmoid) {
      top = fminf(top, 0.f);
      const float t = expf(-fabsf(l));
      rest = (l >= 0.f ? t : 1.f) / (1.f + t);                       // 1 - sigmoid(l), without cancellation
      s = l >= 0.f ? 1.f / (1.f + t) : expf(l - top) / (1.f + t);
    } else {
      s = expf(l - top);
    }
    if (id < 0) s = 0.f;
    const float total = warp_sum_f(s);
    const float q = id >= 0 ? s / total : 0.f;
    v = q * rest * (g - warp_sum_f(q * g));
  } else if (p.sigmoid) {
    const float t = expf(-fabsf(l));
    v = id >= 0 ? g * t / ((1.f + t) * (1.f + t)) : 0.f;             // s (1 - s)
  } else {
    float mx = -INFINITY;
    for (int e = lane; e < p.experts; e += 32) mx = fmaxf(mx, clean(to_float(row[e])));
    row_max = warp_max_f(mx);
    float sum = 0.f;
    for (int e = lane; e < p.experts; e += 32) {
      const float x = clean(to_float(row[e]));
      sum += x > -INFINITY ? expf(x - row_max) : 0.f;
    }
    sum = warp_sum_f(sum);
    inv = sum > 0.f ? 1.f / sum : 0.f;
    const float s = id >= 0 ? expf(l - row_max) * inv : 0.f;
    dot = warp_sum_f(s * g);
    v = s * g;
  }
  // an expert named twice in a row gets both parts, from the first lane that names it
  const unsigned same = __match_any_sync(kAll, id);
  if (__any_sync(kAll, id >= 0 && __popc(same) > 1)) {
    float all = 0.f;
    for (int t = 0; t < p.top_k; ++t) {
      const float other = __shfl_sync(kAll, v, t);
      if (same >> t & 1u) all += other;
    }
    if (id >= 0) v = all;
  }
  // the row as it is without the chosen experts, then the chosen ones over it
  constexpr int V = VECTOR ? 16 / static_cast<int>(sizeof(T)) : 1;      // elements a lane writes at once
  auto rest = [&](int e) {
    const float x = clean(to_float(row[e]));
    return x > -INFINITY ? -expf(x - row_max) * inv * dot : 0.f;
  };
  for (int e0 = lane * V; e0 < p.experts; e0 += 32 * V) {
    if constexpr (VECTOR) {
      uint4 o = make_uint4(0, 0, 0, 0);
      if (dense) {
        T* t = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = from_float<T>(rest(e0 + i));
      }
      *reinterpret_cast<uint4*>(out + e0) = o;
    } else {
      out[e0] = from_float<T>(dense ? rest(e0) : 0.f);
    }
  }
  __syncwarp();
  if (id >= 0 && lane == __ffs(same) - 1) out[id] = from_float<T>(dense ? v + rest(id) : v);
}

// ------------------------------------------------------------------------------------------------ layout tables
// A stable counting sort of the (token, slot) pairs by expert, on integers only: the same input gives the same tables.
// Every block owns a run of consecutive pairs, every warp of it a run of those. How many pairs of an expert lie before
// a warp's run follows from the blocks' counts (first kernel, or the one block's own) and the warps' counts (shared
// memory); inside a warp 32 pairs are ranked at a time with match.any. 524288 pairs, 256 experts: 16 us for both kernels (moving
// their 13 MB would take 2); 512 pairs: 6.6 us in the one. What takes the time is the chain of short passes with barriers between
// them, not any resource: issue slots are 29 % used. Runs of up to 4096 pairs per block stay in registers, experts and ranks, between the passes.
struct LayoutParams {
  const void* ids;
  int ids_64;
  long long pairs;
  int top_k, experts, alignment, max_rows;    // max_rows > 0: the masked layout
  long long rows;                             // rows of the layout = entries of row_token
  int* block_counts;                          // [blocks, experts rounded up to 4]
  long long* pair_row;
  long long* row_token;
  long long* rows_per_expert;                 // contiguous
  int* offsets;                               // contiguous [2 * experts]
  int* expert_list;                           // contiguous [experts + 1]
  int* masked_m;                              // masked [experts]
  int* status;
  long long run;                              // pairs per block, a multiple of the block's threads
};

constexpr int kLayoutThreads = 1024;
constexpr int kLayoutWarps = kLayoutThreads / 32;

__host__ __device__ constexpr int padded_experts(int experts) { return (experts + 3) & ~3; }

__device__ __forceinline__ int pair_expert(const LayoutParams& p, long long i, bool report) {
  const long long e = p.ids_64 ? __ldg(static_cast<const long long*>(p.ids) + i) : __ldg(static_cast<const int*>(p.ids) + i);
  if (e >= 0 && e < p.experts) return static_cast<int>(e);
  if (report && e != -1 && p.status != nullptr) atomicCAS(p.status, 0, AG_EP_BAD_EXPERT | (static_cast<int>(blockIdx.x) << 8));
  return -1;
}

__global__ void __launch_bounds__(kLayoutThreads) layout_count_kernel(const LayoutParams p) {
  extern __shared__ int count[];
  for (int e = threadIdx.x; e < p.experts; e += kLayoutThreads) count[e] = 0;
  __syncthreads();
  const long long begin = blockIdx.x * p.run, end = min(begin + p.run, p.pairs);
  for (long long i = begin + threadIdx.x; i < end; i += kLayoutThreads) {
    const int e = pair_expert(p, i, false);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += kLayoutThreads) p.block_counts[static_cast<long long>(blockIdx.x) * padded_experts(p.experts) + e] = count[e];
}

// ONE: the pairs are one block's, which needs no counts of others. The launch's further blocks, if any, count the same pairs and only
// take part in marking the rows that none has.
template <bool ONE>
__global__ void __launch_bounds__(kLayoutThreads) layout_place_kernel(const LayoutParams p) {
  extern __shared__ int smem[];
  int* total = smem;                    // [experts] pairs of the expert
  int* start = total + p.experts;       // [experts + 1] first row of its segment
  int* seen = start + p.experts + 1;    // [experts] its pairs in the blocks before this one
  int* mine = seen + p.experts;         // [warps, experts] its pairs in each warp's run, then those before the run
  __shared__ int warp_sums[kLayoutWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = p.experts;
  for (int e = threadIdx.x; e < E; e += kLayoutThreads) total[e] = seen[e] = 0;
  for (int i = threadIdx.x; i < kLayoutWarps * E; i += kLayoutThreads) mine[i] = 0;
  __syncthreads();

  const long long begin = ONE ? 0 : blockIdx.x * p.run, end = min(begin + p.run, p.pairs);
  const long long share = p.run / kLayoutWarps;            // a multiple of 32
  const long long from = begin + warp * share, to = min(from + share, end);
  // the warp's pairs, kept in registers 4 x 32 at a time so that their loads are under way together (a run of 4096 pairs per
  // block is the most that stays; a longer one is read again below)
  constexpr int kAhead = 4;
  int mine_e[kAhead];
  unsigned same_e[kAhead];      // lanes with the same expert
  auto load_pairs = [&](long long i0, bool report) {
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const long long i = i0 + 32 * q + lane;
      mine_e[q] = i < to ? pair_expert(p, i, report) : -1;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) same_e[q] = __match_any_sync(kAll, mine_e[q]);
  };
  for (long long i0 = from; i0 < to; i0 += 32 * kAhead) {
    load_pairs(i0, !ONE || blockIdx.x == 0);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int e = mine_e[q];
      const unsigned same = same_e[q];
      if (e >= 0 && lane == __ffs(same) - 1) mine[warp * E + e] += __popc(same);
      __syncwarp();
    }
  }
  if (!ONE) {
    // all blocks' counts, four experts at a time, `parts` threads for each four; integer sums, so their order does not matter
    const int fours = padded_experts(E) / 4, parts = kLayoutThreads / fours;
    const int part = static_cast<int>(threadIdx.x) / fours, e0 = static_cast<int>(threadIdx.x) % fours * 4;
    if (part < parts) {
      int all[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0};
#pragma unroll 8
      for (int b = part; b < static_cast<int>(gridDim.x); b += parts) {
        const int4 v = __ldg(reinterpret_cast<const int4*>(p.block_counts) + static_cast<long long>(b) * fours + e0 / 4);
        const int c[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          all[j] += c[j];
          before[j] += b < static_cast<int>(blockIdx.x) ? c[j] : 0;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (e0 + j >= E) break;      // what the padding holds is not used
        atomicAdd(&total[e0 + j], all[j]);
        atomicAdd(&seen[e0 + j], before[j]);
      }
    }
  }
  __syncthreads();
  // pairs of the expert before each warp's run, in this block
  for (int e = threadIdx.x; e < E; e += kLayoutThreads) {
    int before = seen[e];
    for (int w0 = 0; w0 < kLayoutWarps; w0 += 8) {
      int v[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) v[w] = mine[(w0 + w) * E + e];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        mine[(w0 + w) * E + e] = before;
        before += v[w];
      }
    }
    if (ONE) total[e] = before;
  }
  __syncthreads();
  // first row of every segment: a running sum over the experts, one per thread
  {
    const int e = threadIdx.x;
    int size = 0;
    if (e < E) size = p.max_rows > 0 ? p.max_rows : (total[e] + p.alignment - 1) / p.alignment * p.alignment;
    int sum = size;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kAll, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) warp_sums[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      int v = warp_sums[lane], s = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kAll, s, o);
        if (lane >= o) s += u;
      }
      warp_sums[lane] = s - v;
    }
    __syncthreads();
    sum += warp_sums[warp];
    if (e < E) {
      start[e] = sum - size;
      if (e == E - 1) start[E] = sum;
      if (blockIdx.x == 0) {
        if (p.max_rows > 0) {
          p.masked_m[e] = min(total[e], p.max_rows);
        } else {
          p.rows_per_expert[e] = total[e];
          p.offsets[2 * e] = sum - size;
          p.offsets[2 * e + 1] = sum;
          p.expert_list[e] = e;
          if (e == E - 1) p.expert_list[E] = -1;
        }
      }
    }
    __syncthreads();
  }
  for (long long i0 = from; i0 < to && (!ONE || blockIdx.x == 0); i0 += 32 * kAhead) {
    if (to - from > 32 * kAhead) load_pairs(i0, false);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const long long i = i0 + 32 * q + lane;
      const int e = mine_e[q];
      const unsigned same = same_e[q];
      int base = 0;
      if (e >= 0) base = mine[warp * E + e];
      __syncwarp();
      if (e >= 0 && lane == __ffs(same) - 1) mine[warp * E + e] = base + __popc(same);
      __syncwarp();
      if (i < to) {
        const int within = base + __popc(same & ((1u << lane) - 1u));
        const bool placed = e >= 0 && (p.max_rows == 0 || within < p.max_rows);
        const long long row = placed ? static_cast<long long>(start[e]) + within : -1;
        p.pair_row[i] = row;
        if (placed) p.row_token[row] = static_cast<unsigned>(i) / static_cast<unsigned>(p.top_k);      // pairs < 2^30
      }
    }
  }
  // rows that no pair has: the end of every expert's segment, a warp of the launch each, and what lies behind the last
  for (int e = blockIdx.x * kLayoutWarps + warp; e < E; e += gridDim.x * kLayoutWarps) {
    const int end_row = start[e + 1];
    for (int r = start[e] + min(total[e], end_row - start[e]) + lane; r < end_row; r += 32) p.row_token[r] = -1;
  }
  for (long long r = start[E] + static_cast<long long>(blockIdx.x) * kLayoutThreads + threadIdx.x; r < p.rows; r += static_cast<long long>(gridDim.x) * kLayoutThreads)
    p.row_token[r] = -1;
}

}  // namespace agb

namespace {

int launch_check() {
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? AG_OK : agb_fail(AG_E_CUDA, cudaGetErrorString(e));
}
bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
int size_of(int dtype) { return dtype == AG_T_FP32 ? 4 : 2; }

template <typename T, int VPL>
void launch_route_as(const agb::RouteParams& p, int sms, cudaStream_t stream) {
  constexpr int kWarps = 4, kBlocksPerSm = VPL <= 8 ? 8 : VPL == 16 ? 6 : 4;
  const long long blocks = (p.tokens + kWarps - 1) / kWarps, most = static_cast<long long>(sms) * kBlocksPerSm;
  agb::route_topk_kernel<T, VPL><<<static_cast<unsigned>(blocks < most ? blocks : most), 32 * kWarps, 0, stream>>>(p);
}
template <typename T>
void launch_top8(const agb::RouteParams& p, cudaStream_t stream) {
  const long long rows = 4 * (32 / p.row_lanes);
  const unsigned grid = static_cast<unsigned>((p.tokens + rows - 1) / rows);
  const int lane_bytes = p.part.per_lane * static_cast<int>(sizeof(T));
  if (p.part.vector_rows && lane_bytes >= 64)
    agb::route_top8_kernel<T, true><<<grid, 128, 128 * (lane_bytes + 16), stream>>>(p);
  else
    agb::route_top8_kernel<T, false><<<grid, 128, 0, stream>>>(p);
}
// Measured at 65536 x 256 fp32: top 8, softmax 37 us; top 8 of 4 of 8 groups, sigmoid and bias 53 us (550 instructions per row, issue
// slots 73 % used; reading the logits would take 10 us). Top 16 takes 89 to 93 us on a warp per
// row without groups, 128 with sigmoid, bias and 4 of 8 groups; the 53 us case took 104 there.
template <typename T>
void launch_route(const agb::RouteParams& p, int sms, cudaStream_t stream) {
  if (p.top_k <= 8) {
    launch_top8<T>(p, stream);
  } else if (p.warp.per_lane <= 8) {
    launch_route_as<T, 8>(p, sms, stream);
  } else if (p.warp.per_lane <= 16) {
    launch_route_as<T, 16>(p, sms, stream);
  } else {
    launch_route_as<T, 32>(p, sms, stream);
  }
}

// The map of a row onto `lanes` lanes; per_lane is above 32 where they are too few.
agb::LaneMap lane_map(const ag_route_desc_t* r, int lanes) {
  agb::LaneMap m{};
  int across = lanes;
  while (across * r->groups > lanes) across >>= 1;
  if (across == 0) {
    m.per_lane = agb::kRouteMaxPerLane + 1;
    return m;
  }
  while ((1 << m.shift) < across) ++m.shift;
  const int size = r->experts / r->groups;
  m.per_lane = (size + across - 1) / across;
  // vector loads want lanes full of slots, 8, 16 or 32 of them
  const bool full = (m.per_lane & (m.per_lane - 1)) == 0 && m.per_lane >= 8 && size == m.per_lane * across;
  while (full && (1 << m.lane_shift) < m.per_lane) ++m.lane_shift;
  m.vector_rows = full && aligned_to(r->logits, 16) && r->ld * size_of(r->dtype) % 16 == 0;
  m.vector_bias = full && aligned_to(r->bias, 16);
  return m;
}

template <typename T>
void launch_route_backward(const agb::RouteGradParams& p, bool vector, cudaStream_t stream) {
  const unsigned grid = static_cast<unsigned>((p.tokens + 3) / 4);
  if (vector) agb::route_topk_backward_kernel<T, true><<<grid, 128, 0, stream>>>(p);
  else agb::route_topk_backward_kernel<T, false><<<grid, 128, 0, stream>>>(p);
}

// Pairs per block. Up to 2048 one block saves the counting launch (256 experts: 2048 pairs 8.4 us in one, 10.7 in two; 4096 pairs 12.1
// and 9.8). Then runs of 1024, one pair per thread (32768 pairs: 9.6 us; in runs of 2048 11.5, of 4096 15.1), but no more than 128
// blocks, because every block sums the counts of all others (524288 pairs: 16 us on 128 blocks, 23 on 256).
constexpr int64_t kLayoutFill = 4096, kLayoutRun = 1024;
long long layout_run(long long pairs) {
  if (pairs <= 2048) return 2048;
  const long long run = (pairs + 127) / 128;
  const long long least = run > kLayoutRun ? run : kLayoutRun;
  return (least + agb::kLayoutThreads - 1) / agb::kLayoutThreads * agb::kLayoutThreads;
}

// Shared memory of the placing kernel. Its limit is raised once per device, for the most experts: the limit belongs to the function,
// so a call that set it to its own needs could lower it between another thread's setting and launch.
constexpr size_t layout_memory(int experts) { return (static_cast<size_t>(experts) * (3 + agb::kLayoutWarps) + 1) * 4; }
cudaError_t allow_layout_memory(void (*place)(agb::LayoutParams), std::atomic<bool> (&allowed)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && allowed[dev].load(std::memory_order_relaxed))) return e;
  e = cudaFuncSetAttribute(place, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(layout_memory(agb::kLayoutMaxExperts)));
  if (e == cudaSuccess && dev < 64) allowed[dev].store(true, std::memory_order_relaxed);
  return e;
}

}  // namespace

extern "C" {

int ag_route_topk(const ag_route_desc_t* r) {
  if (r == nullptr) return agb_fail(AG_E_INVALID, "desc is NULL");
  if (r->dtype < AG_T_BF16 || r->dtype > AG_T_FP32) return agb_fail(AG_E_INVALID, "logits must be bf16, fp16 or fp32");
  if (r->tokens < 0 || r->experts <= 0 || r->top_k <= 0 || r->ld < r->experts) return agb_fail(AG_E_INVALID, "bad sizes");
  if (r->scoring != AG_SCORE_SOFTMAX && r->scoring != AG_SCORE_SIGMOID) return agb_fail(AG_E_INVALID, "unknown scoring");
  if (r->groups <= 0 || r->groups > 32 || r->experts % r->groups != 0 || r->top_groups <= 0 || r->top_groups > r->groups)
    return agb_fail(AG_E_INVALID, "the groups (1 .. 32) must divide the experts, and top_groups must be 1 .. groups");
  const int size = r->experts / r->groups;
  if (r->top_k > agb::kRouteMaxTopK || r->top_k > r->top_groups * size)
    return agb_fail(AG_E_INVALID, "top_k must be at most 32 and at most the experts of top_groups groups");
  const agb::LaneMap warp = lane_map(r, 32);
  if (warp.per_lane > agb::kRouteMaxPerLane) return agb_fail(AG_E_INVALID, "too many experts (at most 32 per lane: 1024 in one group, 1024 / groups rounded to a power of two in each of several)");
  if (!aligned_to(r->logits, size_of(r->dtype)) || !aligned_to(r->bias, 4) || !aligned_to(r->rows_used, 4) || !aligned_to(r->ids, 8) ||
      !aligned_to(r->weights, 4))
    return agb_fail(AG_E_INVALID, "pointers must be aligned to their element type");
  if (r->tokens == 0) return AG_OK;
  if (r->logits == nullptr || r->ids == nullptr || r->weights == nullptr) return agb_fail(AG_E_INVALID, "logits, ids and weights must be non-NULL");
  if (r->tokens > 4LL * 0x7fffffff) return agb_fail(AG_E_INVALID, "too many tokens");
  agb::RouteParams p{};
  p.logits = r->logits;
  p.bias = r->bias;
  p.rows_used = r->rows_used;
  p.ids = reinterpret_cast<long long*>(r->ids);
  p.weights = r->weights;
  p.tokens = r->tokens;
  p.ld = r->ld;
  p.experts = r->experts;
  p.top_k = r->top_k;
  p.groups = r->groups;
  p.top_groups = r->top_groups;
  p.group_size = size;
  p.warp = warp;
  p.sigmoid = r->scoring == AG_SCORE_SIGMOID;
  p.group_max = r->group_max != 0;
  p.renormalize = r->renormalize != 0;
  p.scale = r->scale;
  int sms = 0;
  if (int rc = agb_device_sm_count(&sms)) return rc;
  // Few tokens: a row on a whole warp, for the shorter way through it. Many: as few lanes as hold it, for the fewer instructions.
  p.row_lanes = r->tokens <= 4 * sms ? 32 : 8;
  while ((p.part = lane_map(r, p.row_lanes)).per_lane > agb::kRouteMaxPerLane) p.row_lanes *= 2;
  while ((1 << p.index_bits) < r->experts) ++p.index_bits;
  cudaStream_t stream = static_cast<cudaStream_t>(r->stream);
  if (r->dtype == AG_T_BF16) launch_route<__nv_bfloat16>(p, sms, stream);
  else if (r->dtype == AG_T_FP16) launch_route<__half>(p, sms, stream);
  else launch_route<float>(p, sms, stream);
  return launch_check();
}

int ag_route_topk_backward(const void* logits, int32_t dtype, int64_t tokens, int64_t ld, int32_t experts, const float* dweights, const int64_t* ids,
                           int32_t top_k, int32_t scoring, int32_t renormalize, float scale, void* dlogits, void* stream) {
  if (dtype < AG_T_BF16 || dtype > AG_T_FP32) return agb_fail(AG_E_INVALID, "logits must be bf16, fp16 or fp32");
  if (tokens < 0 || experts <= 0 || top_k <= 0 || top_k > agb::kRouteMaxTopK || ld < experts || tokens > 4LL * 0x7fffffff)
    return agb_fail(AG_E_INVALID, "bad sizes (top_k must be 1 .. 32)");
  if (scoring != AG_SCORE_SOFTMAX && scoring != AG_SCORE_SIGMOID) return agb_fail(AG_E_INVALID, "unknown scoring");
  const int size = size_of(dtype);
  if (!aligned_to(logits, size) || !aligned_to(dlogits, size) || !aligned_to(dweights, 4) || !aligned_to(ids, 8))
    return agb_fail(AG_E_INVALID, "pointers must be aligned to their element type");
  if (tokens == 0) return AG_OK;
  if (!logits || !dweights || !ids || !dlogits) return agb_fail(AG_E_INVALID, "logits, dweights, ids and dlogits must be non-NULL");
  agb::RouteGradParams p{};
  p.logits = logits;
  p.dweights = dweights;
  p.ids = reinterpret_cast<const long long*>(ids);
  p.dlogits = dlogits;
  p.tokens = tokens;
  p.ld = ld;
  p.experts = experts;
  p.top_k = top_k;
  p.sigmoid = scoring == AG_SCORE_SIGMOID;
  p.renormalize = renormalize != 0;
  p.scale = scale;
  const bool vector = static_cast<int64_t>(experts) * size % 16 == 0 && aligned_to(dlogits, 16);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == AG_T_BF16) launch_route_backward<__nv_bfloat16>(p, vector, s);
  else if (dtype == AG_T_FP16) launch_route_backward<__half>(p, vector, s);
  else launch_route_backward<float>(p, vector, s);
  return launch_check();
}

uint64_t ag_route_layout_workspace_bytes(int64_t pairs, int32_t experts) {
  if (pairs <= 0 || experts <= 0) return 0;
  const int64_t blocks = (pairs + layout_run(pairs) - 1) / layout_run(pairs);
  return blocks > 1 ? static_cast<uint64_t>(blocks) * agb::padded_experts(experts) * 4 : 0;
}

int ag_route_layout(const ag_route_layout_desc_t* r) {
  if (r == nullptr) return agb_fail(AG_E_INVALID, "desc is NULL");
  if (r->tokens < 0 || r->tokens > 0x7fffffffLL || r->top_k <= 0 || r->experts <= 0 || r->experts > agb::kLayoutMaxExperts || r->max_rows < 0 || r->rows < 0)
    return agb_fail(AG_E_INVALID, "bad sizes (at most 1024 experts)");
  const int64_t pairs = r->tokens * r->top_k;
  if (pairs > 0x7fffffffLL / 2 || r->rows > 0x7fffffffLL) return agb_fail(AG_E_INVALID, "too many (token, slot) pairs");
  if (!aligned_to(r->ids, r->ids_64 ? 8 : 4) || !aligned_to(r->pair_row, 8) || !aligned_to(r->row_token, 8) || !aligned_to(r->rows_per_expert, 8) ||
      !aligned_to(r->offsets, 4) || !aligned_to(r->expert_list, 4) || !aligned_to(r->masked_m, 4) || !aligned_to(r->workspace, 16))
    return agb_fail(AG_E_INVALID, "pointers must be aligned to their element type, the workspace to 16 bytes");
  if ((pairs > 0 && (r->ids == nullptr || r->pair_row == nullptr)) || (r->rows > 0 && r->row_token == nullptr))
    return agb_fail(AG_E_INVALID, "ids, pair_row and row_token must be non-NULL");
  if (r->max_rows > 0) {
    if (r->masked_m == nullptr || r->rows != static_cast<int64_t>(r->experts) * r->max_rows)
      return agb_fail(AG_E_INVALID, "the masked layout wants masked_m and experts * max_rows rows");
  } else {
    if (r->alignment <= 0 || r->rows_per_expert == nullptr || r->offsets == nullptr || r->expert_list == nullptr)
      return agb_fail(AG_E_INVALID, "the contiguous layout wants a positive alignment, rows_per_expert, offsets and expert_list");
    // every expert's segment ends less than one alignment past its pairs
    if (r->rows < pairs + static_cast<int64_t>(r->experts) * (r->alignment - 1) && r->rows < pairs * r->alignment)
      return agb_fail(AG_E_INVALID, "rows must cover every expert's padded segment");
  }
  const int64_t run = layout_run(pairs);
  const int blocks = pairs > 0 ? static_cast<int>((pairs + run - 1) / run) : 1;
  if (blocks > 1 && (r->workspace == nullptr || r->workspace_bytes < ag_route_layout_workspace_bytes(pairs, r->experts)))
    return agb_fail(AG_E_INVALID, "workspace too small (ag_route_layout_workspace_bytes)");
  agb::LayoutParams p{};
  p.ids = r->ids;
  p.ids_64 = r->ids_64;
  p.pairs = pairs;
  p.top_k = r->top_k;
  p.experts = r->experts;
  p.alignment = r->alignment;
  p.max_rows = r->max_rows;
  p.rows = r->rows;
  p.block_counts = static_cast<int*>(r->workspace);
  p.pair_row = reinterpret_cast<long long*>(r->pair_row);
  p.row_token = reinterpret_cast<long long*>(r->row_token);
  p.rows_per_expert = reinterpret_cast<long long*>(r->rows_per_expert);
  p.offsets = r->offsets;
  p.expert_list = r->expert_list;
  p.masked_m = r->masked_m;
  p.status = r->status;
  p.run = run;
  cudaStream_t stream = static_cast<cudaStream_t>(r->stream);
  auto place = blocks == 1 ? agb::layout_place_kernel<true> : agb::layout_place_kernel<false>;
  static std::atomic<bool> allowed[2][64];
  const cudaError_t e = allow_layout_memory(place, allowed[blocks == 1]);
  if (e != cudaSuccess) return agb_fail(AG_E_CUDA, cudaGetErrorString(e));
  if (blocks > 1) agb::layout_count_kernel<<<blocks, agb::kLayoutThreads, static_cast<size_t>(r->experts) * 4, stream>>>(p);
  // few pairs: a block more for every kLayoutFill rows to be marked (64 pairs x 8, 256 experts, 33280 rows: 10.5 us on one block, 6.6 on 9)
  const int64_t fill = (r->rows + kLayoutFill - 1) / kLayoutFill;
  const int grid = blocks > 1 ? blocks : fill < 1 ? 1 : fill > 64 ? 64 : static_cast<int>(fill);
  place<<<grid, agb::kLayoutThreads, layout_memory(r->experts), stream>>>(p);
  return launch_check();
}

}  // extern "C"
