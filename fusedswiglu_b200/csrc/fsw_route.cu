// Routing of tokens to experts: scores, selection, weights, and the gradient of the logits.
//
//   s = softmax(z) or sigmoid(z) per token, c = s + bias (bias only steers the selection)
//   num_groups > 1: a group's score is the sum of its two largest c; only experts of the
//   topk_groups best groups stay eligible
//   idx = the k largest c, ties to the lowest index;  w = scale * s[idx] (/ sum of s[idx])
//
// One warp per token; expert e sits in lane e % 32, so a row is read once, coalesced, and
// lives in registers.  Selection is k rounds of redux.sync over order-preserving 32-bit
// keys.  The bytes (T*E logits in, T*k*8 out) would take 2.7 us for 16384 x 256 fp32
// logits; instructions bound the kernel.  Measured on one B200: 13 us for the top 8 of these,
// 27 with a bias, 37 with a bias and 4 of 8 groups; 8191 x 128 bf16 7.1 us, its gradient 5.9.
//
// The selection is that of exact arithmetic.  Without a bias s grows with z, so z itself is
// compared and nothing is rounded.  With a bias, or for group scores, c is computed in
// fp32 with a bound on its error; a row in which two neighbours in the order are closer
// than their bounds is selected again from 64-bit scores.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "fsw_host.h"

namespace fsw {
namespace {

constexpr int kRouteWarps = 4;
constexpr unsigned kFull = 0xffffffffu;

struct RouteParams {
  const void* logits;
  int64_t ld;          // elements between rows of logits
  const float* bias;   // (E) or nullptr
  float* weights;      // (T, k)
  int* indices;        // (T, k)
  const float* dweights;  // backward: (T, k)
  void* dlogits;          // backward: (T, E), dense
  int64_t T;
  int E, k, groups, topk_groups;
  int sigmoid, renorm;
  float scale;
  uint32_t group_magic;  // e / (E / groups) = umulhi(e, group_magic) for e < 1024; 0: groups of one
};

template <typename T>
__device__ __forceinline__ float as_f32(T v);
template <>
__device__ __forceinline__ float as_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float as_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float as_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}

// Keys: 0 = not eligible or already taken, 1 = masked (-inf or NaN), else the value's bits
// mapped so that unsigned order is value order (-FLT_MAX maps to 2^23).  -0 and +0 are equal.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 1u;  // -inf and NaN
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  if (!(v > -INFINITY)) return 1ull;
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// Largest key of the warp; ties to the lowest index.
__device__ __forceinline__ uint32_t warp_best(uint32_t key, int index, int& winner) {
  const uint32_t top = __reduce_max_sync(kFull, key);
  const unsigned lanes = __ballot_sync(kFull, key == top);
  if ((lanes & (lanes - 1u)) == 0u)  // one lane, nearly always: a vote and a shuffle, not a second reduction
    winner = __shfl_sync(kFull, index, __ffs(lanes) - 1);
  else
    winner = static_cast<int>(__reduce_min_sync(kFull, key == top ? static_cast<unsigned>(index) : 0x7fffffffu));
  return top;
}
__device__ __forceinline__ unsigned long long warp_best(unsigned long long key, int index, int& winner) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long k2 = __shfl_xor_sync(kFull, key, o);
    const int i2 = __shfl_xor_sync(kFull, index, o);
    if (k2 > key || (k2 == key && i2 < index)) {
      key = k2;
      index = i2;
    }
  }
  winner = index;
  return key;
}

// A run of picks among the lanes' keys: each lane keeps its two best at hand, and looks through its
// keys for the next one only when it has given both.
template <int EPL>
struct Picker {
  uint32_t (&key)[EPL];
  int lane;
  uint32_t first = 0u, second = 0u, taken = 0u;  // taken: keys of this lane already picked
  int first_at = 0, second_at = 0;
  bool have_second = true;

  __device__ __forceinline__ Picker(uint32_t (&k)[EPL], int l) : key(k), lane(l) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      if (key[i] > first) {  // strict: of equal keys the lowest index comes first
        second = first;
        second_at = first_at;
        first = key[i];
        first_at = i;
      } else if (key[i] > second) {
        second = key[i];
        second_at = i;
      }
    }
  }

  __device__ __forceinline__ uint32_t take(int& winner) {
    const uint32_t top = warp_best(first, lane + 32 * first_at, winner);
    bool again = false;
    if ((winner & 31) == lane) {
      taken |= 1u << first_at;
      again = !have_second;
      first = second;
      first_at = second_at;
      have_second = false;
    }
    if (__any_sync(kFull, again)) {
      uint32_t best = 0u;
      int at = 0;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const uint32_t k = ((taken >> i) & 1u) ? 0u : key[i];
        if (k > best) {
          best = k;
          at = i;
        }
      }
      if (again) {
        first = best;
        first_at = at;
      }
    }
    return top;
  }
};

// Sum of the two largest c of group `lane / lanes_per_group`, from the warp's row of c in
// shared memory.  Masked experts hold -inf and add nothing; a group of only such scores -inf.
template <typename F>
__device__ __forceinline__ void group_score(const F* c, int lane, int groups, int size, F& score) {
  const int lpg = groups <= 1 ? 32 : 32 / groups >= 16 ? 16 : 32 / groups >= 8 ? 8 : 32 / groups >= 4 ? 4 : 32 / groups >= 2 ? 2 : 1;
  const int g = lane / lpg, r = lane % lpg;
  const F low = -INFINITY;
  F m1 = low, m2 = low;
  if (g < groups)
    for (int j = r; j < size; j += lpg) {
      const F v = c[g * size + j];
      m2 = max(m2, min(m1, v));
      m1 = max(m1, v);
    }
  for (int o = lpg >> 1; o > 0; o >>= 1) {
    const F a = __shfl_xor_sync(kFull, m1, o), b = __shfl_xor_sync(kFull, m2, o);
    m2 = max(max(m2, b), min(m1, a));
    m1 = max(m1, a);
  }
  // lane g of the result (all lanes of a group agree)
  const F sum = (m2 > low) ? m1 + m2 : m1;
  score = __shfl_sync(kFull, sum, lane < groups ? lane * lpg : 0);
  if (lane >= groups) score = low;
}

// Error bound of a score as route_kernel computes it for the selection, and of c = s + bias, in
// units of 2^-23.  The exponential by ex2.approx is good to a few units and |argument| roundings
// of 2^-24 each; sigmoid: s changes by s (1 - s) of that, plus the sum and the reciprocal: 8 + |z|
// units of s cover it.  softmax: up to 40 roundings from the sum of the row, and the rounded
// difference d = z - max: 64 + |d| units of s.
__device__ __forceinline__ float score_tolerance(bool sigmoid, float s, float arg, float c) {
  return 1.2e-7f * (s * (fabsf(arg) + (sigmoid ? 8.0f : 64.0f)) + fabsf(c)) + 1e-37f;
}

// The selection from scores in 64 bits: lane j gets pick j.  Runs for the few rows whose fp32
// order is not certain; small rather than fast (loops, the row's keys in shared memory), so
// that it costs the other rows neither registers nor instruction cache.
template <typename T>
__device__ __noinline__ int select64(const RouteParams& p, const T* row, float zmax, double* c, int lane) {
  double sum = 0.0;
  if (!p.sigmoid) {
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32) {
      const float z = as_f32(row[e]);
      if (z != -INFINITY) sum += exp(static_cast<double>(z) - static_cast<double>(zmax));
    }
    sum = warp_sum(sum);
  }
#pragma unroll 1
  for (int e = lane; e < p.E; e += 32) {
    const float z = as_f32(row[e]);
    const double d = exp(p.sigmoid ? -static_cast<double>(z) : static_cast<double>(z) - static_cast<double>(zmax));
    double v = p.sigmoid ? 1.0 / (1.0 + d) : d / sum;
    if (p.bias != nullptr) v += static_cast<double>(p.bias[e]);
    c[e] = (z > -INFINITY && v > -INFINITY) ? v : -INFINITY;
  }
  __syncwarp();
  uint32_t allowed = ~0u;
  const int size = p.E / p.groups;
  if (p.groups > 1) {
    double gs;
    group_score<double>(c, lane, p.groups, size, gs);
    unsigned long long key = lane < p.groups ? order_key(gs) : 0ull;
    allowed = 0u;
#pragma unroll 1
    for (int j = 0; j < p.topk_groups; ++j) {
      int win;
      warp_best(key, lane, win);
      if (win == lane) key = 0ull;
      allowed |= 1u << win;
    }
    __syncwarp();
  }
  unsigned long long* key = reinterpret_cast<unsigned long long*>(c);
#pragma unroll 1
  for (int e = lane; e < p.E; e += 32) {
    const double v = p.bias != nullptr ? c[e] : static_cast<double>(as_f32(row[e]));
    key[e] = (p.groups == 1 || ((allowed >> (e / size)) & 1u)) ? order_key(v) : 0ull;
  }
  int mine = 0;
#pragma unroll 1
  for (int j = 0; j < p.k; ++j) {
    unsigned long long best = 0ull;
    int at = lane, win;
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32)  // each lane reads and clears only its own keys
      if (key[e] > best) {
        best = key[e];
        at = e;
      }
    warp_best(best, at, win);
    if ((win & 31) == lane) key[win] = 0ull;
    if (lane == j) mine = win;
  }
  __syncwarp();
  return mine;
}

// Lane j < k holds logit z of pick j: its share p of the selected scores (renorm), or its
// score s.  Shares are exact ratios: softmax shares do not need the row's sum; sigmoid
// shares go through log(sigmoid) where the scores themselves would underflow.
__device__ __forceinline__ float pick_share(const RouteParams& p, float z, int lane) {
  const bool on = lane < p.k;
  if (!p.sigmoid) {
    const float m = warp_max(on ? z : -INFINITY);
    const float v = (on && z > -INFINITY) ? expf(z - m) : (z != z && on) ? z : 0.0f;
    const float sum = warp_sum(v);
    return sum > 0.0f ? v / sum : sum;  // sum 0: every pick is masked; NaN stays
  }
  float v = on ? 1.0f / (1.0f + expf(-z)) : 0.0f;
  float sum = warp_sum(v);
  if (sum < 1e-30f) {
    const float ls = fminf(z, 0.0f) - log1pf(expf(-fabsf(z)));
    const float m = warp_max(on ? ls : -INFINITY);
    v = (on && ls > -INFINITY) ? expf(ls - m) : 0.0f;
    sum = warp_sum(v);
  }
  return sum != 0.0f ? v / sum : 0.0f;
}

// One warp per token.  EPL = experts per lane (a power of two, 32 * EPL >= E).
template <typename T, int EPL, bool SIGMOID, bool BIAS, bool GROUPS>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const __grid_constant__ RouteParams p) {
  extern __shared__ double route_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double* crow64 = route_smem + static_cast<size_t>(warp) * p.E;  // with a bias or groups only
  float* crow = reinterpret_cast<float*>(crow64);
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (t >= p.T) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  float z[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    z[i] = e < p.E ? as_f32(row[e]) : -INFINITY;
  }
  float zmax = -INFINITY, denom = 1.0f;
  if (!SIGMOID) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) zmax = fmaxf(zmax, z[i]);
    zmax = warp_max(zmax);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += z[i] == -INFINITY ? 0.0f : expf(z[i] - zmax);  // NaN and +inf make it NaN
    denom = warp_sum(sum);
  }
  const float rdenom = 1.0f / denom, base = zmax > -INFINITY ? zmax : 0.0f;
  auto score = [&](float v) {  // -inf scores 0
    return SIGMOID ? __fdividef(1.0f, 1.0f + __expf(-v)) : __expf(v - base) * rdenom;
  };
  // The scores enter the selection only with a bias or groups.  `worst` bounds the error of
  // every c of the row: s (8 + |z|) <= 18 where that bound is near the truth (z <= 10; beyond
  // it s is 1 to the last bits), and s (64 + |d|) <= 66 max s.
  constexpr bool by_score = BIAS || GROUPS;
  float c[EPL];
  float worst = 0.0f;
  if constexpr (by_score) {
    float largest = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      c[i] = score(z[i]);
      if (BIAS && e < p.E) c[i] += p.bias[e];
      const bool open = z[i] > -INFINITY && c[i] > -INFINITY;  // neither -inf nor NaN
      largest = fmaxf(largest, open ? fabsf(c[i]) : 0.0f);
      c[i] = open ? c[i] : -INFINITY;
    }
    worst = 1.2e-7f * ((SIGMOID ? 18.0f : 66.0f * rdenom) + warp_max(largest)) + 1e-37f;
  }

  bool unsure = false;
  uint32_t allowed = ~0u;
  const int size = GROUPS ? p.E / p.groups : p.E;
  if constexpr (GROUPS) {
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane + 32 * i < p.E) crow[lane + 32 * i] = c[i];
    __syncwarp();
    float gs;
    group_score<float>(crow, lane, p.groups, size, gs);
    uint32_t key = lane < p.groups ? order_key(gs) : 0u;
    allowed = 0u;
    uint32_t prev = 0u;
    const int rounds = p.topk_groups < p.groups ? p.topk_groups + 1 : p.topk_groups;
    for (int j = 0; j < rounds; ++j) {
      int win;
      const uint32_t top = warp_best(key, lane, win);
      if (win == lane) key = 0u;
      if (j < p.topk_groups) allowed |= 1u << win;
      // only the border between kept and dropped groups matters; sums of two: two bounds each,
      // and the rounding of the sums
      if (j == p.topk_groups && top > 1u)
        unsure = key_value(prev) - key_value(top) <= 4.0f * worst + 1.2e-7f * (fabsf(key_value(prev)) + fabsf(key_value(top)));
      prev = top;
    }
    __syncwarp();
  }

  int mine = 0;
  if (!unsure) {
    uint32_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      const uint32_t g = p.group_magic ? __umulhi(e, p.group_magic) : e;
      const bool eligible = e < p.E && (!GROUPS || ((allowed >> (g & 31u)) & 1u));
      key[i] = eligible ? order_key(BIAS ? c[i] : z[i]) : 0u;
    }
    Picker<EPL> picker(key, lane);
    if constexpr (!BIAS) {
      for (int j = 0; j < p.k; ++j) {
        int win;
        picker.take(win);
        if (lane == j) mine = win;
      }
    } else {
      // Neighbours in the fp32 order must differ by more than their bounds, through the first
      // expert that is dropped.  Equal logits with equal biases tie exactly in any precision;
      // a run of them must end in a certain gap too, which is looked for a few places further.
      // The row's bound settles nearly all neighbours; the others are looked at one by one.
      float prev_c = INFINITY;
      int prev_win = 0;
      bool tie = false;
      for (int j = 0; j <= p.k + 8; ++j) {
        int win;
        const uint32_t top = picker.take(win);
        if (j < p.k && lane == j) mine = win;
        if (top <= 1u) {  // from here on only masked experts, which rank by index, or none
          tie = false;
          if (j >= p.k) break;
          continue;
        }
        const float cw = key_value(top);
        tie = false;
        if (prev_c - cw <= 2.0f * worst) {
          const float za = as_f32(row[prev_win]), zb = as_f32(row[win]);
          tie = za == zb && p.bias[prev_win] == p.bias[win];
          if (!tie)
            unsure = prev_c - cw <= score_tolerance(SIGMOID, score(za), SIGMOID ? za : za - base, prev_c) +
                                        score_tolerance(SIGMOID, score(zb), SIGMOID ? zb : zb - base, cw);
        }
        if (unsure || (j >= p.k && !tie)) break;
        prev_c = cw;
        prev_win = win;
      }
      if (tie) unsure = true;
    }
  }
  if (by_score && unsure) mine = select64<T>(p, row, zmax, crow64, lane);

  const float zp = lane < p.k ? as_f32(row[mine]) : -INFINITY;
  float w;
  if (p.renorm) {
    w = pick_share(p, zp, lane);
    if (!SIGMOID && !(denom == denom)) w = denom;  // a NaN or +inf in a softmax row: NaN
  } else {
    w = zp == -INFINITY ? 0.0f : SIGMOID ? 1.0f / (1.0f + expf(-zp)) : expf(zp - zmax) / denom;
    if (!SIGMOID && zp == -INFINITY && !(denom == denom)) w = denom;
  }
  if (lane < p.k) {
    p.weights[t * p.k + lane] = w * p.scale;
    p.indices[t * p.k + lane] = mine;
  }
}

// d logits.  ds_j = scale * dw_j;  renormalised: share p_j, dz_j = p_j (ds_j - sum p ds)
// [* (1 - s_j) for sigmoid], others 0;  plain softmax: dz_e = s_e ([e picked] ds - sum s ds);
// plain sigmoid: dz_j = ds_j s_j (1 - s_j).  Reads the row again only for plain softmax;
// writes it whole (T*E is what bounds it).
template <typename T, int EPL>
__global__ void __launch_bounds__(kRouteWarps * 32) route_backward_kernel(const RouteParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (t >= p.T) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.ld;
  const bool on = lane < p.k;
  int idx = on ? p.indices[t * p.k + lane] : -1;
  if (idx >= p.E) idx = -1;
  const float ds = on ? p.scale * p.dweights[t * p.k + lane] : 0.0f;
  const float zp = idx >= 0 ? as_f32(row[idx]) : -INFINITY;

  float z[EPL];
  float zmax = -INFINITY, denom = 1.0f;
  const bool whole_row = !p.sigmoid && !p.renorm;
  if (whole_row) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      z[i] = e < p.E ? as_f32(row[e]) : -INFINITY;
      zmax = fmaxf(zmax, z[i]);
    }
    zmax = warp_max(zmax);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) sum += z[i] == -INFINITY ? 0.0f : expf(z[i] - zmax);
    denom = warp_sum(sum);
  }

  float mine;         // gradient of pick `lane`
  float dot = 0.0f;   // what every other expert of a plain softmax row loses, times s_e
  if (p.renorm) {
    const float share = pick_share(p, zp, lane);
    const float mean = warp_sum(share * ds);
    mine = share * (ds - mean);
    if (p.sigmoid) mine *= 1.0f / (1.0f + expf(zp));  // 1 - s without cancellation
  } else if (p.sigmoid) {
    const float s = 1.0f / (1.0f + expf(-zp));
    mine = zp == -INFINITY ? 0.0f : ds * s * (1.0f / (1.0f + expf(zp)));
  } else {
    const float s = zp == -INFINITY ? 0.0f : expf(zp - zmax) / denom;
    dot = warp_sum(s * ds);
    mine = s * (ds - dot);
  }

  T* out = static_cast<T*>(p.dlogits) + t * p.E;
  const float rdenom = 1.0f / denom;
  float v[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    v[i] = 0.0f;
    if (whole_row) v[i] = z[i] == -INFINITY ? 0.0f : -expf(z[i] - zmax) * rdenom * dot;
  }
  for (int j = 0; j < p.k; ++j) {
    const int e = __shfl_sync(kFull, idx, j);
    const float g = __shfl_sync(kFull, mine, j);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (lane + 32 * i == e) v[i] = g;
  }
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    if (e < p.E) out[e] = from_f32<T>(v[i]);
  }
}

// What a call does not ask for is not in its kernel: the tests of it per expert cost as much
// as the selection.
template <typename T, int EPL, bool SIGMOID>
void launch_kind(const RouteParams& p, unsigned blocks, size_t smem, cudaStream_t st) {
  auto* kernel = p.bias != nullptr
                     ? (p.groups > 1 ? route_kernel<T, EPL, SIGMOID, true, true> : route_kernel<T, EPL, SIGMOID, true, false>)
                     : (p.groups > 1 ? route_kernel<T, EPL, SIGMOID, false, true> : route_kernel<T, EPL, SIGMOID, false, false>);
  kernel<<<blocks, kRouteWarps * 32, smem, st>>>(p);
}
template <typename T, int EPL>
void launch_forward(const RouteParams& p, unsigned blocks, size_t smem, cudaStream_t st) {
  if (p.sigmoid)
    launch_kind<T, EPL, true>(p, blocks, smem, st);
  else
    launch_kind<T, EPL, false>(p, blocks, smem, st);
}

template <typename T>
cudaError_t launch_route(const RouteParams& p, bool backward, cudaStream_t st) {
  const unsigned blocks = static_cast<unsigned>((p.T + kRouteWarps - 1) / kRouteWarps);
  const size_t smem = (!backward && (p.groups > 1 || p.bias != nullptr)) ? static_cast<size_t>(kRouteWarps) * p.E * sizeof(double) : 0;
  ++g_kernel_launches;
#define FSW_ROUTE(EPL)                                                         \
  if (p.E <= 32 * EPL) {                                                       \
    if (backward)                                                              \
      route_backward_kernel<T, EPL><<<blocks, kRouteWarps * 32, 0, st>>>(p);   \
    else                                                                       \
      launch_forward<T, EPL>(p, blocks, smem, st);                             \
    return cudaGetLastError();                                                 \
  }
  FSW_ROUTE(1)
  FSW_ROUTE(2)
  FSW_ROUTE(4)
  FSW_ROUTE(8)
  FSW_ROUTE(16)
  FSW_ROUTE(32)
#undef FSW_ROUTE
  return cudaErrorInvalidValue;
}

int check_route(int64_t T, int64_t ld, int E, int k, int dtype, int score, int groups, int topk_groups, float scale) {
  if (dtype != FSW_BF16 && dtype != FSW_FP16 && dtype != FSW_FP32) return fail(FSW_EINVAL, "unknown dtype %d", dtype);
  if (score != FSW_SCORE_SOFTMAX && score != FSW_SCORE_SIGMOID) return fail(FSW_EINVAL, "unknown score function %d", score);
  if (T < 0 || T >= (1ll << 31)) return fail(FSW_EINVAL, "bad number of tokens %lld", (long long)T);
  if (E < 1 || E > FSW_MAX_EXPERTS) return fail(FSW_EINVAL, "number of experts %d is not in [1, %d]", E, FSW_MAX_EXPERTS);
  if (k < 1 || k > FSW_MAX_TOP_K || k > E)
    return fail(FSW_EINVAL, "top_k %d is not in [1, min(%d, number of experts %d)]", k, FSW_MAX_TOP_K, E);
  if (groups < 1 || groups > 32 || E % groups)
    return fail(FSW_EINVAL, "num_groups %d must be in [1, 32] and divide the number of experts %d", groups, E);
  if (topk_groups < 1 || topk_groups > groups)
    return fail(FSW_EINVAL, "topk_groups %d is not in [1, num_groups %d]", topk_groups, groups);
  if (k > topk_groups * (E / groups))
    return fail(FSW_EINVAL, "top_k %d exceeds the %d experts of %d groups", k, topk_groups * (E / groups), topk_groups);
  if (!std::isfinite(scale)) return fail(FSW_EINVAL, "scale is not finite");
  if (ld < E) return fail(FSW_EINVAL, "row stride %lld is less than the number of experts %d", (long long)ld, E);
  return FSW_OK;
}

}  // namespace
}  // namespace fsw

using namespace fsw;

extern "C" {

int fsw_route(const void* logits, int64_t ld, const void* bias, void* weights, void* indices, int64_t T, int E, int k,
              int dtype, int score, int renormalize, float scale, int num_groups, int topk_groups, void* stream) {
  int rc = check_route(T, ld, E, k, dtype, score, num_groups, topk_groups, scale);
  if (rc != FSW_OK) return rc;
  if (T == 0) return FSW_OK;
  if (!logits || !weights || !indices) return fail(FSW_EINVAL, "NULL pointer");
  DeviceInfo* d = nullptr;
  if ((rc = ensure_device(&d)) != FSW_OK) return rc;
  RouteParams p = {};
  p.logits = logits;
  p.ld = ld;
  p.bias = static_cast<const float*>(bias);
  p.weights = static_cast<float*>(weights);
  p.indices = static_cast<int*>(indices);
  p.T = T;
  p.E = E;
  p.k = k;
  p.groups = num_groups;
  p.topk_groups = topk_groups;
  p.sigmoid = score == FSW_SCORE_SIGMOID;
  p.renorm = renormalize != 0;
  p.scale = scale;
  const unsigned size = (unsigned)(E / num_groups);
  p.group_magic = size > 1 ? (uint32_t)(((1ull << 32) + size - 1) / size) : 0u;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FSW_BF16)
    FSW_CUDA(launch_route<__nv_bfloat16>(p, false, st));
  else if (dtype == FSW_FP16)
    FSW_CUDA(launch_route<__half>(p, false, st));
  else
    FSW_CUDA(launch_route<float>(p, false, st));
  return FSW_OK;
}

int fsw_route_backward(const void* logits, int64_t ld, const void* indices, const void* dweights, void* dlogits,
                       int64_t T, int E, int k, int dtype, int score, int renormalize, float scale, void* stream) {
  int rc = check_route(T, ld, E, k, dtype, score, 1, 1, scale);
  if (rc != FSW_OK) return rc;
  if (T == 0) return FSW_OK;
  if (!logits || !indices || !dweights || !dlogits) return fail(FSW_EINVAL, "NULL pointer");
  DeviceInfo* d = nullptr;
  if ((rc = ensure_device(&d)) != FSW_OK) return rc;
  RouteParams p = {};
  p.logits = logits;
  p.ld = ld;
  p.indices = static_cast<int*>(const_cast<void*>(indices));
  p.dweights = static_cast<const float*>(dweights);
  p.dlogits = dlogits;
  p.T = T;
  p.E = E;
  p.k = k;
  p.groups = p.topk_groups = 1;
  p.sigmoid = score == FSW_SCORE_SIGMOID;
  p.renorm = renormalize != 0;
  p.scale = scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FSW_BF16)
    FSW_CUDA(launch_route<__nv_bfloat16>(p, true, st));
  else if (dtype == FSW_FP16)
    FSW_CUDA(launch_route<__half>(p, true, st));
  else
    FSW_CUDA(launch_route<float>(p, true, st));
  return FSW_OK;
}

}  // extern "C"
