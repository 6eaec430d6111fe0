// Routed SwiGLU experts for a handful of tokens: reading the weights is all there is to do.
//
//   h[p] = silu(x_t Wg_e) * (x_t Wu_e)       for every pair p = (t, j), e its expert
//   y[t] = sum over j of w_tj h[p] Wd_e      one sum over the k * f rows of the k experts
//
// The matrix kernels would give a 128-row tile to every expert that has a row: with 6 experts
// of 1408 columns only 66 CTAs read, and 148 SMs are needed to draw the HBM's rate.  Here a
// block reads 128 columns, 16 lanes of 16 bytes each, two rows of the weight to a warp; the rows
// are divided over the 8 warps of a block and over the CTAs of a cluster, whose sums are added
// through (distributed) shared memory in a fixed order.  Nothing is sorted or copied, and h and
// the sums stay in fp32.  Two tokens with one expert read it twice, the second time from L2.
//
// Measured on one B200, weights in HBM, graph replay (the matrix kernels in brackets): one token,
// 6 of 64 experts of 4096 x 1408: 53 us (70); 2 of 8 of 4096 x 14336: 141 us (193); four tokens, 31
// of 128 of 2048 x 768: 70 us (86).  With more column tiles than the SMs can hold at once the matrix
// kernels read faster (7 experts of 4096 x 14336: 401 against 459 us): few_rows_apply draws the line.
#include "fsw_experts.h"
#include "fsw_gemm.cuh"

namespace fsw {
namespace {

constexpr int kCols = 128, kThreads = 256, kWarps = 8;
constexpr int kUnroll = 4;

template <typename T>
__device__ __forceinline__ void fma8(float (&acc)[8], const uint4& w, float x) {
  const uint32_t* q = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    unpack2<T>(q[i], lo, hi);
    acc[2 * i] = fmaf(x, lo, acc[2 * i]);
    acc[2 * i + 1] = fmaf(x, hi, acc[2 * i + 1]);
  }
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

// Sum of this CTA's partial sums: acc of the two half-warps, then of the warps, into
// total[128]; part is [8][128].
__device__ __forceinline__ void block_total(float (&acc)[8], float* part, float* total, int lane, int warp) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], 16);
  if (lane < 16)
#pragma unroll
    for (int i = 0; i < 8; ++i) part[warp * kCols + lane * 8 + i] = acc[i];
  __syncthreads();
  if (threadIdx.x < kCols) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += part[w * kCols + threadIdx.x];
    total[threadIdx.x] = s;
  }
  __syncthreads();
}

// Column c of the tile summed over the cluster's CTAs, in rank order.
__device__ __forceinline__ float cluster_total(const float* total, int c, int splits) {
  if (splits == 1) return total[c];
  float s = 0.0f;
  const uint32_t at = ptx::smem_u32(total + c);
  for (int r = 0; r < splits; ++r) s += ld_cluster(ptx::mapa(at, r));
  return s;
}

// Grid (splits * column tiles, pairs), cluster (splits, 1).
template <typename T>
__global__ void __launch_bounds__(kThreads) few_gate_kernel(const T* __restrict__ x, const int* __restrict__ indices,
                                                            const T* __restrict__ wg, const T* __restrict__ wu,
                                                            float* __restrict__ h, int k, int E, int d, int f, int splits) {
  extern __shared__ float xs[];  // this CTA's part of the token's row
  __shared__ float part[kWarps * kCols], total_g[kCols], total_u[kCols];
  ptx::allow_successor();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits, pair = blockIdx.y;
  const int e = indices[pair];
  const int k0 = static_cast<int>(static_cast<long long>(d) * rank / splits);
  const int k1 = static_cast<int>(static_cast<long long>(d) * (rank + 1) / splits);
  const int col = tile * kCols + (lane & 15) * 8;
  const bool on = e >= 0 && e < E && col < f;
  for (int i = k0 + threadIdx.x; i < k1; i += kThreads) {
    float lo, hi;
    unpack2<T>(reinterpret_cast<const unsigned short*>(x)[static_cast<int64_t>(pair / k) * d + i], lo, hi);
    xs[i - k0] = lo;
  }
  __syncthreads();
  float ag[8], au[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) ag[i] = au[i] = 0.0f;
  if (on) {
    const int64_t base = static_cast<int64_t>(e) * d * f + col;
    constexpr int step = 2 * kWarps;
    for (int r0 = k0 + warp * 2 + (lane >> 4); r0 < k1; r0 += step * kUnroll) {
      uint4 vg[kUnroll], vu[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        const int r = r0 + i * step;
        if (r < k1) {
          vg[i] = ld_stream(wg + base + static_cast<int64_t>(r) * f);
          vu[i] = ld_stream(wu + base + static_cast<int64_t>(r) * f);
        }
      }
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        const int r = r0 + i * step;
        if (r < k1) {
          fma8<T>(ag, vg[i], xs[r - k0]);
          fma8<T>(au, vu[i], xs[r - k0]);
        }
      }
    }
  }
  block_total(ag, part, total_g, lane, warp);
  block_total(au, part, total_u, lane, warp);
  if (splits > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  const int per = kCols / splits, c = rank * per + static_cast<int>(threadIdx.x);
  if (static_cast<int>(threadIdx.x) < per && tile * kCols + c < f) {
    const float g = cluster_total(total_g, c, splits), u = cluster_total(total_u, c, splits);
    h[static_cast<int64_t>(pair) * f + tile * kCols + c] = g * sigmoid_f32(g) * u;
  }
  if (splits > 1) {  // the totals are read until here
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
}

// Grid (splits * column tiles, tokens), cluster (splits, 1).
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) few_down_kernel(const float* __restrict__ h, const int* __restrict__ indices,
                                                            const W* __restrict__ weights, const T* __restrict__ wd,
                                                            T* __restrict__ y, int k, int E, int f, int d_out, int splits) {
  extern __shared__ float hw[];  // this CTA's part of the token's k * f values w h
  __shared__ float part[kWarps * kCols], total[kCols];
  ptx::allow_successor();
  ptx::wait_predecessor();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int64_t t = blockIdx.y;
  const int rows = k * f;
  const int q0 = static_cast<int>(static_cast<long long>(rows) * rank / splits);
  const int q1 = static_cast<int>(static_cast<long long>(rows) * (rank + 1) / splits);
  for (int q = q0 + threadIdx.x; q < q1; q += kThreads) {
    const int64_t pair = t * k + q / f;
    float w;
    if constexpr (sizeof(W) == 4)
      w = weights[pair];
    else {
      float hi;
      unpack2<T>(reinterpret_cast<const unsigned short*>(weights)[pair], w, hi);
    }
    hw[q - q0] = w * h[t * rows + q];
  }
  __syncthreads();
  const int col = tile * kCols + (lane & 15) * 8;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  for (int j = q0 / f; j < k && j * f < q1; ++j) {
    const int e = indices[t * k + j];
    if (e < 0 || e >= E || col >= d_out) continue;
    const int a = (q0 > j * f ? q0 : j * f), b = (q1 < (j + 1) * f ? q1 : (j + 1) * f);
    const T* base = wd + (static_cast<int64_t>(e) * f - static_cast<int64_t>(j) * f) * d_out + col;
    constexpr int step = 2 * kWarps, unroll = 2 * kUnroll;
    for (int r0 = a + warp * 2 + (lane >> 4); r0 < b; r0 += step * unroll) {
      uint4 v[unroll];
#pragma unroll
      for (int i = 0; i < unroll; ++i) {
        const int r = r0 + i * step;
        if (r < b) v[i] = ld_stream(base + static_cast<int64_t>(r) * d_out);
      }
#pragma unroll
      for (int i = 0; i < unroll; ++i) {
        const int r = r0 + i * step;
        if (r < b) fma8<T>(acc, v[i], hw[r - q0]);
      }
    }
  }
  block_total(acc, part, total, lane, warp);
  if (splits > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  const int per = kCols / splits / 2, c = rank * (kCols / splits) + 2 * static_cast<int>(threadIdx.x);
  if (static_cast<int>(threadIdx.x) < per && tile * kCols + c < d_out)
    reinterpret_cast<uint32_t*>(y)[(t * d_out + tile * kCols + c) >> 1] =
        pack2<T>(cluster_total(total, c, splits), cluster_total(total, c + 1, splits));
  if (splits > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
}

constexpr int kFewSmem = 32 * 1024;  // of the part of a row a CTA keeps

// CTAs that share a column tile: enough blocks for two per SM, parts that fit, at least 64 rows each.
int choose_splits(int64_t blocks, int64_t rows, int sms) {
  int s = 1;
  while (s < 8 && ((blocks * s < 2 * sms && rows >= 128 * s) || rows * 4 > (int64_t)kFewSmem * s)) s *= 2;
  return s;
}

}  // namespace

bool few_rows_apply(int64_t T, int k, int64_t d, int64_t f, int sms) {
  return (T <= 2 || (T <= 8 && T * k * ((f + kCols - 1) / kCols) <= 2 * sms)) && d * 4 <= 8 * kFewSmem &&
         k * f * 4 <= 8 * (int64_t)kFewSmem;
}

int experts_few_rows(const void* x, const void* weights, int wtype, const int* indices, const void* w_gate, const void* w_up,
                     const void* w_down, void* y, float* h, int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out,
                     int dtype, DeviceInfo* dev, cudaStream_t st) {
  const int tiles1 = (int)((f + kCols - 1) / kCols), tiles2 = (int)((d_out + kCols - 1) / kCols);
  const int s1 = choose_splits(T * k * tiles1, d, dev->sm_count), s2 = choose_splits(T * tiles2, k * f, dev->sm_count);
  const size_t m1 = (size_t)((d + s1 - 1) / s1 + 1) * 4, m2 = (size_t)((k * f + s2 - 1) / s2 + 1) * 4;
  const dim3 g1(s1 * tiles1, (unsigned)(T * k)), g2(s2 * tiles2, (unsigned)T);
  auto run = [&](auto tag) -> cudaError_t {
    using E16 = decltype(tag);
    cudaError_t e = launch_dependent(few_gate_kernel<E16>, g1, kThreads, m1, st, false, s1, static_cast<const E16*>(x), indices,
                                     static_cast<const E16*>(w_gate), static_cast<const E16*>(w_up), h, k, E, (int)d, (int)f, s1);
    if (e != cudaSuccess) return e;
    if (wtype == FSW_FP32)
      return launch_dependent(few_down_kernel<E16, float>, g2, kThreads, m2, st, true, s2, h, indices,
                              static_cast<const float*>(weights), static_cast<const E16*>(w_down), static_cast<E16*>(y), k, E,
                              (int)f, (int)d_out, s2);
    return launch_dependent(few_down_kernel<E16, E16>, g2, kThreads, m2, st, true, s2, h, indices,
                            static_cast<const E16*>(weights), static_cast<const E16*>(w_down), static_cast<E16*>(y), k, E,
                            (int)f, (int)d_out, s2);
  };
  FSW_CUDA(dtype == FSW_BF16 ? run(__nv_bfloat16()) : run(__half()));
  return FSW_OK;
}

}  // namespace fsw
