// Routed SwiGLU experts:  y_t = sum_j w_tj * (silu(x_t Wg_e) * (x_t Wu_e)) Wd_e,  e = index_tj,
// forward and backward.
//
//   plan      sort the (token, expert) pairs by expert           (fsw_experts.h)
//   gather    xs[row] = x[token]
//   GFWD      h = silu(xs Wg_e) * (xs Wu_e)        one dual GEMM over all experts
//   GNN       ys = h Wd_e                          fp32
//   combine   y_t = sum_j w_tj ys[row of (t, j)]   fp32, fixed order, one rounding
// backward
//   gather    dys[row] = dy[token]
//   GNT       dh = dys Wd_e^T                      fp32
//   gate      dw_tj = <h, dh>;  dg, du from w dh;  hs = w h
//   GTN       dWd_e = hs^T dys
//   GDX       dxs = dg Wg_e^T + du Wu_e^T          fp32
//   GDW       dWg_e, dWu_e = xs^T [dg | du]
//   combine   dx_t = sum_j dxs[row of (t, j)]
//
// The products are the tcgen05 kernel of fsw_gemm.cuh.  Measured on one B200, bf16: a training step
// of 8192 tokens, 2 of 8 experts of 4096 x 14336, 15.6 ms (1.11 PFLOP/s; the power-capped rate of a
// library product is 1.36); 2047 tokens, 6 of 64 experts of 4096 x 1408, forward, 776 us, bound by
// the operand traffic of 128-row tiles from L2 (256-row tiles, 676 against 600 us in a graph, lose
// more to padding at 192 rows an expert).  What becomes an operand of the next product (h, hs, dg, du) is rounded to the
// tensors' 16-bit type once, there (the tensor cores take 16-bit operands); g, u, dh, ys and
// dxs, the gate and the sums are fp32.  Nothing is summed with atomics: results do not
// depend on the order of execution.
#include <cstring>

#include "fsw_experts.h"
#include "fsw_gemm.cuh"

namespace fsw {

// -------------------------------------------------------------------- plan --
namespace {

// Adds this warp's pairs [begin, end) to its histogram.
__device__ __forceinline__ void count_pairs(const int* indices, int begin, int end, int E, int* hist, int lane) {
  for (int i = begin; i < end; i += 32) {
    int e = -1;
    if (i + lane < end) e = indices[i + lane];
    if (e < 0 || e >= E) e = -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same) - 1) hist[e] += __popc(same);
    __syncwarp();
  }
}

// Gives this warp's pairs their rows; next[e] is the next free row of expert e for this warp.
__device__ __forceinline__ void rank_pairs(const int* indices, int begin, int end, int E, int* next, int lane,
                                           int* pair_row, int* row_pair) {
  for (int i = begin; i < end; i += 32) {
    const int at = i + lane;
    int e = -1;
    if (at < end) e = indices[at];
    if (e < 0 || e >= E) e = -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    int row = -1;
    if (e >= 0) {
      row = next[e] + __popc(same & ((1u << lane) - 1u));
      row_pair[row] = at;
    }
    if (at < end) pair_row[at] = row;
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) next[e] += __popc(same);
    __syncwarp();
  }
}

// Exclusive prefix sum over the block of one value per thread (blockDim.x a multiple of 32).
__device__ __forceinline__ int block_prefix(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  __syncthreads();
  return before + x - v;
}

// Turns the experts' counts (count(e) for e < E) into offsets, the tile table and the
// padding's marks; all threads of one block take part.
template <class Count>
__device__ __forceinline__ void place_experts(const ExpertPlan& p, int* plan, int* warp_sums, Count count) {
  int base = 0;
  for (int e0 = 0; e0 < p.E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    const int c = e < p.E ? count(e) : 0;
    const int tiles = (c + p.tile_rows - 1) / p.tile_rows;
    int total;
    const int first = base + block_prefix(tiles, warp_sums, total);
    if (e < p.E) {
      plan[p.counts + e] = c;
      plan[p.offsets + e] = first * p.tile_rows;
      for (int j = 0; j < tiles; ++j) plan[p.tile_expert + first + j] = e;
      for (int r = c; r < tiles * p.tile_rows; ++r) plan[p.row_pair + (int64_t)first * p.tile_rows + r] = -1;
    }
    base += total;
  }
  if (threadIdx.x == 0) {
    plan[0] = base;
    plan[1] = base * p.tile_rows;
    plan[p.offsets + p.E] = base * p.tile_rows;
  }
}

// Pairs of warp `warp` of block `block`: a contiguous range, a multiple of 32 long.
__device__ __forceinline__ void warp_range(const ExpertPlan& p, int block, int warp, int& begin, int& end) {
  begin = (block * p.warps + warp) * kPlanWarpPairs;
  end = begin + kPlanWarpPairs < p.pairs ? begin + kPlanWarpPairs : p.pairs;
}

// Histogram per warp in shared memory; with `whole` the one block also places and ranks.
template <bool whole>
__global__ void __launch_bounds__(1024) plan_count_kernel(const ExpertPlan p, const int* indices, int* plan) {
  extern __shared__ int hist[];  // [warps][E]
  __shared__ int warp_sums[32];
  ptx::allow_successor();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < p.warps * p.E; i += blockDim.x) hist[i] = 0;
  __syncthreads();
  int begin, end;
  warp_range(p, blockIdx.x, warp, begin, end);
  count_pairs(indices, begin, end, p.E, hist + warp * p.E, lane);
  __syncthreads();
  auto total = [&](int e) {
    int c = 0;
    for (int w = 0; w < p.warps; ++w) c += hist[w * p.E + e];
    return c;
  };
  if (!whole) {
    for (int e = threadIdx.x; e < p.E; e += blockDim.x) plan[p.block_hist + (int64_t)blockIdx.x * p.E + e] = total(e);
    return;
  }
  place_experts(p, plan, warp_sums, total);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int next = plan[p.offsets + e];
    for (int w = 0; w < p.warps; ++w) {
      const int c = hist[w * p.E + e];
      hist[w * p.E + e] = next;
      next += c;
    }
  }
  __syncthreads();
  rank_pairs(indices, begin, end, p.E, hist + warp * p.E, lane, plan + p.pair_row, plan + p.row_pair);
}

// One block: block_hist[b][e] becomes the number of pairs of e before block b.
__global__ void __launch_bounds__(1024) plan_place_kernel(const ExpertPlan p, int* plan) {
  __shared__ int warp_sums[32];
  ptx::allow_successor();
  ptx::wait_predecessor();
  place_experts(p, plan, warp_sums, [&](int e) {
    int c = 0;
    int* h = plan + p.block_hist + e;
    for (int b = 0; b < p.blocks; b += 8) {  // eight loads in flight
      int v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = b + i < p.blocks ? h[(int64_t)(b + i) * p.E] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (b + i < p.blocks) {
          h[(int64_t)(b + i) * p.E] = c;
          c += v[i];
        }
    }
    return c;
  });
}

__global__ void __launch_bounds__(1024) plan_rank_kernel(const ExpertPlan p, const int* indices, int* plan) {
  extern __shared__ int hist[];
  ptx::allow_successor();
  ptx::wait_predecessor();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < p.warps * p.E; i += blockDim.x) hist[i] = 0;
  __syncthreads();
  int begin, end;
  warp_range(p, blockIdx.x, warp, begin, end);
  count_pairs(indices, begin, end, p.E, hist + warp * p.E, lane);
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += blockDim.x) {
    int next = plan[p.offsets + e] + plan[p.block_hist + (int64_t)blockIdx.x * p.E + e];
    for (int w = 0; w < p.warps; ++w) {
      const int c = hist[w * p.E + e];
      hist[w * p.E + e] = next;
      next += c;
    }
  }
  __syncthreads();
  rank_pairs(indices, begin, end, p.E, hist + warp * p.E, lane, plan + p.pair_row, plan + p.row_pair);
}

// --------------------------------------------------------- rows in and out --
// Blocks [0, T) copy one token's row to the rows of its k pairs; with zero padding, block
// T + e clears the rows behind the last of expert e.
__global__ void __launch_bounds__(128) gather_kernel(const ExpertPlan p, const int* __restrict__ plan,
                                                     const uint4* __restrict__ src, uint4* __restrict__ dst, int vecs) {
  ptx::allow_successor();
  ptx::wait_predecessor();
  if (blockIdx.x < static_cast<unsigned>(p.T)) {
    const int64_t t = blockIdx.x;
    const int* rows = plan + p.pair_row + t * p.k;
    for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
      const uint4 x = src[t * vecs + v];
      for (int j = 0; j < p.k; ++j) {
        const int r = rows[j];
        if (r >= 0) dst[static_cast<int64_t>(r) * vecs + v] = x;
      }
    }
    return;
  }
  const int e = blockIdx.x - p.T;
  const int64_t first = plan[p.offsets + e] + plan[p.counts + e], last = plan[p.offsets + e + 1];
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int64_t v = first * vecs + threadIdx.x; v < last * vecs; v += blockDim.x) dst[v] = zero;
}

template <typename W>
__device__ __forceinline__ float weight_value(const void* w, int64_t i) {
  if constexpr (sizeof(W) == 4) return static_cast<const float*>(w)[i];
  else if constexpr (std::is_same<W, __half>::value) return __half2float(static_cast<const __half*>(w)[i]);
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// S: type of the rows, T or float.
template <typename T, typename W, bool WEIGHTED, typename S>
__global__ void __launch_bounds__(128) combine_kernel(const ExpertPlan p, const int* __restrict__ plan,
                                                      const uint4* __restrict__ src, const void* __restrict__ weights,
                                                      uint4* __restrict__ y, int vecs) {
  constexpr int PARTS = sizeof(S) / 2;  // 16-byte vectors that 8 columns take
  ptx::allow_successor();
  ptx::wait_predecessor();
  const int64_t t = blockIdx.x;
  const int* rows = plan + p.pair_row + t * p.k;
  for (int v = blockIdx.y * blockDim.x + threadIdx.x; v < vecs; v += blockDim.x * gridDim.y) {
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
    for (int j0 = 0; j0 < p.k; j0 += 4) {
      uint4 x[4][PARTS];
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = j0 + j < p.k ? rows[j0 + j] : -1;
        w[j] = 0.0f;
#pragma unroll
        for (int h = 0; h < PARTS; ++h)
          x[j][h] = r >= 0 ? ld_stream(src + (static_cast<int64_t>(r) * vecs + v) * PARTS + h) : make_uint4(0u, 0u, 0u, 0u);
        if (r >= 0) {
          w[j] = WEIGHTED ? weight_value<W>(weights, t * p.k + j0 + j) : 1.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(&x[j][0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float lo, hi;
          if constexpr (PARTS == 2) {
            lo = __uint_as_float(q[2 * i]);
            hi = __uint_as_float(q[2 * i + 1]);
          } else {
            unpack2<T>(q[i], lo, hi);
          }
          acc[2 * i] = fmaf(w[j], lo, acc[2 * i]);
          acc[2 * i + 1] = fmaf(w[j], hi, acc[2 * i + 1]);
        }
      }
    }
    uint4 o;
    o.x = pack2<T>(acc[0], acc[1]);
    o.y = pack2<T>(acc[2], acc[3]);
    o.z = pack2<T>(acc[4], acc[5]);
    o.w = pack2<T>(acc[6], acc[7]);
    y[t * vecs + v] = o;
  }
}

// -------------------------------------------------------- gate and weights --
// One block per row.  h = silu(g) u;  dw = <h, dh>;  with d = w dh:  du = d silu(g),
// dg = d u silu'(g);  hs = w h.  fp32 in, 16-bit operands out.
// Rows of the padding get zeros, whatever the weights held.
template <typename T, typename W>
__global__ void __launch_bounds__(256) expert_gate_kernel(const ExpertPlan p, const int* __restrict__ plan,
                                                          const float4* __restrict__ dh, const float4* __restrict__ g,
                                                          const float4* __restrict__ u, const void* __restrict__ weights,
                                                          uint2* __restrict__ dg, uint2* __restrict__ du,
                                                          uint2* __restrict__ hs, void* dweights, int vecs) {
  ptx::allow_successor();
  ptx::wait_predecessor();
  const int64_t row = blockIdx.x;
  if (row >= plan[1]) return;
  const int pair = plan[p.row_pair + row];
  const float w = pair >= 0 ? weight_value<W>(weights, pair) : 0.0f;
  float dot = 0.0f;
  constexpr int kUnroll = 2;  // both vectors' loads in flight together
  for (int v0 = threadIdx.x; v0 < vecs; v0 += kUnroll * blockDim.x) {
    float4 vd[kUnroll], vg[kUnroll], vu[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int v = v0 + i * blockDim.x;
      if (pair >= 0 && v < vecs) {
        const int64_t at = row * vecs + v;
        vd[i] = __ldcs(dh + at);
        vg[i] = __ldcs(g + at);
        vu[i] = __ldcs(u + at);
      }
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int v = v0 + i * blockDim.x;
      if (v >= vecs) continue;
      uint2 odg = make_uint2(0u, 0u), odu = odg, ohs = odg;
      if (pair >= 0) {
        const float d4[4] = {vd[i].x, vd[i].y, vd[i].z, vd[i].w}, g4[4] = {vg[i].x, vg[i].y, vg[i].z, vg[i].w},
                    u4[4] = {vu[i].x, vu[i].y, vu[i].z, vu[i].w};
        float rg[4], ru[4], rh[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float s = sigmoid_f32(g4[c]), silu = g4[c] * s, h = silu * u4[c], d = w * d4[c];
          dot = fmaf(h, d4[c], dot);
          ru[c] = d * silu;
          rg[c] = d * u4[c] * fmaf(silu, 1.0f - s, s);
          rh[c] = w * h;
        }
        odg = make_uint2(pack2<T>(rg[0], rg[1]), pack2<T>(rg[2], rg[3]));
        odu = make_uint2(pack2<T>(ru[0], ru[1]), pack2<T>(ru[2], ru[3]));
        ohs = make_uint2(pack2<T>(rh[0], rh[1]), pack2<T>(rh[2], rh[3]));
      }
      const int64_t at = row * vecs + v;
      dg[at] = odg;
      du[at] = odu;
      if (hs != nullptr) hs[at] = ohs;
    }
  }
  if (dweights == nullptr || pair < 0) return;
  __shared__ float part[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
  __syncthreads();
  if (threadIdx.x == 0) {
    float total = 0.0f;
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) total += part[i];
    if constexpr (sizeof(W) == 4)
      static_cast<float*>(dweights)[pair] = total;
    else if constexpr (std::is_same<W, __half>::value)
      static_cast<__half*>(dweights)[pair] = __float2half_rn(total);
    else
      static_cast<__nv_bfloat16*>(dweights)[pair] = __float2bfloat16_rn(total);
  }
}

// A pair whose index is outside [0, E) has no row: its weight's gradient is zero.
template <typename W>
__global__ void __launch_bounds__(256) dropped_weights_kernel(const ExpertPlan p, const int* __restrict__ plan, W* dweights) {
  ptx::allow_successor();
  ptx::wait_predecessor();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i < p.pairs && plan[p.pair_row + i] < 0) dweights[i] = W(0.0f);
}

}  // namespace

int build_plan(const ExpertPlan& p, const int* indices, int* plan, cudaStream_t st) {
  const size_t smem = sizeof(int) * p.warps * p.E;  // at most 45 KB
  const int threads = p.warps * 32;
  if (p.blocks <= 1) {
    FSW_CUDA(launch_dependent(plan_count_kernel<true>, dim3(1), threads, smem, st, false, 1, p, indices, plan));
    return FSW_OK;
  }
  FSW_CUDA(launch_dependent(plan_count_kernel<false>, dim3(p.blocks), threads, smem, st, false, 1, p, indices, plan));
  FSW_CUDA(launch_dependent(plan_place_kernel, dim3(1), 1024, 0, st, true, 1, p, plan));
  FSW_CUDA(launch_dependent(plan_rank_kernel, dim3(p.blocks), threads, smem, st, true, 1, p, indices, plan));
  return FSW_OK;
}

int gather_rows(const ExpertPlan& p, const int* plan, const void* src, void* dst, int64_t row_bytes,
                bool zero_padding, bool dependent, cudaStream_t st) {
  FSW_CUDA(launch_dependent(gather_kernel, dim3(p.T + (zero_padding ? p.E : 0)), 128, 0, st, dependent, 1, p, plan,
                            static_cast<const uint4*>(src), static_cast<uint4*>(dst), (int)(row_bytes / 16)));
  return FSW_OK;
}

template <typename T, typename S>
static cudaError_t launch_combine(const ExpertPlan& p, const int* plan, const void* src, const void* weights, int wtype,
                                  void* y, int vecs, cudaStream_t st) {
  const uint4* s = static_cast<const uint4*>(src);
  uint4* o = static_cast<uint4*>(y);
  // a row per block; a row of few tokens is cut into pieces so that the GPU has some to do
  dim3 grid(p.T, p.T >= 512 ? 1 : (vecs + 127) / 128);
  if (weights == nullptr)
    return launch_dependent(combine_kernel<T, float, false, S>, grid, 128, 0, st, true, 1, p, plan, s, weights, o, vecs);
  if (wtype == FSW_FP32)
    return launch_dependent(combine_kernel<T, float, true, S>, grid, 128, 0, st, true, 1, p, plan, s, weights, o, vecs);
  return launch_dependent(combine_kernel<T, T, true, S>, grid, 128, 0, st, true, 1, p, plan, s, weights, o, vecs);
}

int combine_rows(const ExpertPlan& p, const int* plan, const void* src, bool src_f32, const void* weights, int wtype, void* y,
                 int64_t cols, int dtype, cudaStream_t st) {
  auto* run = dtype == FSW_BF16
                  ? (src_f32 ? launch_combine<__nv_bfloat16, float> : launch_combine<__nv_bfloat16, __nv_bfloat16>)
                  : (src_f32 ? launch_combine<__half, float> : launch_combine<__half, __half>);
  FSW_CUDA(run(p, plan, src, weights, wtype, y, (int)(cols / 8), st));
  return FSW_OK;
}

template <typename T, typename W>
static int launch_gate(const ExpertPlan& p, const int* plan, const void* dh, const void* g, const void* u, const void* weights,
                       void* dg, void* du, void* hs, void* dweights, int64_t cols, cudaStream_t st) {
  const int vecs = (int)(cols / 4);
  const int threads = vecs >= 512 ? 256 : vecs > 128 ? 128 : 64;
  FSW_CUDA(launch_dependent(expert_gate_kernel<T, W>, dim3(p.rows), threads, 0, st, true, 1, p, plan,
                            static_cast<const float4*>(dh), static_cast<const float4*>(g), static_cast<const float4*>(u),
                            weights, static_cast<uint2*>(dg), static_cast<uint2*>(du), static_cast<uint2*>(hs), dweights, vecs));
  if (dweights != nullptr)
    FSW_CUDA(launch_dependent(dropped_weights_kernel<W>, dim3((p.pairs + 255) / 256), 256, 0, st, true, 1, p, plan,
                              static_cast<W*>(dweights)));
  return FSW_OK;
}

// -------------------------------------------------------------------- GEMMs --
namespace {

template <int MODE, int CG, int NSUB, typename T>
int launch_grouped_one(const GemmParams& p, int grid, cudaStream_t st) {
  // per device: the attribute belongs to the current device's copy of the kernel
  static std::atomic<uint64_t> prepared{0};
  int dev = 0;
  FSW_CUDA(cudaGetDevice(&dev));
  if (!(prepared.load() >> (dev & 63) & 1)) {
    FSW_CUDA(cudaFuncSetAttribute(gemm_kernel<MODE, CG, NSUB, T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  TileCfg<MODE, CG, NSUB>::SMEM_BYTES));
    prepared.fetch_or(1ull << (dev & 63));
  }
  FSW_CUDA(launch_dependent(gemm_kernel<MODE, CG, NSUB, T, false>, dim3(grid), TileCfg<MODE, CG, NSUB>::THREADS,
                            TileCfg<MODE, CG, NSUB>::SMEM_BYTES, st, true, CG, p));
  return FSW_OK;
}

// Columns of one tile.
template <int MODE>
constexpr int tile_cols(int nsub) {
  return (is_dual(MODE) ? 128 : 256) * nsub;
}

// 512-column tiles of a CTA pair run at 1 / 0.84 of the speed of 256-column ones on full
// tiles (the dense kernels' sweep); columns beyond N are wasted.
template <int MODE>
int choose_nsub(int64_t N) {
  const double wide = (double)N / (double)((N + tile_cols<MODE>(2) - 1) / tile_cols<MODE>(2) * tile_cols<MODE>(2));
  const double narrow = (double)N / (double)((N + tile_cols<MODE>(1) - 1) / tile_cols<MODE>(1) * tile_cols<MODE>(1));
  return wide >= 0.84 * narrow ? 2 : 1;
}

// Fills in what all grouped launches share and launches.  M: rows of the output tiles' grid
// (all rows for the row-grouped modes, one weight's rows for the weight gradients).
template <int MODE>
int run_grouped(GemmParams& p, const ExpertPlan& plan, const int* plan_dev, int64_t M, int64_t N, int cg, int nsub,
                int dtype, DeviceInfo* d, cudaStream_t st) {
  p.M = (int)M;
  p.N = (int)N;
  p.ldc = (int)N;
  p.grp_meta = plan_dev;
  p.grp_counts = plan_dev + plan.counts;
  p.grp_offsets = plan_dev + plan.offsets;
  p.grp_tile_expert = plan_dev + plan.tile_expert;
  p.grp_experts = plan.E;
  p.num_m_tiles = is_grouped_k(MODE) ? (int)((M + 128 * cg - 1) / (128 * cg)) : plan.tiles;
  p.num_n_tiles = (int)((N + tile_cols<MODE>(nsub) - 1) / tile_cols<MODE>(nsub));
  const long long tiles = (long long)p.num_m_tiles * p.num_n_tiles * (is_grouped_k(MODE) ? plan.E : 1);
  if (tiles >= (1ll << 31)) return fail(FSW_EINVAL, "too many tiles");
  p.status = d->status;
  p.clk_probe = d->clk_probe;
  p.l2_a = (int)opt_l2_a();
  p.l2_b = (int)opt_l2_b();
  p.l2_out = (int)opt_l2_out();
  p.wait_limit_ns = (unsigned long long)opt_wait_limit_ms() * 1000000ull;
  p.stall_producer = (int)opt_stall_producer();
  const int a_major = a_is_mn(MODE) ? MAJOR_MN : MAJOR_K, b_major = b_is_k(MODE) ? MAJOR_K : MAJOR_MN;
  fill_operand_desc(a_major, &p.a_desc, &p.a_kadv);
  fill_operand_desc(b_major, &p.b_desc, &p.b_kadv);
  p.idesc = make_idesc(dtype, false, a_major, b_major, 128 * cg, 256);
  p.group_m = 12;  // rows of tiles swept together; sqrt(2 * 74), as the dense kernels'
  const int workers = cg == 2 ? d->max_pairs : d->sm_count;
  const int grid = (int)(tiles < workers ? tiles : workers) * cg;
#define FSW_GROUPED(CG, NSUB)                                                                       \
  return dtype == FSW_BF16 ? launch_grouped_one<MODE, CG, NSUB, __nv_bfloat16>(p, grid, st)         \
                           : launch_grouped_one<MODE, CG, NSUB, __half>(p, grid, st)
  if (cg == 1) FSW_GROUPED(1, 1);
  if (nsub == 1) FSW_GROUPED(2, 1);
  FSW_GROUPED(2, 2);
#undef FSW_GROUPED
}

// One call's sizes and buffers.
struct Experts {
  ExpertPlan plan;
  int64_t d, f, d_out;
  int dtype, cg;
  DeviceInfo* dev;
  cudaStream_t st;
  const int* plan_dev;

  // Rows of the A boxes: all 128, or as many as there are pairs if those are few (then
  // nothing behind an expert's last row may be read later).
  int a_rows(bool whole) const {
    if (whole || plan.pairs > 120) return 128;
    return (plan.pairs + 7) / 8 * 8;
  }

  // c (rows, N) = a (rows, K) @ w_e, w (E, K, N), or w (E, N, K) transposed
  template <int MODE>
  int product(const void* a, const void* w, void* c, int64_t K, int64_t N, bool whole) const {
    GemmParams p;
    memset(&p, 0, sizeof(p));
    int rc;
    const int ar = a_rows(whole);
    p.grp_a_rows = ar == 128 ? 0 : ar;
    const int nsub = cg == 2 ? choose_nsub<MODE>(N) : 1;
    if ((rc = make_map(&p.a0, a, dtype, K, plan.rows, ar, "rows")) != FSW_OK) return rc;
    if (b_is_k(MODE))
      rc = make_map(&p.b0, w, dtype, K, N, 256 / cg, "weights", 64, 0, plan.E);
    else
      rc = make_map(&p.b0, w, dtype, N, K, 64, "weights", 64, 0, plan.E);
    if (rc != FSW_OK) return rc;
    p.b1 = p.b0;
    p.c0_ptr = c;
    p.num_k_blocks = (int)((K + 63) / 64);
    return run_grouped<MODE>(p, plan, plan_dev, plan.rows, N, cg, nsub, dtype, dev, st);
  }

  int swiglu(const void* xs, const void* wg, const void* wu, void* h, void* g, void* u) const {
    GemmParams p;
    memset(&p, 0, sizeof(p));
    int rc;
    const int ar = a_rows(g != nullptr);
    p.grp_a_rows = ar == 128 ? 0 : ar;
    const int nsub = cg == 2 ? choose_nsub<MODE_GFWD>(f) : 1;
    if ((rc = make_map(&p.a0, xs, dtype, d, plan.rows, ar, "xs")) != FSW_OK) return rc;
    if ((rc = make_map(&p.b0, wg, dtype, f, d, 64, "w_gate", 64, 0, plan.E)) != FSW_OK) return rc;
    if ((rc = make_map(&p.b1, wu, dtype, f, d, 64, "w_up", 64, 0, plan.E)) != FSW_OK) return rc;
    if ((rc = make_map(&p.so, h, dtype, f, plan.rows, 32, "h", 32)) != FSW_OK) return rc;
    p.sg = p.su = p.so;  // g and u are written by plain stores
    p.store_gu = g != nullptr;
    p.c0_ptr = g;
    p.c1_ptr = u;
    p.c2_ptr = h;
    p.num_k_blocks = (int)((d + 63) / 64);
    return run_grouped<MODE_GFWD>(p, plan, plan_dev, plan.rows, f, cg, nsub, dtype, dev, st);
  }

  int grad_rows(const void* dg, const void* du, const void* wg, const void* wu, void* dxs) const {
    GemmParams p;
    memset(&p, 0, sizeof(p));
    int rc;
    const int nsub = cg == 2 ? choose_nsub<MODE_GDX>(d) : 1;
    if ((rc = make_map(&p.a0, dg, dtype, f, plan.rows, 128, "dg")) != FSW_OK) return rc;
    if ((rc = make_map(&p.a1, du, dtype, f, plan.rows, 128, "du")) != FSW_OK) return rc;
    if ((rc = make_map(&p.b0, wg, dtype, f, d, 256 / cg, "w_gate", 64, 0, plan.E)) != FSW_OK) return rc;
    if ((rc = make_map(&p.b1, wu, dtype, f, d, 256 / cg, "w_up", 64, 0, plan.E)) != FSW_OK) return rc;
    p.c0_ptr = dxs;
    p.num_k_blocks = (int)((f + 63) / 64);
    return run_grouped<MODE_GDX>(p, plan, plan_dev, plan.rows, d, cg, nsub, dtype, dev, st);
  }

  // c0, c1 (E, M, N) = a^T @ b0, b1 over each expert's rows; c1 only for MODE_GDW
  template <int MODE>
  int grad_weight(const void* a, const void* b0, const void* b1, void* c0, void* c1, int64_t M, int64_t N) const {
    GemmParams p;
    memset(&p, 0, sizeof(p));
    int rc;
    // pairs of CTAs halve the operand traffic, but rows beyond M are wasted
    const int wcg = M % 256 == 0 || M > 1024 ? 2 : 1;
    const int nsub = wcg == 2 ? choose_nsub<MODE>(N) : 1;
    if ((rc = make_map(&p.a0, a, dtype, M, plan.rows, 64, "rows")) != FSW_OK) return rc;
    if ((rc = make_map(&p.b0, b0, dtype, N, plan.rows, 64, "gradients")) != FSW_OK) return rc;
    p.b1 = p.b0;
    if (b1 != nullptr && (rc = make_map(&p.b1, b1, dtype, N, plan.rows, 64, "gradients")) != FSW_OK) return rc;
    p.c0_ptr = c0;
    p.c1_ptr = c1;
    return run_grouped<MODE>(p, plan, plan_dev, M, N, wcg, nsub, dtype, dev, st);
  }
};

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace

int check_experts(int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out, int dtype, int wtype) {
  if (dtype != FSW_BF16 && dtype != FSW_FP16) return fail(FSW_EINVAL, "unknown dtype %d", dtype);
  if (wtype != FSW_FP32 && wtype != dtype) return fail(FSW_EINVAL, "weights must be fp32 or of the tensors' type");
  if (T < 0 || k < 1 || k > FSW_MAX_TOP_K) return fail(FSW_EINVAL, "bad number of tokens %lld or top_k %d", (long long)T, k);
  if (E < 1 || E > FSW_MAX_EXPERTS) return fail(FSW_EINVAL, "number of experts %d is not in [1, %d]", E, FSW_MAX_EXPERTS);
  if (d <= 0 || f <= 0 || d_out <= 0 || d >= (1 << 24) || f >= (1 << 24) || d_out >= (1 << 24))
    return fail(FSW_EINVAL, "bad feature sizes %lld, %lld, %lld", (long long)d, (long long)f, (long long)d_out);
  return FSW_OK;
}

static int check_16bit(int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out, int dtype, int wtype, ExpertPlan* plan) {
  int rc = check_experts(T, k, E, d, f, d_out, dtype, wtype);
  if (rc != FSW_OK) return rc;
  if ((d & 7) || (f & 7) || (d_out & 7))
    return fail(FSW_EINVAL, "feature sizes %lld, %lld, %lld must be multiples of 8", (long long)d, (long long)f, (long long)d_out);
  if (T >= (1ll << 31) || !make_plan(plan, T, k, E, choose_tile_rows(T * k, E)))
    return fail(FSW_EINVAL, "too many tokens");
  return FSW_OK;
}

// Byte offsets of what a forward keeps for its backward (plan, xs, g, u), the same without
// a backward (plan, xs), and of the scratch of each direction.
struct ExpertBuffers {
  int64_t xs, g, u, saved;        // saved: plan at 0
  int64_t h, ys, scratch;         // forward scratch (training: h, ys; inference: plus plan and xs)
  int64_t dys, dh, dg, du, hs, dxs, back;  // backward scratch; dxs takes dh's place
};
static ExpertBuffers expert_buffers(const ExpertPlan& p, int64_t d, int64_t f, int64_t d_out) {
  ExpertBuffers b;
  const int64_t R = p.rows;
  b.xs = align256(p.ints * 4);
  b.g = b.xs + align256(R * d * 2);
  b.u = b.g + align256(R * f * 4);
  b.saved = b.u + align256(R * f * 4);
  b.h = 0;
  b.ys = align256(R * f * 2);
  b.scratch = b.ys + align256(R * d_out * 4);
  b.dys = 0;
  b.dh = align256(R * d_out * 2);
  b.dxs = b.dh;
  b.dg = b.dh + align256(R * (f > d ? f : d) * 4);
  b.du = b.dg + align256(R * f * 2);
  b.hs = b.du + align256(R * f * 2);
  b.back = b.hs + align256(R * f * 2);
  return b;
}

}  // namespace fsw

using namespace fsw;

extern "C" {

int fsw_experts_sizes(int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out, int64_t* saved_bytes,
                      int64_t* forward_bytes, int64_t* inference_bytes, int64_t* backward_bytes) {
  ExpertPlan plan;
  int rc = check_16bit(T, k, E, d, f, d_out, FSW_BF16, FSW_FP32, &plan);
  if (rc != FSW_OK) return rc;
  const ExpertBuffers b = expert_buffers(plan, d, f, d_out);
  if (saved_bytes) *saved_bytes = b.saved;
  if (forward_bytes) *forward_bytes = b.scratch;
  if (inference_bytes) *inference_bytes = b.g + b.scratch;
  if (backward_bytes) *backward_bytes = b.back;
  return FSW_OK;
}

int fsw_experts_forward(const void* x, const void* weights, const void* indices, const void* w_gate, const void* w_up,
                        const void* w_down, void* y, void* saved, int64_t saved_bytes, void* scratch,
                        int64_t scratch_bytes, int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out, int dtype,
                        int weights_dtype, void* stream) {
  Experts x_;
  int rc = check_16bit(T, k, E, d, f, d_out, dtype, weights_dtype, &x_.plan);
  if (rc != FSW_OK) return rc;
  if (T == 0) return FSW_OK;
  if (!x || !weights || !indices || !w_gate || !w_up || !w_down || !y || !scratch) return fail(FSW_EINVAL, "NULL pointer");
  if (!aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(w_down) || !aligned16(y) ||
      !aligned16(saved) || !aligned16(scratch))
    return fail(FSW_EINVAL, "pointers must be 16-byte aligned");
  const ExpertBuffers b = expert_buffers(x_.plan, d, f, d_out);
  const bool train = saved != nullptr;
  if ((train && saved_bytes < b.saved) || scratch_bytes < (train ? b.scratch : b.g + b.scratch))
    return fail(FSW_EINVAL, "buffers of %lld and %lld bytes are too small (see fsw_experts_sizes)",
                (long long)saved_bytes, (long long)scratch_bytes);
  if ((rc = ensure_device(&x_.dev)) != FSW_OK) return rc;
  x_.d = d;
  x_.f = f;
  x_.d_out = d_out;
  x_.dtype = dtype;
  x_.cg = x_.plan.tile_rows / 128;
  x_.st = static_cast<cudaStream_t>(stream);
  if (!train && few_rows_apply(T, k, d, f, x_.dev->sm_count) && scratch_bytes >= T * k * f * 4)
    return experts_few_rows(x, weights, weights_dtype, static_cast<const int*>(indices), w_gate, w_up, w_down, y,
                            static_cast<float*>(scratch), T, k, E, d, f, d_out, dtype, x_.dev, x_.st);
  char* keep = static_cast<char*>(train ? saved : scratch);
  char* tmp = static_cast<char*>(scratch) + (train ? 0 : b.g);
  int* plan = reinterpret_cast<int*>(keep);
  x_.plan_dev = plan;
  if ((rc = build_plan(x_.plan, static_cast<const int*>(indices), plan, x_.st)) != FSW_OK) return rc;
  if ((rc = gather_rows(x_.plan, plan, x, keep + b.xs, d * 2, train, true, x_.st)) != FSW_OK) return rc;
  if ((rc = x_.swiglu(keep + b.xs, w_gate, w_up, tmp + b.h, train ? keep + b.g : nullptr, train ? keep + b.u : nullptr)) != FSW_OK)
    return rc;
  if ((rc = x_.product<MODE_GNN>(tmp + b.h, w_down, tmp + b.ys, f, d_out, false)) != FSW_OK) return rc;
  return combine_rows(x_.plan, plan, tmp + b.ys, true, weights, weights_dtype, y, d_out, dtype, x_.st);
}

int fsw_experts_backward(const void* dy, const void* weights, const void* w_gate, const void* w_up, const void* w_down,
                         const void* saved, int64_t saved_bytes, void* scratch, int64_t scratch_bytes, void* dx,
                         void* dweights, void* dw_gate, void* dw_up, void* dw_down, int64_t T, int k, int E, int64_t d,
                         int64_t f, int64_t d_out, int dtype, int weights_dtype, void* stream) {
  Experts x_;
  int rc = check_16bit(T, k, E, d, f, d_out, dtype, weights_dtype, &x_.plan);
  if (rc != FSW_OK) return rc;
  if (!dw_gate != !dw_up) return fail(FSW_EINVAL, "dw_gate and dw_up are computed together: pass both or neither");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t wbytes = (int64_t)E * d * f * 2;
  if (T == 0) {
    DeviceInfo* dev;
    if ((rc = ensure_device(&dev)) != FSW_OK) return rc;
    if (dw_gate) FSW_CUDA(cudaMemsetAsync(dw_gate, 0, wbytes, st));
    if (dw_up) FSW_CUDA(cudaMemsetAsync(dw_up, 0, wbytes, st));
    if (dw_down) FSW_CUDA(cudaMemsetAsync(dw_down, 0, (int64_t)E * f * d_out * 2, st));
    return FSW_OK;
  }
  if (!dy || !weights || !w_gate || !w_up || !w_down || !saved || !scratch) return fail(FSW_EINVAL, "NULL pointer");
  if (!aligned16(dy) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(w_down) || !aligned16(saved) ||
      !aligned16(scratch) || !aligned16(dx) || !aligned16(dw_gate) || !aligned16(dw_up) || !aligned16(dw_down))
    return fail(FSW_EINVAL, "pointers must be 16-byte aligned");
  const ExpertBuffers b = expert_buffers(x_.plan, d, f, d_out);
  if (saved_bytes < b.saved || scratch_bytes < b.back)
    return fail(FSW_EINVAL, "buffers of %lld and %lld bytes are too small (see fsw_experts_sizes)",
                (long long)saved_bytes, (long long)scratch_bytes);
  if ((rc = ensure_device(&x_.dev)) != FSW_OK) return rc;
  x_.d = d;
  x_.f = f;
  x_.d_out = d_out;
  x_.dtype = dtype;
  x_.cg = x_.plan.tile_rows / 128;
  x_.st = st;
  const char* keep = static_cast<const char*>(saved);
  char* tmp = static_cast<char*>(scratch);
  const int* plan = reinterpret_cast<const int*>(keep);
  x_.plan_dev = plan;
  if ((rc = gather_rows(x_.plan, plan, dy, tmp + b.dys, d_out * 2, true, false, st)) != FSW_OK) return rc;
  if ((rc = x_.product<MODE_GNT>(tmp + b.dys, w_down, tmp + b.dh, d_out, f, true)) != FSW_OK) return rc;
  void* hs = dw_down ? tmp + b.hs : nullptr;
  const bool w32 = weights_dtype == FSW_FP32;
  auto* gate = dtype == FSW_BF16 ? (w32 ? launch_gate<__nv_bfloat16, float> : launch_gate<__nv_bfloat16, __nv_bfloat16>)
                                 : (w32 ? launch_gate<__half, float> : launch_gate<__half, __half>);
  if ((rc = gate(x_.plan, plan, tmp + b.dh, keep + b.g, keep + b.u, weights, tmp + b.dg, tmp + b.du, hs, dweights, f, st)) != FSW_OK) return rc;
  const char *dg = tmp + b.dg, *du = tmp + b.du;
  if (dw_down && (rc = x_.grad_weight<MODE_GTN>(hs, tmp + b.dys, nullptr, dw_down, nullptr, f, d_out)) != FSW_OK) return rc;
  if (dx) {
    if ((rc = x_.grad_rows(dg, du, w_gate, w_up, tmp + b.dxs)) != FSW_OK) return rc;
    if ((rc = combine_rows(x_.plan, plan, tmp + b.dxs, true, nullptr, FSW_FP32, dx, d, dtype, st)) != FSW_OK) return rc;
  }
  if (dw_gate && (rc = x_.grad_weight<MODE_GDW>(keep + b.xs, dg, du, dw_gate, dw_up, d, f)) != FSW_OK) return rc;
  return FSW_OK;
}

}  // extern "C"
