// Host-side internals shared by the translation units of libfused_swiglu_sm100.so:
// error reporting, the per-device cache and the tensor-map encoder (defined in fsw_api.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/fused_swiglu.h"

namespace fsw {

// Records the calling thread's error message and returns `code`.
int fail(int code, const char* fmt, ...);

#define FSW_CUDA(call)                                                                   \
  do {                                                                                   \
    cudaError_t e_ = (call);                                                             \
    if (e_ != cudaSuccess)                                                               \
      return fail(FSW_ECUDA, "%s failed: %s", #call, cudaGetErrorString(e_));            \
  } while (0)

struct DeviceInfo {
  bool ready = false;
  int sm_count = 0, cc_major = 0, cc_minor = 0;
  int64_t smem_optin = 0;
  int max_pairs = 0;  // co-resident 2-CTA clusters of the GEMM kernels
  uint32_t* status = nullptr;
  unsigned long long* clk_probe = nullptr;
  unsigned int* pace = nullptr;
  unsigned int* ew_ctrl = nullptr;
  unsigned int ew_next = 0;     // next slot of g_ew_ctrl to hand out
  unsigned int pace_next = 0;   // next slot of g_pace to hand out
  unsigned int pace_last = 0;   // slot the last paced launch used
};
// The current device's entry, set up on first use.
int ensure_device(DeviceInfo** out);

// Kernels this library has launched in this process.
extern std::atomic<long long> g_kernel_launches;

// Tensor map of a row-major array: rank 2 (outer rows of `inner` elements) or, with
// depth > 0, rank 3 (depth arrays of that shape, densely packed).  elem_bytes 2 (dtype
// FSW_BF16 / FSW_FP16) or 1 (bytes).  The box is box_outer rows of box_inner elements:
// 128 bytes wide with the 128-byte swizzle, or 64 bytes wide with the 64-byte swizzle.
// `row_elems` is the distance between rows in elements when the map covers a column
// range of a wider array (0 = dense, rows are `inner` elements apart).
int make_map(CUtensorMap* m, const void* ptr, int dtype, uint64_t inner, uint64_t outer,
             uint32_t box_outer, const char* what, uint32_t box_inner = 64,
             uint64_t row_elems = 0, uint64_t depth = 0, int elem_bytes = 2);

uint32_t make_idesc(int dtype, bool acc16, int a_major, int b_major, int m, int n);
uint64_t make_sdesc(uint32_t lbo_bytes, uint32_t sbo_bytes);
void fill_operand_desc(int major, uint64_t* desc, uint32_t* kadv);

// Options the other units read.
int64_t opt_l2_a();
int64_t opt_l2_b();
int64_t opt_l2_out();
int64_t opt_wait_limit_ms();
int64_t opt_stall_producer();

// Launches `kernel`.  With `dependent` it may be scheduled before the kernel ahead of it in the
// stream has finished (and, if that one is, ahead of that one's results): it has to call
// ptx::wait_predecessor before it touches anything another kernel of the chain writes or reads.
// The first kernel of a call is launched without it, so a call starts after all earlier work.
template <class... Params, class... Args>
inline cudaError_t launch_dependent(void (*kernel)(Params...), dim3 grid, int block, size_t smem, cudaStream_t st,
                                    bool dependent, int cluster, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (dependent) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  ++g_kernel_launches;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace fsw
