// Products in 8-bit floating point (e4m3) with a scale for each block of 128:
//
//   y[t, n] = sum over b of xs[t, b] * ws[n / 128, b] * sum over k in block b of xq[t, k] wq[n, k]
//
// and the SwiGLU gate on top of two of them, with its result quantised again:
//   h = silu(x Wg) * (x Wu),  hs[t, b] = 2^e with the smallest e that makes the largest |h| of
//   the block at most 448,  hq = round(h / hs).
// Activations have one scale per row and 128 columns, weights one per 128 x 128.  Activation
// scales made here are powers of two: dividing by them is exact, so a value is rounded once;
// the weights' scales may be any fp32 numbers.
//
// The tensor cores add the 128 products of a block in tensor memory (kind::f8f6f4, fp32);
// the blocks' sums are scaled and added in fp32 registers by the epilogue warps, beside the
// MMAs of the next block.  A tile is 128 tokens x 256 weight rows per CTA (256 x 256 per CTA
// pair); in 512 cycles of MMAs per block and pair the epilogue reads 128 x 256 sums per SM
// from tensor memory (256 cycles) and issues 128 packed FMAs per scheduler.
//
// Measured on one B200: 8192 x 4096 -> 14336 432 us (2.2 PFLOP/s) alone, where the same kernel without
// the scaling takes 323 us; 77 x 14336 -> 4104 23 us; one token 4096 -> 14336 19 us with its
// quantisation.  Bound by the epilogue: a warp needs about 575 cycles from a block's sums to their
// release and 235 to the next, next to 512 of MMAs.  256-column MMAs with two regions: four
// regions of 128 would hide more, but read the rows twice as often from shared memory (580 us).
//
// Few rows: the A box holds only the rows there are, and with fewer tiles than SMs the K
// blocks of a tile are divided over the CTAs of a cluster, which add their sums through
// distributed shared memory in a fixed order.
#include <cuda_fp8.h>

#include <cstring>

#include "fsw_experts.h"
#include "fsw_gemm.cuh"

namespace fsw {
namespace {

constexpr int kBlock = 128;
constexpr int kMaxSplits = 8;  // portable cluster size

struct Fp8Params {
  CUtensorMap a, b0, b1;
  uint64_t desc;
  uint32_t idesc;
  const float* xs;          // xs[row * xs_row + block * xs_block]
  int64_t xs_row, xs_block;
  const float *ws0, *ws1;   // (E, row blocks, K blocks)
  int ws_rows, num_kb;
  int M, N;                 // output rows and columns
  int num_m_tiles, num_n_tiles, group_m;
  void* out;                // (M, N) of the output type
  int wide_rows;            // every row of out starts on a 32-byte boundary
  uint8_t* hq;              // dual: (M, N) e4m3
  float* hs;                // dual: hs[block * hs_pitch + row]
  int64_t hs_pitch;
  const int *grp_meta, *grp_tile_expert, *grp_offsets, *grp_counts;  // grp_meta nullptr: one weight
  int a_rows;               // rows of an A box
  int splits;               // CTAs of a cluster that share a tile's K blocks (CG == 1, one tile each)
  uint32_t* status;
  unsigned long long wait_limit_ns;
  int stall_producer;
};

template <int CG>
struct Fp8Cfg {
  static constexpr int A_BYTES = 128 * kBlock;
  static constexpr int B_BYTES = 256 / CG * kBlock;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = CG == 2 ? 6 : 4;
  static constexpr int EPI_WARPS = 8;
  static constexpr int AMAX_BYTES = 2 * EPI_WARPS * 32 * 4;  // DUAL: row maxima, two tiles in turn
  static constexpr int SCALE_SLOTS = 4;
  static constexpr int SCALE_BYTES = SCALE_SLOTS * 2 * 128 * 4;
  static constexpr int BAR_BYTES = 512;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + AMAX_BYTES + SCALE_BYTES + BAR_BYTES + 1024;
  // Three warpgroups: producer, MMA issuer, scale warp and an idle one; twice four epilogue warps.  The
  // block starts with 168 registers a thread (168 * 384 = 64512); the first group keeps 104 and
  // the others take 200 (104 * 128 + 200 * 256 = 64512): 128 sums, two chunks of 16 in flight.
  static constexpr int THREADS = 128 + 32 * EPI_WARPS;
  static constexpr int REGS_FIRST = 104, REGS_EPILOGUE = 200;
  static_assert(REGS_FIRST * 128 + REGS_EPILOGUE * 32 * EPI_WARPS <= 168 * THREADS, "registers");
  static_assert(SMEM_BYTES <= kSmemBudget, "shared memory");
  // A split tile's sums overlay the operand stages: 128 rows of 256 columns, padded so that
  // the 16-byte writes of lanes with adjacent rows fall into different banks.
  static constexpr int PART_LD = 260;
  static_assert(128 * PART_LD * 4 <= STAGES * STAGE_BYTES, "partial sums");
};

template <int CG>
__device__ __forceinline__ void mma_f8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
        "}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Completes the loads in flight; the registers pass through it, so that no use moves ahead.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// acc[0..15] += s * t[0..15], as packed pairs.
__device__ __forceinline__ void scaled_add16(float* acc, const uint32_t (&t)[16], float s) {
  unsigned long long s2;
  asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    unsigned long long t2, a2;
    asm("mov.b64 %0, {%1, %2};" : "=l"(t2) : "r"(t[2 * i]), "r"(t[2 * i + 1]));
    asm("mov.b64 %0, {%1, %2};" : "=l"(a2) : "f"(acc[2 * i]), "f"(acc[2 * i + 1]));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a2) : "l"(t2), "l"(s2));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[2 * i]), "=f"(acc[2 * i + 1]) : "l"(a2));
  }
}

// Scale of a block whose largest magnitude has these bits: the smallest power of two 2^e with
// amax <= 448 * 2^e (448 = 1.75 * 2^8), at least 2^-126; 1 for a block of zeros; NaN if the
// block holds inf or NaN (its products are then NaN).  `inv` is the exact inverse.
__device__ __forceinline__ float block_scale(uint32_t amax_bits, float& inv) {
  if (amax_bits == 0u) {
    inv = 1.0f;
    return 1.0f;
  }
  if (amax_bits >= 0x7f800000u) {
    inv = 1.0f;
    return __uint_as_float(0x7fc00000u);
  }
  int e = static_cast<int>(amax_bits >> 23) - ((amax_bits & 0x7fffffu) <= 0x600000u ? 8 : 7);  // biased exponent
  if (e < 1) e = 1;
  inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
  return __uint_as_float(static_cast<uint32_t>(e) << 23);
}
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Not volatile: the loads of all shares may be in flight together (the barriers around them are).
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// Columns [col, col + 32) of a row of N, rounded to T; whole sectors where the rows are aligned.
template <typename T>
__device__ __forceinline__ void store_row32(T* row, int col, int N, bool wide, const float* v) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
  if (wide) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (col + h * 16 < N)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row + col + h * 16),
                     "r"(w[8 * h]), "r"(w[8 * h + 1]), "r"(w[8 * h + 2]), "r"(w[8 * h + 3]), "r"(w[8 * h + 4]),
                     "r"(w[8 * h + 5]), "r"(w[8 * h + 6]), "r"(w[8 * h + 7])
                     : "memory");
  } else {
#pragma unroll
    for (int h = 0; h < 4; ++h)
      if (col + h * 8 < N) ptx::st_global_v4(row + col + h * 8, w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
  }
}

struct Fp8Work {
  int m_tile, n_tile, expert, rows;  // rows: valid rows from the tile's first on
};

// --------------------------------------------------------------------- GEMM --
template <int CG, bool DUAL, typename T>
__global__ void __launch_bounds__(Fp8Cfg<CG>::THREADS, 1) fp8_gemm_kernel(const __grid_constant__ Fp8Params p) {
  using C = Fp8Cfg<CG>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = ptx::smem_u32(smem_raw);
  const uint32_t smem_base = (raw_u32 + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - raw_u32);
  const uint32_t amax_off = STAGES * C::STAGE_BYTES;
  // [slot][which of the tile's two weight blocks][row]: the row's scale times the block's
  float* scale_ring = reinterpret_cast<float*>(smem_gen + amax_off + C::AMAX_BYTES);
  const uint32_t bar_base = smem_base + amax_off + C::AMAX_BYTES + C::SCALE_BYTES;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
  const uint32_t misc_off = (bar_base - smem_base) + 8u * (2 * STAGES + 4);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_gen + misc_off);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem_gen + misc_off + 4);
  const AbortCtl ctl{abort_flag, p.status, p.wait_limit_ns ? p.wait_limit_ns : kWaitLimitNs};
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = (CG == 2 || p.splits > 1) ? ptx::cluster_ctarank() : 0u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar(s), 1);
      ptx::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(tfull_bar(a), 2);  // the MMAs' commit and the scale warp
      ptx::mbar_init(tempty_bar(a), C::EPI_WARPS * CG);
    }
    *abort_flag = 0u;
    ptx::fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tensormap(&p.a);
    ptx::prefetch_tensormap(&p.b0);
    if (DUAL) ptx::prefetch_tensormap(&p.b1);
  }
  if (warp == 1) {
    ptx::tmem_alloc<CG>(bar_base + 8u * (2 * STAGES + 4), 512);
    ptx::tmem_relinquish<CG>();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (CG == 2) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  ptx::allow_successor();
  // The kernel ahead makes the rows (and the plan); a dense weight is older than both, so the
  // producer fills the pipeline with its tiles before it waits.
  const bool early = p.grp_meta == nullptr && warp == 0 && lane == 0 && !p.stall_producer;
  if (!early) ptx::wait_predecessor();

  const int cluster = CG * p.splits;
  const int num_clusters = gridDim.x / cluster, cluster_id = blockIdx.x / cluster;
  const int m_tiles = p.grp_meta != nullptr ? p.grp_meta[0] : p.num_m_tiles;
  // this CTA's share of a tile's K blocks
  const int share = p.splits > 1 ? static_cast<int>(rank) : 0;
  const int kb0 = static_cast<int>(static_cast<long long>(p.num_kb) * share / p.splits);
  const int kb1 = static_cast<int>(static_cast<long long>(p.num_kb) * (share + 1) / p.splits);
  auto get_work = [&](int idx, Fp8Work& w) {
    const long long t = cluster_id + static_cast<long long>(idx) * num_clusters;
    if (t >= static_cast<long long>(m_tiles) * p.num_n_tiles) return false;
    decode_tile_order(static_cast<int>(t), m_tiles, p.num_n_tiles, p.group_m, w.m_tile, w.n_tile);
    const int row0 = w.m_tile * 128 * CG;
    if (p.grp_meta != nullptr) {
      w.expert = p.grp_tile_expert[w.m_tile];
      w.rows = p.grp_offsets[w.expert] + p.grp_counts[w.expert] - row0;
    } else {
      w.expert = 0;
      w.rows = p.M - row0;
    }
    return true;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_FIRST));
    if (warp == 0) {
      // ======================= TMA producer (one thread) =======================
      if (lane == 0 && !p.stall_producer) {
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        const uint64_t pol = ptx::make_l2_policy(2);
        const uint32_t bytes = CG * (static_cast<uint32_t>(p.a_rows) * kBlock + C::B_BYTES);
        Fp8Work w;
        auto row_of = [&]() { return w.m_tile * 128 * CG + (CG == 2 ? static_cast<int>(rank) * 128 : 0); };
        auto bar_of = [&](int st) { return CG == 2 ? ptx::mapa(full_bar(st), 0) : full_bar(st); };
        auto load_rows = [&](int kb, int st) {
          const uint32_t dst = smem_base + st * C::STAGE_BYTES;
          if constexpr (CG == 2)
            ptx::tma_load_2d_pair(dst, &p.a, bar_of(st), kb * kBlock, row_of(), pol);
          else
            ptx::tma_load_2d(dst, &p.a, full_bar(st), kb * kBlock, row_of(), pol);
        };
        auto load_weight = [&](int kb, int st) {
          const uint32_t dst = smem_base + st * C::STAGE_BYTES + C::A_BYTES;
          const int k0 = kb * kBlock, n0 = w.n_tile * (DUAL ? 128 : 256);
          if (CG == 1 || rank == 0) ptx::mbar_arrive_expect_tx(full_bar(st), bytes);
          if constexpr (CG == 2) {
            // each CTA stages one half of the tile's weight rows
            ptx::tma_load_3d_pair(dst, (DUAL && rank) ? &p.b1 : &p.b0, bar_of(st), k0,
                                  DUAL ? n0 : n0 + static_cast<int>(rank) * 128, w.expert, pol);
          } else {
            ptx::tma_load_3d(dst, &p.b0, full_bar(st), k0, n0, w.expert, pol);
            ptx::tma_load_3d(dst + 128 * kBlock, DUAL ? &p.b1 : &p.b0, full_bar(st), k0, DUAL ? n0 : n0 + 128, w.expert, pol);
          }
        };
        int ahead = 0;  // blocks of the first tile whose weight tiles are on their way
        if (early) {
          if (get_work(0, w)) {
            ahead = kb1 - kb0 < STAGES ? kb1 - kb0 : STAGES;
            for (int i = 0; i < ahead; ++i) load_weight(kb0 + i, i);
          }
          ptx::wait_predecessor();
        }
        for (int idx = 0; ok && get_work(idx, w); ++idx) {
          for (int kb = kb0; kb < kb1; ++kb) {
            if (ahead > 0) {
              --ahead;  // the pipeline is empty: stage s is kb - kb0
            } else {
              ok = bounded_wait_thread(empty_bar(s), ph ^ 1u, ctl, WAIT_PRODUCER_EMPTY);
              if (!ok) break;
              load_weight(kb, s);
            }
            load_rows(kb, s);
            if (++s == STAGES) {
              s = 0;
              ph ^= 1u;
            }
          }
        }
      }
    } else if (warp == 1) {
      // ================ MMA issuer (one thread of the pair leader) ================
      if ((CG == 1 || rank == 0) && lane == 0) {
        int s = 0, a = 0;
        uint32_t ph = 0, aph = 0;
        bool ok = true;
        auto commit = [&](uint32_t bar) {
          if (CG == 2)
            ptx::mma_commit_pair(bar, 3);
          else
            ptx::mma_commit(bar);
        };
        Fp8Work w;
        for (int idx = 0; ok && get_work(idx, w); ++idx) {
          for (int kb = kb0; kb < kb1; ++kb) {
            ok = bounded_wait_thread(full_bar(s), ph, ctl, WAIT_MMA_FULL);
            if (!ok) break;
            ok = bounded_wait_thread(tempty_bar(a), aph ^ 1u, ctl, WAIT_MMA_TMEM_EMPTY);
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const uint32_t a_addr = smem_base + s * C::STAGE_BYTES, b_addr = a_addr + C::A_BYTES;
#pragma unroll
            for (int k = 0; k < kBlock / 32; ++k)
              mma_f8_ss<CG>(tmem_base + a * 256, p.desc | (((a_addr + k * 32u) & 0x3FFFFu) >> 4),
                            p.desc | (((b_addr + k * 32u) & 0x3FFFFu) >> 4), p.idesc, k != 0 ? 1u : 0u);
            commit(tfull_bar(a));
            commit(empty_bar(s));
            a ^= 1;
            if (a == 0) aph ^= 1u;
            if (++s == STAGES) {
              s = 0;
              ph ^= 1u;
            }
          }
        }
      }
    } else if (warp == 2) {
      // ================ scales of each block's rows, for the epilogue ================
      // Slot kb % 4 is written once the MMAs of block kb - 2 are complete: they began after the
      // epilogue had finished with block kb - 4.  Global loads run kAhead blocks ahead: a load
      // asked for one block before its use cost more time than the block's MMAs.
      constexpr int kAhead = 4;
      int n = 0;  // blocks of all tiles so far
      bool ok = true;
      Fp8Work w;
      for (int idx = 0; ok && get_work(idx, w); ++idx) {
        const int row0 = w.m_tile * 128 * CG + (CG == 2 ? static_cast<int>(rank) * 128 : 0);
        const float* x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = row0 + i * 32 + lane;
          x[i] = p.xs + static_cast<int64_t>(row < p.M ? row : p.M - 1) * p.xs_row;
        }
        const int nb = DUAL ? w.n_tile : 2 * w.n_tile;
        const int64_t wbase = (static_cast<int64_t>(w.expert) * p.ws_rows + nb) * p.num_kb;
        const float* w0 = p.ws0 + wbase;
        // the second block of a tile may lie behind the weight's last
        const float* w1 = DUAL ? p.ws1 + wbase : (nb + 1 < p.ws_rows ? w0 + p.num_kb : w0);
        float xv[kAhead][4], wv[kAhead][2];
        auto fetch = [&](int kb, int i) {
          kb = kb < kb1 ? kb : kb1 - 1;
#pragma unroll
          for (int r = 0; r < 4; ++r) xv[i][r] = x[r][kb * p.xs_block];
          wv[i][0] = w0[kb];
          wv[i][1] = w1[kb];
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) fetch(kb0 + i, i);
        for (int kbase = kb0; kbase < kb1 && ok; kbase += kAhead) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            if (kbase + i < kb1 && ok) {
              // block n - 2 used the same region: its phase is the one before
              if (n >= 2) ok = bounded_wait_warp(tfull_bar(n & 1), ((n >> 1) - 1) & 1, ctl, WAIT_EPI_TMEM_FULL);
              if (ok) {
                float* slot = scale_ring + (n & 3) * 256 + lane;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  slot[r * 32] = xv[i][r] * wv[i][0];
                  slot[128 + r * 32] = xv[i][r] * wv[i][1];
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(tfull_bar(n & 1));
                ++n;
                fetch(kbase + i + kAhead, i);
              }
            }
          }
        }
      }
    }
  } else {
    // ======================= epilogue: scale, add, write =======================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_EPILOGUE));
    const int q = warp & 3, ew = warp - 4, half = ew >> 2;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    // This warp's columns: the same 64 of each half of a block's 256, so that a thread holds
    // gate and up of its columns.
    const uint32_t my_tempty = (CG == 2) ? ptx::mapa(tempty_bar(0), 0) : tempty_bar(0);
    int a = 0;
    uint32_t aph = 0;
    bool ok = true;
    int parity = 0, slot = 0;
    Fp8Work w;
    for (int idx = 0; ok && get_work(idx, w); ++idx) {
      const int tile_row = (CG == 2 ? static_cast<int>(rank) * 128 : 0) + q * 32;  // of this warp, in the tile
      const int row0 = w.m_tile * 128 * CG + tile_row;
      const bool active = tile_row < w.rows;  // no valid row here: nothing is added up or stored
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
      auto wait_block = [&]() {
        ok = bounded_wait_warp(tfull_bar(a), aph, ctl, WAIT_EPI_TMEM_FULL);
        if (ok) ptx::tc_fence_after_sync();
        return ok;
      };
      auto release = [&]() {
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2)
            ptx::mbar_arrive_cluster_relaxed(my_tempty + 8u * a);
          else
            ptx::mbar_arrive_relaxed(my_tempty + 8u * a);
        }
      };
      auto next_block = [&]() {
        a ^= 1;
        if (a == 0) aph ^= 1u;
        slot = (slot + 1) & (C::SCALE_SLOTS - 1);
      };
      if (!active) {
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          if (wait_block()) release();
          next_block();
        }
      } else if (wait_block()) {
        // eight chunks of 16 columns; the next one is on its way while one is added
        const uint32_t t0 = lane_base + half * 64;
        uint32_t r0[16], r1[16];
        for (int kb = kb0;;) {
          const uint32_t t = t0 + a * 256;
          ptx::tmem_ld_32x16(t, r0);
          const float* sc = scale_ring + slot * 256 + q * 32 + lane;
          const float s_lo = sc[0], s_hi = sc[128];
#pragma unroll
          for (int c = 0; c < 8; c += 2) {
            tmem_wait16(r0);
            ptx::tmem_ld_32x16(t + (c < 4 ? (c + 1) * 16 : 64 + (c + 1) * 16), r1);
            scaled_add16(acc + c * 16, r0, c < 4 ? s_lo : s_hi);
            tmem_wait16(r1);
            if (c < 6)
              ptx::tmem_ld_32x16(t + (c < 2 ? (c + 2) * 16 : 64 + (c + 2) * 16), r0);
            else
              release();
            scaled_add16(acc + (c + 1) * 16, r1, c < 4 ? s_lo : s_hi);
          }
          next_block();
          if (++kb == kb1 || !wait_block()) break;
        }
      }
      // The two warps of a lane quadrant meet once a tile (below).  One that gives up arrives
      // there without waiting, and none waits once the flag is up: no warp is left behind.
      if (DUAL && ok) ok = __all_sync(0xffffffffu, *abort_flag == 0u);
      if (!ok) {
        if (DUAL) asm volatile("bar.arrive %0, 64;" ::"r"(1 + q) : "memory");
        break;
      }

      if (!DUAL && p.splits > 1) {
        // Partial sums of this share, added up behind the cluster barrier.  Every MMA and load of
        // this CTA is complete: the stages are free.
        if (active && tile_row + lane < w.rows) {
          const uint32_t mine = smem_base + ((tile_row + lane) * C::PART_LD + half * 64) * 4;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            ptx::st_shared_v4(mine + ((i >> 4) * 128 + (i & 15) * 4) * 4, __float_as_uint(acc[4 * i]),
                              __float_as_uint(acc[4 * i + 1]), __float_as_uint(acc[4 * i + 2]),
                              __float_as_uint(acc[4 * i + 3]));
        }
      } else if constexpr (!DUAL) {
        // a thread holds 64 consecutive columns of its row in each half: whole sectors
        if (active && row0 + lane < p.M) {
          T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(row0 + lane) * p.N;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            store_row32<T>(dst, w.n_tile * 256 + (j >> 1) * 128 + half * 64 + (j & 1) * 32, p.N, p.wide_rows != 0, acc + j * 32);
        }
      } else {
        // h = silu(g) u in fp32; the row's block of 128 columns is shared by the two warps of
        // this lane quadrant, which exchange their largest magnitudes
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const float g = acc[i];
          acc[i] = g * sigmoid_f32(g) * acc[64 + i];
          const uint32_t m = magnitude_bits(acc[i]);
          top = top > m ? top : m;
        }
        volatile uint32_t* mine = reinterpret_cast<volatile uint32_t*>(smem_gen + amax_off) + (parity * C::EPI_WARPS) * 32;
        mine[ew * 32 + lane] = top;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
        const uint32_t other = mine[(ew ^ 4) * 32 + lane];
        parity ^= 1;
        float inv;
        const float scale = block_scale(top > other ? top : other, inv);
        if (active && row0 + lane < p.M) {
          if (half == 0) p.hs[w.n_tile * p.hs_pitch + row0 + lane] = scale;
          uint8_t* dst = p.hq + static_cast<int64_t>(row0 + lane) * p.N;
          const int col = w.n_tile * 128 + half * 64;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float* h = acc + c * 16 + i * 4;
              v[i] = to_e4m3x4(h[0] * inv, h[1] * inv, h[2] * inv, h[3] * inv);
            }
            if (col + c * 16 < p.N) ptx::st_global_v4(dst + col + c * 16, v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
  }

  // ======================= shares of one tile, teardown =======================
  __syncwarp();
  if (CG == 1 && !DUAL && p.splits > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
    Fp8Work w;
    if (warp >= 4 && get_work(0, w) && *abort_flag == 0u) {
      // This CTA adds and writes 4-column groups [g0, g1) of the tile's 64, shares in order.
      const int g0 = 64 * static_cast<int>(rank) / p.splits, g1 = 64 * (static_cast<int>(rank) + 1) / p.splits;
      const int rows = w.rows < 128 ? w.rows : 128, groups = g1 - g0;
      for (int i = threadIdx.x - 128; i < rows * groups; i += 32 * C::EPI_WARPS) {
        const int r = i / groups, g = g0 + i - r * groups;
        const uint32_t at = smem_base + (r * C::PART_LD + g * 4) * 4;
        float4 v[kMaxSplits];
#pragma unroll
        for (int c = 0; c < kMaxSplits; ++c)
          if (c < p.splits) v[c] = ld_cluster_f32x4(ptx::mapa(at, c));
        float4 sum = v[0];
#pragma unroll
        for (int c = 1; c < kMaxSplits; ++c)
          if (c < p.splits) {
            sum.x += v[c].x;
            sum.y += v[c].y;
            sum.z += v[c].z;
            sum.w += v[c].w;
          }
        const int col = w.n_tile * 256 + g * 4;
        if (col < p.N)
          *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + static_cast<int64_t>(w.m_tile * 128 + r) * p.N + col) =
              make_uint2(pack2<T>(sum.x, sum.y), pack2<T>(sum.z, sum.w));
      }
    }
    __syncwarp();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < kDrainNs) __nanosleep(1000);
  }
  if (CG == 2 || p.splits > 1) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<CG>(tmem_base, 512);
  }
}

// ------------------------------------------------------------- quantisation --
template <typename T>
__device__ __forceinline__ void load8(const T* src, float (&v)[8]) {
  const uint4 x = *reinterpret_cast<const uint4*>(src);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
}

// One token per block row; 16 lanes take the 8-element pieces of a block of 128 columns.
// With a plan the token's row goes to the rows of its k pairs.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                            float* __restrict__ scales, int64_t pitch, int d,
                                                            const ExpertPlan plan, const int* __restrict__ plan_dev) {
  ptx::allow_successor();
  ptx::wait_predecessor();
  const int64_t t = blockIdx.x;
  const int k = plan_dev != nullptr ? plan.k : 1;
  for (int c0 = (blockIdx.y * 256 + threadIdx.x) * 8; c0 - static_cast<int>(threadIdx.x & 15) * 8 < d; c0 += gridDim.y * 256 * 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (c0 < d) load8<T>(x + t * d + c0, v);
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude_bits(v[i]));
    const unsigned half_mask = 0xffffu << (threadIdx.x & 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(half_mask, top, o));
    float inv;
    const float scale = block_scale(top, inv);
    const uint2 packed = make_uint2(to_e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                                    to_e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
    for (int j = 0; j < k; ++j) {
      const int64_t row = plan_dev != nullptr ? plan_dev[plan.pair_row + t * k + j] : t;
      if (row < 0) continue;
      if (c0 < d) *reinterpret_cast<uint2*>(q + row * d + c0) = packed;
      if ((threadIdx.x & 15) == 0) scales[(c0 >> 7) * pitch + row] = scale;
    }
  }
}

// w (d_in, d_out) -> q (d_out, d_in) and a power-of-two scale per 128 x 128 block.
// One block of threads per block of the weight; runs once per weight.
template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(const T* __restrict__ w, uint8_t* __restrict__ q,
                                                              float* __restrict__ scales, int d_in, int d_out) {
  __shared__ __align__(16) uint8_t tile[128][132];
  __shared__ uint32_t tops[8];
  const int64_t e = blockIdx.z;
  const int k0 = blockIdx.x * 128, n0 = blockIdx.y * 128;
  const T* src = w + e * d_in * d_out;
  uint32_t top = 0u;
  float v[8][8];
  const int piece = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int kk = k0 + i * 16 + (threadIdx.x >> 4), n = n0 + piece * 8;
#pragma unroll
    for (int c = 0; c < 8; ++c) v[i][c] = 0.0f;
    if (kk < d_in && n < d_out) load8<T>(src + static_cast<int64_t>(kk) * d_out + n, v[i]);
#pragma unroll
    for (int c = 0; c < 8; ++c) top = max(top, magnitude_bits(v[i][c]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, tops[i]);
  float inv;
  const float scale = block_scale(top, inv);
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int c = 0; c < 8; c += 4) {
      const uint32_t b = to_e4m3x4(v[i][c] * inv, v[i][c + 1] * inv, v[i][c + 2] * inv, v[i][c + 3] * inv);
#pragma unroll
      for (int j = 0; j < 4; ++j) tile[piece * 8 + c + j][i * 16 + (threadIdx.x >> 4)] = static_cast<uint8_t>(b >> (8 * j));
    }
  if (threadIdx.x == 0) scales[(e * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = scale;
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * 32; i += 256) {
    const int n = i >> 5, kk = (i & 31) * 4;
    if (n0 + n < d_out && k0 + kk < d_in)
      *reinterpret_cast<uint32_t*>(q + (e * d_out + n0 + n) * static_cast<int64_t>(d_in) + k0 + kk) =
          *reinterpret_cast<const uint32_t*>(&tile[n][kk]);
  }
}

// ------------------------------------------------------------------ launches --
template <int CG, bool DUAL, typename T>
int launch_fp8_one(const Fp8Params& p, int grid, bool dependent, cudaStream_t st) {
  static std::atomic<uint64_t> prepared{0};
  int dev = 0;
  FSW_CUDA(cudaGetDevice(&dev));
  if (!(prepared.load() >> (dev & 63) & 1)) {
    FSW_CUDA(cudaFuncSetAttribute(fp8_gemm_kernel<CG, DUAL, T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  Fp8Cfg<CG>::SMEM_BYTES));
    // The warpgroups trade registers within what the block is launched with; a build that
    // launches with fewer would leave the epilogue waiting for its share.
    cudaFuncAttributes attr;
    FSW_CUDA(cudaFuncGetAttributes(&attr, fp8_gemm_kernel<CG, DUAL, T>));
    if (attr.numRegs * Fp8Cfg<CG>::THREADS < Fp8Cfg<CG>::REGS_FIRST * 128 + Fp8Cfg<CG>::REGS_EPILOGUE * 32 * Fp8Cfg<CG>::EPI_WARPS)
      return fail(FSW_EUNAVAILABLE, "the 8-bit kernel was built with %d registers a thread", attr.numRegs);
    prepared.fetch_or(1ull << (dev & 63));
  }
  FSW_CUDA(launch_dependent(fp8_gemm_kernel<CG, DUAL, T>, dim3(grid), Fp8Cfg<CG>::THREADS, Fp8Cfg<CG>::SMEM_BYTES, st,
                            dependent, CG * p.splits, p));
  return FSW_OK;
}

// How many clusters of c single-CTA tiles can be resident at once on the current device.
int resident_clusters(int c, int* fit) {
  static std::atomic<int> known[64][kMaxSplits + 1];  // value + 1; 0 = not asked yet
  int dev = 0;
  FSW_CUDA(cudaGetDevice(&dev));
  std::atomic<int>& slot = known[dev & 63][c];
  int v = slot.load();
  if (v == 0) {
    FSW_CUDA(cudaFuncSetAttribute(fp8_gemm_kernel<1, false, __nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  Fp8Cfg<1>::SMEM_BYTES));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c * 256, 1, 1);
    cfg.blockDim = dim3(Fp8Cfg<1>::THREADS, 1, 1);
    cfg.dynamicSmemBytes = Fp8Cfg<1>::SMEM_BYTES;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, fp8_gemm_kernel<1, false, __nv_bfloat16>, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    v = n + 1;
    slot.store(v);
  }
  *fit = v - 1;
  return FSW_OK;
}

// The rows an 8-bit product works on: T dense rows, or a plan's.
struct Fp8Rows {
  int64_t rows;                 // of the arrays
  int64_t most;                 // most rows a weight can have
  const ExpertPlan* plan;       // nullptr: dense
  const int* plan_dev;
};

// out (rows, N) = x @ w^T, or with w1 hq, hs = quantised silu(x w^T) * (x w1^T).
int run_fp8(const Fp8Rows& r, const void* xq, const float* xs, int64_t xs_row, int64_t xs_block, const void* w,
            const float* ws, const void* w1, const float* ws1, void* out, uint8_t* hq, float* hs, int64_t K, int64_t N,
            int dtype, DeviceInfo* d, cudaStream_t st, bool dependent = true) {
  const bool dual = w1 != nullptr;
  const int E = r.plan != nullptr ? r.plan->E : 1;
  const int tile_n = dual ? 128 : 256;
  Fp8Params p;
  memset(&p, 0, sizeof(p));
  p.num_kb = (int)((K + kBlock - 1) / kBlock);
  p.num_n_tiles = (int)((N + tile_n - 1) / tile_n);
  p.ws_rows = (int)((N + kBlock - 1) / kBlock);
  // Pairs of CTAs halve the operand traffic of a tile; a single CTA's tile fits fewer rows.
  int cg;
  if (r.plan != nullptr)
    cg = r.plan->tile_rows / 128;
  else
    cg = (r.rows + 255) / 256 * p.num_n_tiles >= d->max_pairs / 2 && r.rows > 128 ? 2 : 1;
  p.num_m_tiles = r.plan != nullptr ? r.plan->tiles : (int)((r.rows + 128 * cg - 1) / (128 * cg));
  const long long tiles = (long long)p.num_m_tiles * p.num_n_tiles;
  if (tiles >= (1ll << 30)) return fail(FSW_EINVAL, "too many tiles");
  p.splits = 1;
  if (cg == 1 && !dual && r.plan == nullptr) {
    // Fewer tiles than SMs: divide their K blocks, at least 4 a share, over as many CTAs as
    // leave all clusters resident at once (a GPC holds whole clusters only: of 8 CTAs 16 fit,
    // not 148 / 8, and a 17th cluster would double the time).
    for (int c = kMaxSplits; c > 1; --c) {
      if (p.num_kb < 4 * c || tiles * c > d->sm_count) continue;
      int fit = 0;
      const int rc = resident_clusters(c, &fit);
      if (rc != FSW_OK) return rc;
      if (tiles <= fit) {
        p.splits = c;
        break;
      }
    }
  }
  p.a_rows = r.most > 120 ? 128 : (int)((r.most + 7) / 8 * 8);
  if (cg == 2) p.a_rows = 128;
  int rc;
  if ((rc = make_map(&p.a, xq, 0, K, r.rows, p.a_rows, "x", 128, 0, 0, 1)) != FSW_OK) return rc;
  if ((rc = make_map(&p.b0, w, 0, K, N, 128, "weight", 128, 0, E, 1)) != FSW_OK) return rc;
  p.b1 = p.b0;
  if (dual && (rc = make_map(&p.b1, w1, 0, K, N, 128, "w_up", 128, 0, E, 1)) != FSW_OK) return rc;
  uint32_t kadv;
  fill_operand_desc(MAJOR_K, &p.desc, &kadv);
  // kind::f8f6f4: fp32 sums (bit 4), e4m3 operands (0), both K-major
  p.idesc = (1u << 4) | (256u >> 3 << 17) | (static_cast<uint32_t>(128 * cg) >> 4 << 24);
  p.xs = xs;
  p.xs_row = xs_row;
  p.xs_block = xs_block;
  p.ws0 = ws;
  p.ws1 = ws1;
  p.M = (int)r.rows;
  p.N = (int)N;
  p.out = out;
  p.wide_rows = (N & 15) == 0 && (reinterpret_cast<uintptr_t>(out) & 31u) == 0;
  p.hq = hq;
  p.hs = hs;
  p.hs_pitch = r.rows;
  if (r.plan != nullptr) {
    p.grp_meta = r.plan_dev;
    p.grp_counts = r.plan_dev + r.plan->counts;
    p.grp_offsets = r.plan_dev + r.plan->offsets;
    p.grp_tile_expert = r.plan_dev + r.plan->tile_expert;
  }
  p.status = d->status;
  p.wait_limit_ns = (unsigned long long)opt_wait_limit_ms() * 1000000ull;
  p.stall_producer = (int)opt_stall_producer();
  p.group_m = p.num_m_tiles < 8 ? p.num_m_tiles : 8;
  const long long workers = cg == 2 ? d->max_pairs : d->sm_count;
  const int grid = (int)(p.splits > 1 ? tiles * p.splits : (tiles < workers ? tiles : workers) * cg);
  const bool bf = dtype == FSW_BF16;
  if (cg == 2) {
    if (dual) return launch_fp8_one<2, true, __nv_bfloat16>(p, grid, dependent, st);
    return bf ? launch_fp8_one<2, false, __nv_bfloat16>(p, grid, dependent, st) : launch_fp8_one<2, false, __half>(p, grid, dependent, st);
  }
  if (dual) return launch_fp8_one<1, true, __nv_bfloat16>(p, grid, dependent, st);
  return bf ? launch_fp8_one<1, false, __nv_bfloat16>(p, grid, dependent, st) : launch_fp8_one<1, false, __half>(p, grid, dependent, st);
}

int quantize_rows(const void* x, void* q, float* scales, int64_t pitch, int64_t T, int64_t d, int dtype,
                  const ExpertPlan* plan, const int* plan_dev, cudaStream_t st) {
  ExpertPlan none = {};
  // a block covers 2048 columns; few tokens are spread over more blocks
  const dim3 grid((unsigned)T, (unsigned)(T >= 1024 ? 1 : (d + 2047) / 2048));
  const ExpertPlan pl = plan ? *plan : none;
  if (dtype == FSW_BF16)
    FSW_CUDA(launch_dependent(quantize_rows_kernel<__nv_bfloat16>, grid, 256, 0, st, plan != nullptr, 1,
                              static_cast<const __nv_bfloat16*>(x), static_cast<uint8_t*>(q), scales, pitch, (int)d, pl,
                              plan_dev));
  else
    FSW_CUDA(launch_dependent(quantize_rows_kernel<__half>, grid, 256, 0, st, plan != nullptr, 1,
                              static_cast<const __half*>(x), static_cast<uint8_t*>(q), scales, pitch, (int)d, pl, plan_dev));
  return FSW_OK;
}

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
int64_t blocks_of(int64_t v) { return (v + kBlock - 1) / kBlock; }

int check_fp8(int64_t T, int64_t K, int64_t N, int dtype) {
  if (dtype != FSW_BF16 && dtype != FSW_FP16) return fail(FSW_EINVAL, "unknown dtype %d", dtype);
  if (T < 0 || T >= (1ll << 31) - 256) return fail(FSW_EINVAL, "bad number of rows %lld", (long long)T);
  if (K <= 0 || N <= 0 || K >= (1 << 24) || N >= (1 << 24))
    return fail(FSW_EINVAL, "bad feature sizes %lld, %lld", (long long)K, (long long)N);
  if ((K & 15) || (N & 7))
    return fail(FSW_EINVAL, "the inner size %lld must be a multiple of 16 and the outer size %lld of 8", (long long)K, (long long)N);
  return FSW_OK;
}

}  // namespace
}  // namespace fsw

using namespace fsw;

extern "C" {

int fsw_fp8_quantize_rows(const void* x, void* q, void* scales, int64_t T, int64_t d, int dtype, void* stream) {
  int rc = check_fp8(T, d, 8, dtype);
  if (rc != FSW_OK) return rc;
  if (T == 0) return FSW_OK;
  if (!x || !q || !scales) return fail(FSW_EINVAL, "NULL pointer");
  if (!aligned16(x) || !aligned16(q)) return fail(FSW_EINVAL, "pointers must be 16-byte aligned");
  DeviceInfo* dev = nullptr;
  if ((rc = ensure_device(&dev)) != FSW_OK) return rc;
  return quantize_rows(x, q, static_cast<float*>(scales), T, T, d, dtype, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

int fsw_fp8_quantize_weight(const void* w, void* q, void* scales, int E, int64_t d_in, int64_t d_out, int dtype, void* stream) {
  int rc = check_fp8(1, d_in, d_out, dtype);
  if (rc != FSW_OK) return rc;
  if (E < 1 || E > FSW_MAX_EXPERTS || blocks_of(d_out) > 65535) return fail(FSW_EINVAL, "bad number of weights %d or size", E);
  if (!w || !q || !scales) return fail(FSW_EINVAL, "NULL pointer");
  if (!aligned16(w) || !aligned16(q)) return fail(FSW_EINVAL, "pointers must be 16-byte aligned");
  DeviceInfo* dev = nullptr;
  if ((rc = ensure_device(&dev)) != FSW_OK) return rc;
  const dim3 grid((unsigned)blocks_of(d_in), (unsigned)blocks_of(d_out), (unsigned)E);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ++g_kernel_launches;
  if (dtype == FSW_BF16)
    quantize_weight_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(w), static_cast<uint8_t*>(q),
                                                                static_cast<float*>(scales), (int)d_in, (int)d_out);
  else
    quantize_weight_kernel<__half><<<grid, 256, 0, st>>>(static_cast<const __half*>(w), static_cast<uint8_t*>(q),
                                                         static_cast<float*>(scales), (int)d_in, (int)d_out);
  FSW_CUDA(cudaGetLastError());
  return FSW_OK;
}

int fsw_fp8_gemm(const void* xq, const void* xs, int64_t xs_row_stride, int64_t xs_block_stride, const void* w,
                 const void* ws, void* y, int64_t T, int64_t K, int64_t N, int dtype, void* stream) {
  int rc = check_fp8(T, K, N, dtype);
  if (rc != FSW_OK) return rc;
  if (xs_row_stride < 0 || xs_block_stride < 0) return fail(FSW_EINVAL, "negative stride of the scales");
  if (T == 0) return FSW_OK;
  if (!xq || !xs || !w || !ws || !y) return fail(FSW_EINVAL, "NULL pointer");
  if (!aligned16(xq) || !aligned16(w) || !aligned16(y)) return fail(FSW_EINVAL, "pointers must be 16-byte aligned");
  DeviceInfo* dev = nullptr;
  if ((rc = ensure_device(&dev)) != FSW_OK) return rc;
  const Fp8Rows r = {T, T, nullptr, nullptr};
  return run_fp8(r, xq, static_cast<const float*>(xs), xs_row_stride, xs_block_stride, w, static_cast<const float*>(ws),
                 nullptr, nullptr, y, nullptr, nullptr, K, N, dtype, dev, static_cast<cudaStream_t>(stream), false);
}

int64_t fsw_fp8_linear_scratch_bytes(int64_t T, int64_t K) {
  int rc = check_fp8(T, K, 8, FSW_BF16);
  if (rc != FSW_OK) return rc;
  return align256(T * K) + align256(T * blocks_of(K) * 4);
}

int fsw_fp8_linear(const void* x, const void* w, const void* ws, void* y, void* scratch, int64_t scratch_bytes, int64_t T,
                   int64_t K, int64_t N, int dtype, void* stream) {
  int rc = check_fp8(T, K, N, dtype);
  if (rc != FSW_OK) return rc;
  if (T == 0) return FSW_OK;
  if (!x || !w || !ws || !y || !scratch) return fail(FSW_EINVAL, "NULL pointer");
  if (!aligned16(x) || !aligned16(w) || !aligned16(y) || !aligned16(scratch))
    return fail(FSW_EINVAL, "pointers must be 16-byte aligned");
  if (scratch_bytes < fsw_fp8_linear_scratch_bytes(T, K)) return fail(FSW_EINVAL, "scratch of %lld bytes is too small", (long long)scratch_bytes);
  DeviceInfo* dev = nullptr;
  if ((rc = ensure_device(&dev)) != FSW_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* xq = static_cast<uint8_t*>(scratch);
  float* xs = reinterpret_cast<float*>(xq + align256(T * K));
  if ((rc = quantize_rows(x, xq, xs, T, T, K, dtype, nullptr, nullptr, st)) != FSW_OK) return rc;
  const Fp8Rows r = {T, T, nullptr, nullptr};
  return run_fp8(r, xq, xs, 1, T, w, static_cast<const float*>(ws), nullptr, nullptr, y, nullptr, nullptr, K, N, dtype, dev, st);
}

// Scratch: [plan] xq xs hq hs [ys], for T rows (dense) or the plan's.
struct Fp8MlpBuffers {
  int64_t xq, xs, hq, hs, ys, bytes;
};
static Fp8MlpBuffers fp8_mlp_buffers(int64_t plan_bytes, int64_t rows, int64_t d, int64_t f, int64_t ys_cols) {
  Fp8MlpBuffers b;
  b.xq = align256(plan_bytes);
  b.xs = b.xq + align256(rows * d);
  b.hq = b.xs + align256(rows * blocks_of(d) * 4);
  b.hs = b.hq + align256(rows * f);
  b.ys = b.hs + align256(rows * blocks_of(f) * 4);
  b.bytes = b.ys + align256(rows * ys_cols * 2);
  return b;
}

static int check_fp8_mlp(int64_t T, int64_t d, int64_t f, int64_t d_out, int dtype) {
  int rc = check_fp8(T, d, f, dtype);
  return rc != FSW_OK ? rc : check_fp8(T, f, d_out, dtype);
}

int64_t fsw_fp8_mlp_scratch_bytes(int64_t T, int64_t d, int64_t f) {
  int rc = check_fp8_mlp(T, d, f, 8, FSW_BF16);
  if (rc != FSW_OK) return rc;
  return fp8_mlp_buffers(0, T, d, f, 0).bytes;
}

int fsw_fp8_mlp(const void* x, const void* w_gate, const void* s_gate, const void* w_up, const void* s_up,
                const void* w_down, const void* s_down, void* y, void* scratch, int64_t scratch_bytes, int64_t T, int64_t d,
                int64_t f, int64_t d_out, int dtype, void* stream) {
  int rc = check_fp8_mlp(T, d, f, d_out, dtype);
  if (rc != FSW_OK) return rc;
  if (T == 0) return FSW_OK;
  if (!x || !w_gate || !s_gate || !w_up || !s_up || !w_down || !s_down || !y || !scratch) return fail(FSW_EINVAL, "NULL pointer");
  if (!aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(w_down) || !aligned16(y) || !aligned16(scratch))
    return fail(FSW_EINVAL, "pointers must be 16-byte aligned");
  const Fp8MlpBuffers b = fp8_mlp_buffers(0, T, d, f, 0);
  if (scratch_bytes < b.bytes) return fail(FSW_EINVAL, "scratch of %lld bytes is too small", (long long)scratch_bytes);
  DeviceInfo* dev = nullptr;
  if ((rc = ensure_device(&dev)) != FSW_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* s = static_cast<char*>(scratch);
  float *xs = reinterpret_cast<float*>(s + b.xs), *hs = reinterpret_cast<float*>(s + b.hs);
  uint8_t* hq = reinterpret_cast<uint8_t*>(s + b.hq);
  if ((rc = quantize_rows(x, s + b.xq, xs, T, T, d, dtype, nullptr, nullptr, st)) != FSW_OK) return rc;
  const Fp8Rows r = {T, T, nullptr, nullptr};
  if ((rc = run_fp8(r, s + b.xq, xs, 1, T, w_gate, static_cast<const float*>(s_gate), w_up, static_cast<const float*>(s_up),
                    nullptr, hq, hs, d, f, dtype, dev, st)) != FSW_OK)
    return rc;
  return run_fp8(r, hq, hs, 1, T, w_down, static_cast<const float*>(s_down), nullptr, nullptr, y, nullptr, nullptr, f, d_out,
                 dtype, dev, st);
}

static int check_fp8_experts(int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out, int dtype, int wtype, ExpertPlan* plan) {
  int rc = check_experts(T, k, E, d, f, d_out, dtype, wtype);
  if (rc == FSW_OK) rc = check_fp8_mlp(T, d, f, d_out, dtype);
  if (rc != FSW_OK) return rc;
  if (!make_plan(plan, T, k, E, choose_tile_rows(T * k, E))) return fail(FSW_EINVAL, "too many tokens");
  return FSW_OK;
}

int64_t fsw_fp8_experts_scratch_bytes(int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out) {
  ExpertPlan plan;
  int rc = check_fp8_experts(T, k, E, d, f, d_out, FSW_BF16, FSW_FP32, &plan);
  if (rc != FSW_OK) return rc;
  return fp8_mlp_buffers(plan.ints * 4, plan.rows, d, f, d_out).bytes;
}

int fsw_fp8_experts_forward(const void* x, const void* weights, const void* indices, const void* w_gate,
                            const void* s_gate, const void* w_up, const void* s_up, const void* w_down,
                            const void* s_down, void* y, void* scratch, int64_t scratch_bytes, int64_t T, int k, int E,
                            int64_t d, int64_t f, int64_t d_out, int dtype, int weights_dtype, void* stream) {
  ExpertPlan plan;
  int rc = check_fp8_experts(T, k, E, d, f, d_out, dtype, weights_dtype, &plan);
  if (rc != FSW_OK) return rc;
  if (T == 0) return FSW_OK;
  if (!x || !weights || !indices || !w_gate || !s_gate || !w_up || !s_up || !w_down || !s_down || !y || !scratch)
    return fail(FSW_EINVAL, "NULL pointer");
  if (!aligned16(x) || !aligned16(w_gate) || !aligned16(w_up) || !aligned16(w_down) || !aligned16(y) || !aligned16(scratch))
    return fail(FSW_EINVAL, "pointers must be 16-byte aligned");
  const Fp8MlpBuffers b = fp8_mlp_buffers(plan.ints * 4, plan.rows, d, f, d_out);
  if (scratch_bytes < b.bytes) return fail(FSW_EINVAL, "scratch of %lld bytes is too small", (long long)scratch_bytes);
  DeviceInfo* dev = nullptr;
  if ((rc = ensure_device(&dev)) != FSW_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* s = static_cast<char*>(scratch);
  int* plan_dev = reinterpret_cast<int*>(s);
  float *xs = reinterpret_cast<float*>(s + b.xs), *hs = reinterpret_cast<float*>(s + b.hs);
  uint8_t* hq = reinterpret_cast<uint8_t*>(s + b.hq);
  const int64_t R = plan.rows;
  if ((rc = build_plan(plan, static_cast<const int*>(indices), plan_dev, st)) != FSW_OK) return rc;
  if ((rc = quantize_rows(x, s + b.xq, xs, R, T, d, dtype, &plan, plan_dev, st)) != FSW_OK) return rc;
  const Fp8Rows r = {R, plan.pairs, &plan, plan_dev};
  if ((rc = run_fp8(r, s + b.xq, xs, 1, R, w_gate, static_cast<const float*>(s_gate), w_up, static_cast<const float*>(s_up),
                    nullptr, hq, hs, d, f, dtype, dev, st)) != FSW_OK)
    return rc;
  if ((rc = run_fp8(r, hq, hs, 1, R, w_down, static_cast<const float*>(s_down), nullptr, nullptr, s + b.ys, nullptr, nullptr, f,
                    d_out, dtype, dev, st)) != FSW_OK)
    return rc;
  return combine_rows(plan, plan_dev, s + b.ys, false, weights, weights_dtype, y, d_out, dtype, st);
}

}  // extern "C"
