// Layout of the rows of a mixture of experts, shared by the 16-bit and the 8-bit products.
//
// The T*k (token, expert) pairs are sorted by expert, stably, and every expert's rows start
// at a multiple of `tile_rows`, so that a tile of the GEMM kernels has one expert and none
// is cut by a boundary.  The host knows only the bound `rows` on their number; the kernels
// read the rest from the plan, an int32 array in device memory:
//   meta[8]            [0] row tiles in use, [1] rows in use (padding included)
//   counts[E]          rows of each expert (without padding)
//   offsets[E + 1]     first row of each expert
//   tile_expert[tiles] expert of each row tile
//   pair_row[T*k]      row of each pair, -1 for an index outside [0, E)
//   row_pair[rows]     pair of each row, -1 for padding
//   block_hist         scratch of the sort
#pragma once

#include "fsw_host.h"

namespace fsw {

constexpr int kPlanWarpPairs = 128;  // pairs one warp of a sorting block takes, 32 at a time

struct ExpertPlan {
  int T, k, E, tile_rows;
  int pairs, tiles, rows, blocks;
  int warps;  // of a sorting block: 32, or 8 where 32 histograms of E counters would not fit 48 KB
  // offsets into the plan, in ints
  int64_t counts, offsets, tile_expert, pair_row, row_pair, block_hist, ints;
};

// Fills `p`; false if the rows do not fit 31 bits.
inline bool make_plan(ExpertPlan* p, int64_t T, int k, int E, int tile_rows) {
  const int64_t pairs = T * k;
  const int64_t used = pairs < E ? pairs : E;
  const int64_t tiles = (pairs + used * (tile_rows - 1)) / tile_rows;
  if (pairs >= (1ll << 31) - 8192 || tiles * tile_rows >= (1ll << 31) - 1024) return false;
  p->T = (int)T;
  p->k = k;
  p->E = E;
  p->tile_rows = tile_rows;
  p->pairs = (int)pairs;
  p->tiles = (int)tiles;
  p->rows = (int)(tiles * tile_rows);
  p->warps = E <= 352 ? 32 : 8;
  p->blocks = (int)((pairs + p->warps * kPlanWarpPairs - 1) / (p->warps * kPlanWarpPairs));
  p->counts = 8;
  p->offsets = p->counts + E;
  p->tile_expert = p->offsets + E + 1;
  p->pair_row = p->tile_expert + tiles;
  p->row_pair = p->pair_row + pairs;
  p->block_hist = p->row_pair + p->rows;
  p->ints = p->block_hist + (int64_t)p->blocks * E;
  return true;
}

// Height of a row tile: 256 rows (a CTA pair) if an expert has enough rows on average to
// fill such tiles, else 128.
inline int choose_tile_rows(int64_t pairs, int E) { return pairs >= 256ll * E ? 256 : 128; }

// Sorts the pairs (launches on `st`).
int build_plan(const ExpertPlan& p, const int* indices, int* plan, cudaStream_t st);

// dst[row] = src[token of row] for 16-byte multiples of `row_bytes`; optionally zeros the padding.
int gather_rows(const ExpertPlan& p, const int* plan, const void* src, void* dst, int64_t row_bytes,
                bool zero_padding, bool dependent, cudaStream_t st);

// y[t] = sum over j of weight[t, j] * src[row of (t, j)], in fp32, rounded once.
// src: of type dtype or, with src_f32, fp32.  weights: nullptr for 1, else of type wtype (FSW_FP32 or dtype).
int combine_rows(const ExpertPlan& p, const int* plan, const void* src, bool src_f32, const void* weights, int wtype, void* y,
                 int64_t cols, int dtype, cudaStream_t st);

// The forward for a handful of tokens without the sort and the matrix kernels (fsw_few.cu);
// h: T * k * f floats of scratch.
bool few_rows_apply(int64_t T, int k, int64_t d, int64_t f, int sms);
int experts_few_rows(const void* x, const void* weights, int wtype, const int* indices, const void* w_gate, const void* w_up,
                     const void* w_down, void* y, float* h, int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out,
                     int dtype, DeviceInfo* dev, cudaStream_t st);

int check_experts(int64_t T, int k, int E, int64_t d, int64_t f, int64_t d_out, int dtype, int wtype);

}  // namespace fsw
