// msda_norm.cuh -- group norm with an affine map and an activation over the
// levels of a channels-last feature pyramid, forward and backward.
//
// A segment is one level l of one batch entry b: rows_l rows of C channels in
// G groups of cg = C / G.  With n = rows_l * cg and sums over a segment's
// group,
//   mu = sum x / n,  var = sum (x - mu)^2 / n,  r = 1 / sqrt(var + eps)
//   h = (x - mu) r,  z = h w_c + d_c,  y = act(z)
// and, with dz = gy act'(z) and the per-channel sums s1_c = sum dz and
// s2_c = sum dz h over a segment's rows,
//   gx = r (dz w_c - a - h q),  a = sum_c w_c s1_c / n,  q = sum_c w_c s2_c / n
//   gw_c = sum_b s2_c,  gd_c = sum_b s1_c.
//
// Work is cut into units, slabs of whole groups of a segment, and units into
// tiles of rows, a CTA each.  A first launch takes the tiles' statistics, a
// second applies them, from the last tile back: what the first read last is
// then still in L2.
//
// A forward whose segments are small takes one launch instead: a CTA keeps a
// unit's rows in registers from the statistics to the application.
//
// Tiles leave partial results.  Where a unit has few tiles, each CTA of the
// second launch joins those of its groups itself ("direct"): that costs 1 us at
// its start, and neither counters nor a wait.  Else the CTA that finishes a
// group of kNormFan tiles last joins them, and the last of those groups the
// unit's.  Both go in tile order whichever CTA is last, so results
// do not depend on the schedule.  Statistics are carried in fp32 as (count,
// mean, sum of squared deviations): each thread takes the mean and deviations
// of a chunk of rows in registers, chunks and threads are joined pairwise (Chan,
// Golub, LeVeque), and tiles by what their means lie off the first tile's.  So
// a mean far from zero costs no digits but those of its own last place, and
// elements that are all the same have that value as their mean.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "msda_common.cuh"

namespace msda {

constexpr int kNormThreads = 256;
constexpr int kNormMaxSlab = 256;  // channels of a slab of several groups
constexpr int kNormFan = 32;       // tiles whose results are joined at a time

struct NormLevel {
  const char* x;       // first row of batch entry 0
  char* out;           // y, or gx in the backward
  const char* gy;      // backward only
  int64_t x_batch, x_row, out_batch, out_row, gy_batch, gy_row;  // strides in elements
  int64_t rows;
  int32_t tile0;       // first tile of the level, counted over all levels
  int32_t done0;       // first of the level's counters: per unit one, and one per kNormFan tiles
  int32_t tiles;       // tiles per unit
  int32_t tile_rows;
  int32_t slabs;       // slabs per segment
  int32_t slab_groups; // groups per slab; the last may have fewer
};

struct NormArgs {
  NormLevel lv[kMaxLevels];
  int32_t L, C, G, cg;
  float eps;
  const void* weight;  // (C) or (L, C) of the affine dtype, or nullptr: ones
  const void* bias;    // likewise, or nullptr: zeros
  int32_t affine_dtype, affine_level;  // affine_level: elements between levels' maps, 0 if shared
  float2* stats;       // (B, L, G): mean, 1 / sqrt(var + eps)
  float2* partial;     // per tile: per group of the slab (mean, sum of squared deviations);
                       // backward: per channel of the slab (s1, s2)
  int32_t partial_stride;
  int32_t direct;
  unsigned int* done;  // counters of partial results that are written (not direct)
  float2* chan;        // backward, (B, L, C): s1, s2 (not direct)
  float2* coef;        // backward, (B, L, G): a, q (not direct)
  float2* weighted;    // backward, per tile and group of the slab: sum w s1, sum w s2 (direct)
  int32_t tiles;
  // gradients of the affine map, by the second launch's first CTAs
  int32_t B, param_ctas;
  void* gweight;       // as weight, or nullptr
  void* gbias;
};

// Forward of segments that a CTA holds in registers: threads, and vectors of each.
constexpr int kNormOnceThreads = 512, kNormOnceVectors = 8;

constexpr int kNormParamChannels = 8;  // of a CTA that sums gradients of the affine map

// Both launches, or (once) the one of units that are one tile each, with
// vectors of vb bytes (mixed: 16, of several groups); one instance per dtype
// (msda_norm_{f32,f16,bf16}.cu).
template <typename T>
cudaError_t norm_launch(const NormArgs& a, int vb, bool mixed, int act, bool backward, bool once,
                        cudaStream_t st);

}  // namespace msda
