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
// Work is cut into units: a segment, or a slab of whole groups of it, in tiles
// of rows, a CTA each.  A statistics pass and an application pass run over
// each unit; the CTA that finishes a unit's statistics last joins its tiles'
// partial results, in tile order whichever CTA it is, so results do not
// depend on the schedule.  Both passes are limited by memory (about 6 flops a
// byte in 16 bits), so units go in waves that fit in L2, and one launch holds
// the application of a wave and the statistics of the next: the application
// reads the rows that the statistics brought in.
//
// Statistics are carried in fp32 as (count, mean, sum of squared deviations):
// each thread takes the mean and deviations of a chunk of rows in registers,
// and chunks, threads and tiles are joined pairwise (Chan, Golub, LeVeque), so
// a mean far from zero costs no digits.
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
  int64_t block0;      // first tile of the level, counted over all levels
  int32_t done0;       // first of the level's counters: per unit one, and one per kNormFan tiles
  int32_t tiles;       // tiles per unit
  int32_t tile_rows;
  int32_t slabs;       // slabs per segment
  int32_t slab_groups; // groups per slab; the last may have fewer
  int32_t run;         // slabs of a segment that go together, tile by tile
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
  unsigned int* done;  // counters of partial results that are written
  float2* chan;        // backward, (B, L, C): s1, s2
  float2* coef;        // backward, (B, L, G): a, q
};

// Tiles [apply0, apply0 + applies) of one wave, [stats0, stats0 + stats) of the next.
struct NormWave {
  int64_t apply0, stats0;
  int32_t applies, stats;
  int32_t order;
};

struct NormParamGrad {
  const float2* chan;
  int32_t B, L, C;
  int32_t per_level;
  int32_t dtype;
  void* gweight;  // (C) or (L, C), or nullptr
  void* gbias;
};

cudaError_t norm_wave(const NormArgs& a, const NormWave& w, int dtype, int vb, int act,
                      bool backward, cudaStream_t st);
cudaError_t norm_param_grad(const NormParamGrad& p, cudaStream_t st);

// One instance per dtype (msda_norm_{f32,f16,bf16}.cu).
template <typename T>
cudaError_t norm_wave_t(const NormArgs& a, const NormWave& w, int vb, int act, bool backward,
                        cudaStream_t st);

}  // namespace msda
