// msda_norm_kernels.cuh -- device code of msda_norm.cuh's passes.
#pragma once

#include "msda_b200.h"
#include "msda_norm.cuh"

namespace msda {

__device__ __forceinline__ float norm_param(const void* p, int dtype, int64_t i, float none) {
  if (p == nullptr) return none;
  if (dtype == MSDA_FLOAT32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == MSDA_FLOAT16) return __half2float(__ldg(static_cast<const __half*>(p) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
}

// act(z); dact: act'(z).  A NaN stays one.
template <int ACT> __device__ __forceinline__ float norm_act(float z) {
  if (ACT == MSDA_ACT_RELU) return z < 0.f ? 0.f : z;
  if (ACT == MSDA_ACT_SILU) return z / (1.f + __expf(-z));
  if (ACT == MSDA_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678f));
  return z;
}
template <int ACT> __device__ __forceinline__ float norm_dact(float z) {
  if (ACT == MSDA_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
  if (ACT == MSDA_ACT_SILU) {
    const float s = 1.f / (1.f + __expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  if (ACT == MSDA_ACT_GELU)
    return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * __expf(-0.5f * z * z);
  return 1.f;
}

// (n, mean, m2) joined with another set's.
__device__ __forceinline__ void norm_join(float& n, float& mean, float& m2, float nb, float mb,
                                          float sb) {
  if (nb == 0.f) return;
  if (n == 0.f) {
    n = nb;
    mean = mb;
    m2 = sb;
    return;
  }
  const float nn = n + nb, d = mb - mean, f = nb / nn;
  mean += d * f;
  m2 += sb + d * d * n * f;
  n = nn;
}

// Where a tile lies, and which of its vectors a thread takes: column tc (then
// tc + tcols, ... where one group is wider than the CTA), rows tr, tr + trows, ...
template <int EPV> struct NormTile {
  int l, unit, tile, groups, nvc, tcols, trows, tc, tr, rows, g0;
  int64_t b, row0;
  __device__ __forceinline__ NormTile(const NormArgs& a, int64_t block) {
    l = a.L - 1;
    while (block < a.lv[l].block0) --l;
    const NormLevel& v = a.lv[l];
    const int64_t rel = block - v.block0;
    const int u = static_cast<int>(rel / v.tiles);
    tile = static_cast<int>(rel - static_cast<int64_t>(u) * v.tiles);
    unit = v.unit0 + u;
    b = u / v.slabs;
    g0 = (u % v.slabs) * v.slab_groups;
    groups = min(v.slab_groups, a.G - g0);
    row0 = static_cast<int64_t>(tile) * v.tile_rows;
    rows = static_cast<int>(min(static_cast<int64_t>(v.tile_rows), v.rows - row0));
    nvc = groups * a.cg / EPV;
    tcols = min(nvc, kNormThreads);
    trows = kNormThreads / tcols;
    tr = threadIdx.x / tcols;
    tc = threadIdx.x - tr * tcols;
    if (tr >= trows) tr = rows;  // no rows
  }
  __device__ __forceinline__ int64_t segment(const NormArgs& a) const { return b * a.L + l; }
};

// Whether this CTA is the unit's last: every tile's partial results are then visible.
__device__ __forceinline__ bool norm_last(const NormArgs& a, int unit, int tiles) {
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0)
    last = atomicAdd(&a.done[unit], 1u) == static_cast<unsigned int>(tiles - 1);
  __syncthreads();
  __threadfence();
  return last != 0;
}

template <typename T, int VB, int U>
__device__ void norm_stats(const NormArgs& a, int64_t block) {
  constexpr int EPV = Chunk<T, VB>::EPV;
  __shared__ float3 part[kNormThreads];
  const NormTile<EPV> t(a, block);
  const NormLevel& v = a.lv[t.l];
  const T* x = reinterpret_cast<const T*>(v.x) + t.b * v.x_batch + t.row0 * v.x_row +
               static_cast<int64_t>(t.g0) * a.cg;
  float n = 0.f, mean = 0.f, m2 = 0.f;
  for (int col = t.tc; col < t.nvc; col += t.tcols) {
    const T* p = x + col * EPV;
    for (int r = t.tr; r < t.rows; r += t.trows * U) {
      Raw<VB> w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = r + u * t.trows;
        if (row < t.rows) w[u] = ld_chunk<VB>(p + row * v.x_row);
      }
      float s = 0.f, c = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u * t.trows < t.rows) {
          float f[EPV];
          Chunk<T, VB>::unpack(w[u], f);
#pragma unroll
          for (int i = 0; i < EPV; ++i) s += f[i];
          c += EPV;
        }
      const float cm = s / c;
      float q = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u * t.trows < t.rows) {
          float f[EPV];
          Chunk<T, VB>::unpack(w[u], f);
#pragma unroll
          for (int i = 0; i < EPV; ++i) q += (f[i] - cm) * (f[i] - cm);
        }
      norm_join(n, mean, m2, c, cm, q);
    }
  }
  part[threadIdx.x] = make_float3(n, mean, m2);
  __syncthreads();
  // lanes j of a group's `lanes` threads join its threads' results
  int lanes = 32;
  while (lanes * t.groups > kNormThreads) lanes >>= 1;
  const int g = threadIdx.x / lanes, j = threadIdx.x & (lanes - 1);
  const bool on = g < t.groups;
  const int per = t.groups == 1 ? t.tcols : a.cg / EPV;  // columns of a group
  n = mean = m2 = 0.f;
  if (on)
    for (int k = j; k < per * t.trows; k += lanes) {
      const float3 o = part[k / per * t.tcols + g * per + k % per];
      norm_join(n, mean, m2, o.x, o.y, o.z);
    }
  for (int d = 1; d < lanes; d <<= 1) {
    const float nb = __shfl_xor_sync(~0u, n, d), mb = __shfl_xor_sync(~0u, mean, d),
                sb = __shfl_xor_sync(~0u, m2, d);
    norm_join(n, mean, m2, nb, mb, sb);
  }
  if (v.tiles > 1) {
    if (on && j == 0) a.partial[block * a.partial_stride + g] = make_float2(mean, m2);
    if (!norm_last(a, t.unit, v.tiles)) return;
    n = mean = m2 = 0.f;
    if (on) {
      const float2* q = a.partial + (block - t.tile) * a.partial_stride + g;
      const float full = static_cast<float>(v.tile_rows) * a.cg;
      for (int k = j; k < v.tiles; k += lanes) {
        const float2 o = __ldcg(q + static_cast<int64_t>(k) * a.partial_stride);
        const float c = k + 1 < v.tiles ? full
                        : static_cast<float>(v.rows - static_cast<int64_t>(k) * v.tile_rows) * a.cg;
        norm_join(n, mean, m2, c, o.x, o.y);
      }
    }
    for (int d = 1; d < lanes; d <<= 1) {
      const float nb = __shfl_xor_sync(~0u, n, d), mb = __shfl_xor_sync(~0u, mean, d),
                  sb = __shfl_xor_sync(~0u, m2, d);
      norm_join(n, mean, m2, nb, mb, sb);
    }
  }
  if (on && j == 0)
    a.stats[t.segment(a) * a.G + t.g0 + g] = make_float2(mean, rsqrtf(m2 / n + a.eps));
}

template <typename T, int VB, int ACT, int U>
__device__ void norm_apply(const NormArgs& a, int64_t block) {
  constexpr int EPV = Chunk<T, VB>::EPV;
  const NormTile<EPV> t(a, block);
  const NormLevel& v = a.lv[t.l];
  for (int col = t.tc; col < t.nvc; col += t.tcols) {
    const int c0 = t.g0 * a.cg + col * EPV;
    const float2 st = __ldg(a.stats + t.segment(a) * a.G + c0 / a.cg);
    float w[EPV], d[EPV];
#pragma unroll
    for (int i = 0; i < EPV; ++i) {
      const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0 + i;
      w[i] = norm_param(a.weight, a.affine_dtype, at, 1.f) * st.y;
      d[i] = norm_param(a.bias, a.affine_dtype, at, 0.f);
    }
    const T* p = reinterpret_cast<const T*>(v.x) + t.b * v.x_batch + t.row0 * v.x_row + c0;
    T* y = reinterpret_cast<T*>(v.out) + t.b * v.out_batch + t.row0 * v.out_row + c0;
    for (int r = t.tr; r < t.rows; r += t.trows * U) {
      Raw<VB> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = r + u * t.trows;
        if (row < t.rows) raw[u] = ld_chunk<VB>(p + row * v.x_row);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = r + u * t.trows;
        if (row < t.rows) {
          float f[EPV];
          Chunk<T, VB>::unpack(raw[u], f);
#pragma unroll
          for (int i = 0; i < EPV; ++i) f[i] = norm_act<ACT>((f[i] - st.x) * w[i] + d[i]);
          st_chunk<VB>(y + row * v.out_row, Chunk<T, VB>::pack(f));
        }
      }
    }
  }
}

template <typename T, int VB, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads, 2)
norm_fwd_kernel(const __grid_constant__ NormArgs a, const NormWave w) {
  const int i = blockIdx.x;
  if (i < w.applies) norm_apply<T, VB, ACT, U>(a, w.apply0 + i);
  else norm_stats<T, VB, U>(a, w.stats0 + (i - w.applies));
}

// ------------------------------------------------------------------ backward
// Sums s1, s2 per channel of one tile; the unit's last CTA joins the tiles and
// forms the groups' coefficients a, q.
template <typename T, int VB, int ACT, int U>
__device__ void norm_grad_stats(const NormArgs& a, int64_t block) {
  constexpr int EPV = Chunk<T, VB>::EPV;
  __shared__ float2 part[kNormThreads][EPV];
  const NormTile<EPV> t(a, block);
  const NormLevel& v = a.lv[t.l];
  float2* mine = a.partial + block * a.partial_stride;
  for (int col0 = 0; col0 < t.nvc; col0 += t.tcols) {
    const int col = col0 + t.tc;
    float s1[EPV], s2[EPV];
#pragma unroll
    for (int i = 0; i < EPV; ++i) s1[i] = s2[i] = 0.f;
    if (col < t.nvc) {
      const int c0 = t.g0 * a.cg + col * EPV;
      const float2 st = __ldg(a.stats + t.segment(a) * a.G + c0 / a.cg);
      float w[EPV], d[EPV];
      if (ACT != MSDA_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0 + i;
          w[i] = norm_param(a.weight, a.affine_dtype, at, 1.f);
          d[i] = norm_param(a.bias, a.affine_dtype, at, 0.f);
        }
      }
      const T* p = reinterpret_cast<const T*>(v.x) + t.b * v.x_batch + t.row0 * v.x_row + c0;
      const T* g = reinterpret_cast<const T*>(v.gy) + t.b * v.gy_batch + t.row0 * v.gy_row + c0;
      for (int r = t.tr; r < t.rows; r += t.trows * U) {
        Raw<VB> rx[U], rg[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int row = r + u * t.trows;
          if (row < t.rows) {
            rx[u] = ld_chunk<VB>(p + row * v.x_row);
            rg[u] = ld_chunk<VB>(g + row * v.gy_row);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (r + u * t.trows < t.rows) {
            float f[EPV], e[EPV];
            Chunk<T, VB>::unpack(rx[u], f);
            Chunk<T, VB>::unpack(rg[u], e);
#pragma unroll
            for (int i = 0; i < EPV; ++i) {
              const float h = (f[i] - st.x) * st.y;
              const float dz =
                  ACT == MSDA_ACT_NONE ? e[i] : e[i] * norm_dact<ACT>(h * w[i] + d[i]);
              s1[i] += dz;
              s2[i] += dz * h;
            }
          }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EPV; ++i) part[threadIdx.x][i] = make_float2(s1[i], s2[i]);
    __syncthreads();
    const int cols = min(t.tcols, t.nvc - col0);
    for (int c = threadIdx.x; c < cols * EPV; c += kNormThreads) {
      float2 s = make_float2(0.f, 0.f);
      for (int k = 0; k < t.trows; ++k) {
        const float2 o = part[k * t.tcols + c / EPV][c % EPV];
        s.x += o.x;
        s.y += o.y;
      }
      mine[col0 * EPV + c] = s;
    }
  }
  if (!norm_last(a, t.unit, v.tiles)) return;
  const int cw = t.groups * a.cg, c0 = t.g0 * a.cg;
  const float2* q = a.partial + (block - t.tile) * a.partial_stride;
  float2* chan = a.chan + t.segment(a) * a.C + c0;
  // `lanes` threads of a channel take the tiles in turn
  int lanes = 32;
  while (lanes > 1 && lanes * cw > kNormThreads) lanes >>= 1;
  const int per = kNormThreads / lanes;
  for (int base = 0; base < cw; base += per) {
    const int c = base + threadIdx.x / lanes;
    float2 s = make_float2(0.f, 0.f);
    if (c < cw)
      for (int k = threadIdx.x & (lanes - 1); k < v.tiles; k += lanes) {
        const float2 o = __ldcg(q + static_cast<int64_t>(k) * a.partial_stride + c);
        s.x += o.x;
        s.y += o.y;
      }
    for (int d = 1; d < lanes; d <<= 1) {
      s.x += __shfl_xor_sync(~0u, s.x, d);
      s.y += __shfl_xor_sync(~0u, s.y, d);
    }
    if (c < cw && (threadIdx.x & (lanes - 1)) == 0) chan[c] = s;
  }
  __syncthreads();
  const float n = static_cast<float>(v.rows) * a.cg;
  for (int g = threadIdx.x; g < t.groups; g += kNormThreads) {
    float sa = 0.f, sq = 0.f;
    for (int i = 0; i < a.cg; ++i) {
      const int c = g * a.cg + i;
      const float w = norm_param(a.weight, a.affine_dtype,
                                 static_cast<int64_t>(t.l) * a.affine_level + c0 + c, 1.f);
      const float2 s = chan[c];
      sa += w * s.x;
      sq += w * s.y;
    }
    a.coef[t.segment(a) * a.G + t.g0 + g] = make_float2(sa / n, sq / n);
  }
}

template <typename T, int VB, int ACT, int U>
__device__ void norm_grad_apply(const NormArgs& a, int64_t block) {
  constexpr int EPV = Chunk<T, VB>::EPV;
  const NormTile<EPV> t(a, block);
  const NormLevel& v = a.lv[t.l];
  for (int col = t.tc; col < t.nvc; col += t.tcols) {
    const int c0 = t.g0 * a.cg + col * EPV;
    const float2 st = __ldg(a.stats + t.segment(a) * a.G + c0 / a.cg);
    const float2 co = __ldg(a.coef + t.segment(a) * a.G + c0 / a.cg);
    float w[EPV], d[EPV];
#pragma unroll
    for (int i = 0; i < EPV; ++i) {
      const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0 + i;
      w[i] = norm_param(a.weight, a.affine_dtype, at, 1.f);
      if (ACT != MSDA_ACT_NONE) d[i] = norm_param(a.bias, a.affine_dtype, at, 0.f);
    }
    const T* p = reinterpret_cast<const T*>(v.x) + t.b * v.x_batch + t.row0 * v.x_row + c0;
    const T* g = reinterpret_cast<const T*>(v.gy) + t.b * v.gy_batch + t.row0 * v.gy_row + c0;
    T* y = reinterpret_cast<T*>(v.out) + t.b * v.out_batch + t.row0 * v.out_row + c0;
    for (int r = t.tr; r < t.rows; r += t.trows * U) {
      Raw<VB> rx[U], rg[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = r + u * t.trows;
        if (row < t.rows) {
          rx[u] = ld_chunk<VB>(p + row * v.x_row);
          rg[u] = ld_chunk<VB>(g + row * v.gy_row);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = r + u * t.trows;
        if (row < t.rows) {
          float f[EPV], e[EPV];
          Chunk<T, VB>::unpack(rx[u], f);
          Chunk<T, VB>::unpack(rg[u], e);
#pragma unroll
          for (int i = 0; i < EPV; ++i) {
            const float h = (f[i] - st.x) * st.y;
            const float dz = ACT == MSDA_ACT_NONE ? e[i] : e[i] * norm_dact<ACT>(h * w[i] + d[i]);
            f[i] = st.y * (dz * w[i] - co.x - h * co.y);
          }
          st_chunk<VB>(y + row * v.out_row, Chunk<T, VB>::pack(f));
        }
      }
    }
  }
}

template <typename T, int VB, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads, 2)
norm_bwd_kernel(const __grid_constant__ NormArgs a, const NormWave w) {
  const int i = blockIdx.x;
  if (i < w.applies) norm_grad_apply<T, VB, ACT, U>(a, w.apply0 + i);
  else norm_grad_stats<T, VB, ACT, U>(a, w.stats0 + (i - w.applies));
}

// ------------------------------------------------------------------ launches
template <typename T, int VB, int ACT>
cudaError_t norm_launch(const NormArgs& a, const NormWave& w, bool backward, cudaStream_t st) {
  const unsigned int grid = static_cast<unsigned int>(w.applies + w.stats);
  if (grid == 0) return cudaSuccess;
  if (backward) norm_bwd_kernel<T, VB, ACT, 4><<<grid, kNormThreads, 0, st>>>(a, w);
  else norm_fwd_kernel<T, VB, ACT, 8><<<grid, kNormThreads, 0, st>>>(a, w);
  return cudaGetLastError();
}

template <typename T, int VB>
cudaError_t norm_launch_act(const NormArgs& a, const NormWave& w, int act, bool backward,
                            cudaStream_t st) {
  switch (act) {
    case MSDA_ACT_RELU: return norm_launch<T, VB, MSDA_ACT_RELU>(a, w, backward, st);
    case MSDA_ACT_SILU: return norm_launch<T, VB, MSDA_ACT_SILU>(a, w, backward, st);
    case MSDA_ACT_GELU: return norm_launch<T, VB, MSDA_ACT_GELU>(a, w, backward, st);
    default: return norm_launch<T, VB, MSDA_ACT_NONE>(a, w, backward, st);
  }
}

template <typename T>
cudaError_t norm_wave_t(const NormArgs& a, const NormWave& w, int vb, int act, bool backward,
                        cudaStream_t st) {
  switch (vb) {
    case 16: return norm_launch_act<T, 16>(a, w, act, backward, st);
    case 8: return norm_launch_act<T, 8>(a, w, act, backward, st);
    case 4: return norm_launch_act<T, 4>(a, w, act, backward, st);
    default:
      if constexpr (sizeof(T) == 2) return norm_launch_act<T, 2>(a, w, act, backward, st);
      return cudaErrorInvalidValue;
  }
}

}  // namespace msda
