// msda_norm_kernels.cuh -- device code of msda_norm.cuh's passes.
#pragma once

#include "msda_b200.h"
#include "msda_norm.cuh"

namespace msda {

template <int K> struct Count { static constexpr int value = K; };

__device__ __forceinline__ float norm_param(const void* p, int dtype, int64_t i, float none) {
  if (p == nullptr) return none;
  if (dtype == MSDA_FLOAT32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == MSDA_FLOAT16) return __half2float(__ldg(static_cast<const __half*>(p) + i));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
}

// 1 / (1 + exp(-z)): 0 where the exponential overflows.
__device__ __forceinline__ float norm_sigmoid(float z) {
  return __fdividef(1.f, 1.f + __expf(-z));
}

// act(z); dact: act'(z).  A NaN stays one.
template <int ACT> __device__ __forceinline__ float norm_act(float z) {
  if (ACT == MSDA_ACT_RELU) return z < 0.f ? 0.f : z;
  if (ACT == MSDA_ACT_SILU) return z * norm_sigmoid(z);
  if (ACT == MSDA_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678f));
  return z;
}
template <int ACT> __device__ __forceinline__ float norm_dact(float z) {
  if (ACT == MSDA_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
  if (ACT == MSDA_ACT_SILU) {
    const float s = norm_sigmoid(z);
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
  const float nn = n + nb, d = mb - mean, f = __fdividef(nb, nn);
  mean += d * f;
  m2 += sb + d * d * n * f;
  n = nn;
}

// Where a tile lies, and which of its vectors a thread takes: column tc (then
// tc + tcols, ... where one group is wider than the CTA), rows tr, tr + trows, ...
template <int EPV> struct NormTile {
  int l, counter, tile, step, groups, nvc, tcols, trows, tc, tr, rows, g0;  // step: blocks to the unit's next tile
  int64_t b, row0;
  __device__ __forceinline__ NormTile(const NormArgs& a, int64_t block) {
    l = a.L - 1;
    while (block < a.lv[l].block0) --l;
    const NormLevel& v = a.lv[l];
    const int64_t rel = block - v.block0;
    const int64_t seg = static_cast<int64_t>(v.slabs) * v.tiles;
    b = rel / seg;
    int64_t r = rel - b * seg;
    const int64_t together = static_cast<int64_t>(v.run) * v.tiles;
    const int s0 = static_cast<int>(r / together) * v.run;
    r -= static_cast<int64_t>(s0) * v.tiles;
    const int width = min(v.run, v.slabs - s0);
    tile = static_cast<int>(r / width);
    const int slab = s0 + static_cast<int>(r - static_cast<int64_t>(tile) * width);
    step = width;
    counter = v.done0 + (static_cast<int>(b) * v.slabs + slab) * (1 + (v.tiles + kNormFan - 1) / kNormFan);
    g0 = slab * v.slab_groups;
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

// Whether this CTA is the last of `count`: what the others wrote is then visible.
__device__ __forceinline__ bool norm_last(unsigned int* done, int count) {
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(done, 1u) == static_cast<unsigned int>(count - 1);
  __syncthreads();
  __threadfence();
  return last != 0;
}

// Joins a unit's partial results, kNormFan tiles at a time and then those
// groups, by whichever CTA is last.  join(slot, next, count, full, tail, final)
// joins `count` results that lie `next` tiles apart from tile `slot`, each of
// `full` rows (the last of `tail`), into tile `slot`'s or, with `final`, into
// the unit's.
template <typename Join>
__device__ __forceinline__ void norm_join_tiles(const NormArgs& a, const NormLevel& v, int counter,
                                                int tile, Join join) {
  const int group = tile / kNormFan, groups = (v.tiles + kNormFan - 1) / kNormFan;
  const int first = group * kNormFan, count = min(kNormFan, v.tiles - first);
  const int64_t full = v.tile_rows, last = v.rows - (v.tiles - 1) * full;
  if (!norm_last(a.done + counter + 1 + group, count)) return;
  join(first, 1, count, full, group + 1 < groups ? full : last, groups == 1);
  if (groups == 1) return;
  if (!norm_last(a.done + counter, groups)) return;
  join(0, kNormFan, groups, full * kNormFan, v.rows - (groups - 1) * full * kNormFan, true);
}

// A launch may start before the one ahead of it has ended: its statistics need
// nothing of that one, its applications wait for it.
__device__ __forceinline__ void norm_let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void norm_wait_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Whether this CTA applies, and its tile.
__device__ __forceinline__ bool norm_applies(const NormWave& w, int64_t& block) {
  const int i = blockIdx.x;
  if (w.order == 0) {  // apply first
    if (i < w.applies) { block = w.apply0 + i; return true; }
    block = w.stats0 + (i - w.applies);
    return false;
  }
  if (w.order == 1) {
    if (i < w.stats) { block = w.stats0 + i; return false; }
    block = w.apply0 + (i - w.stats);
    return true;
  }
  const int both = min(w.applies, w.stats);
  if (i < 2 * both) {
    block = (i & 1) ? w.apply0 + (i >> 1) : w.stats0 + (i >> 1);
    return i & 1;
  }
  if (w.applies > both) { block = w.apply0 + (i - both); return true; }
  block = w.stats0 + (i - both);
  return false;
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
    const T* p = x + col * EPV + t.tr * v.x_row;
    const int64_t hop = t.trows * v.x_row;
    auto chunk = [&](auto count) {
      constexpr int K = decltype(count)::value;
      Raw<VB> w[K];
#pragma unroll
      for (int u = 0; u < K; ++u) w[u] = ld_chunk<VB>(p + u * hop);
      p += K * hop;
      float s = 0.f, q = 0.f;
#pragma unroll
      for (int u = 0; u < K; ++u) {
        float f[EPV];
        Chunk<T, VB>::unpack(w[u], f);
#pragma unroll
        for (int i = 0; i < EPV; ++i) s += f[i];
      }
      const float cm = s * (1.f / (K * EPV));
#pragma unroll
      for (int u = 0; u < K; ++u) {
        float f[EPV];
        Chunk<T, VB>::unpack(w[u], f);
#pragma unroll
        for (int i = 0; i < EPV; ++i) q += (f[i] - cm) * (f[i] - cm);
      }
      norm_join(n, mean, m2, K * EPV, cm, q);
    };
    int r = t.tr;
    for (; r + (U - 1) * t.trows < t.rows; r += U * t.trows) chunk(Count<U>{});
    for (; r < t.rows; r += t.trows) chunk(Count<1>{});
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
  auto finish = [&](float mu, float var) {
    if (on && j == 0)
      a.stats[t.segment(a) * a.G + t.g0 + g] = make_float2(mu, rsqrtf(var + a.eps));
  };
  if (v.tiles == 1) {
    finish(mean, m2 / n);
    return;
  }
  float2* const mine = a.partial + (block - static_cast<int64_t>(t.tile) * t.step) * a.partial_stride + g;
  const int64_t hop = static_cast<int64_t>(t.step) * a.partial_stride;
  if (on && j == 0) mine[t.tile * hop] = make_float2(mean, m2);
  norm_join_tiles(a, v, t.counter, t.tile, [&](int slot, int next, int count, int64_t full,
                                               int64_t tail, bool final) {
    // the mean of the means, then the deviations from it
    const float nf = static_cast<float>(full) * a.cg, nt = static_cast<float>(tail) * a.cg;
    const float all = nf * (count - 1) + nt;
    const float2* q = mine + slot * hop;
    float mu = 0.f, dev = 0.f;
    if (on)
      for (int k = j; k < count; k += lanes)
        mu += __ldcg(&q[k * next * hop].x) * ((k + 1 < count ? nf : nt) / all);
    for (int d = 1; d < lanes; d <<= 1) mu += __shfl_xor_sync(~0u, mu, d);
    if (on)
      for (int k = j; k < count; k += lanes) {
        const float2 o = __ldcg(q + k * next * hop);
        dev += o.y + (o.x - mu) * (o.x - mu) * (k + 1 < count ? nf : nt);
      }
    for (int d = 1; d < lanes; d <<= 1) dev += __shfl_xor_sync(~0u, dev, d);
    if (final) finish(mu, dev / all);
    else if (on && j == 0) mine[slot * hop] = make_float2(mu, dev);
  });
}

template <typename T, int VB, int ACT, int U>
__device__ void norm_apply(const NormArgs& a, int64_t block) {
  constexpr int EPV = Chunk<T, VB>::EPV;
  const NormTile<EPV> t(a, block);
  const NormLevel& v = a.lv[t.l];
  for (int col = t.tc; col < t.nvc; col += t.tcols) {
    const int c0 = t.g0 * a.cg + col * EPV;
    const float2 st = __ldcg(a.stats + t.segment(a) * a.G + c0 / a.cg);
    float w[EPV], d[EPV];
#pragma unroll
    for (int i = 0; i < EPV; ++i) {
      const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0 + i;
      w[i] = norm_param(a.weight, a.affine_dtype, at, 1.f) * st.y;
      d[i] = norm_param(a.bias, a.affine_dtype, at, 0.f);
      // 16-bit x has no digits that the mean's product could lose: one step less
      if (sizeof(T) == 2) d[i] -= st.x * w[i];
    }
    const T* p = reinterpret_cast<const T*>(v.x) + t.b * v.x_batch + (t.row0 + t.tr) * v.x_row + c0;
    T* y = reinterpret_cast<T*>(v.out) + t.b * v.out_batch + (t.row0 + t.tr) * v.out_row + c0;
    const int64_t hop = t.trows * v.x_row, yhop = t.trows * v.out_row;
    auto chunk = [&](auto count) {
      constexpr int K = decltype(count)::value;
      Raw<VB> raw[K];
#pragma unroll
      for (int u = 0; u < K; ++u) raw[u] = ld_chunk<VB>(p + u * hop);
      p += K * hop;
#pragma unroll
      for (int u = 0; u < K; ++u) {
        float f[EPV];
        Chunk<T, VB>::unpack(raw[u], f);
#pragma unroll
        for (int i = 0; i < EPV; ++i)
          f[i] = norm_act<ACT>((sizeof(T) == 2 ? f[i] : f[i] - st.x) * w[i] + d[i]);
        st_chunk<VB>(y + u * yhop, Chunk<T, VB>::pack(f));
      }
      y += K * yhop;
    };
    int r = t.tr;
    for (; r + (U - 1) * t.trows < t.rows; r += U * t.trows) chunk(Count<U>{});
    for (; r < t.rows; r += t.trows) chunk(Count<1>{});
  }
}

template <typename T, int VB, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads, 4)
norm_fwd_kernel(const __grid_constant__ NormArgs a, const NormWave w) {
  norm_let_next_start();
  int64_t block;
  if (norm_applies(w, block)) {
    norm_wait_previous();
    norm_apply<T, VB, ACT, U>(a, block);
  } else {
    norm_stats<T, VB, U>(a, block);
  }
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
      const float2 st = __ldcg(a.stats + t.segment(a) * a.G + c0 / a.cg);
      float w[EPV], d[EPV];
      if (ACT != MSDA_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0 + i;
          w[i] = norm_param(a.weight, a.affine_dtype, at, 1.f);
          d[i] = norm_param(a.bias, a.affine_dtype, at, 0.f);
        }
      }
      const T* p = reinterpret_cast<const T*>(v.x) + t.b * v.x_batch + (t.row0 + t.tr) * v.x_row + c0;
      const T* g = reinterpret_cast<const T*>(v.gy) + t.b * v.gy_batch + (t.row0 + t.tr) * v.gy_row + c0;
      const int64_t hop = t.trows * v.x_row, ghop = t.trows * v.gy_row;
      auto chunk = [&](auto count) {
        constexpr int K = decltype(count)::value;
        Raw<VB> rx[K], rg[K];
#pragma unroll
        for (int u = 0; u < K; ++u) {
          rx[u] = ld_chunk<VB>(p + u * hop);
          rg[u] = ld_chunk<VB>(g + u * ghop);
        }
        p += K * hop;
        g += K * ghop;
#pragma unroll
        for (int u = 0; u < K; ++u) {
          float f[EPV], e[EPV];
          Chunk<T, VB>::unpack(rx[u], f);
          Chunk<T, VB>::unpack(rg[u], e);
#pragma unroll
          for (int i = 0; i < EPV; ++i) {
            const float h = (f[i] - st.x) * st.y;
            const float dz = ACT == MSDA_ACT_NONE ? e[i] : e[i] * norm_dact<ACT>(h * w[i] + d[i]);
            s1[i] += dz;
            s2[i] += dz * h;
          }
        }
      };
      int r = t.tr;
      for (; r + (U - 1) * t.trows < t.rows; r += U * t.trows) chunk(Count<U>{});
      for (; r < t.rows; r += t.trows) chunk(Count<1>{});
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
  const int cw = t.groups * a.cg, c0 = t.g0 * a.cg;
  float2* const first = a.partial + (block - static_cast<int64_t>(t.tile) * t.step) * a.partial_stride;
  const int64_t hop = static_cast<int64_t>(t.step) * a.partial_stride;
  float2* const chan = a.chan + t.segment(a) * a.C + c0;
  norm_join_tiles(a, v, t.counter, t.tile, [&](int slot, int next, int count, int64_t, int64_t,
                                               bool final) {
    // `lanes` threads of a channel take the tiles in turn
    int lanes = 32;
    while (lanes > 1 && lanes * cw > kNormThreads) lanes >>= 1;
    const int per = kNormThreads / lanes, lane = threadIdx.x & (lanes - 1);
    for (int base = 0; base < cw; base += per) {
      const int c = base + threadIdx.x / lanes;
      float2 s = make_float2(0.f, 0.f);
      if (c < cw) {
#pragma unroll 8
        for (int k = lane; k < count; k += lanes) {
          const float2 o = __ldcg(first + (slot + k * next) * hop + c);
          s.x += o.x;
          s.y += o.y;
        }
      }
      for (int d = 1; d < lanes; d <<= 1) {
        s.x += __shfl_xor_sync(~0u, s.x, d);
        s.y += __shfl_xor_sync(~0u, s.y, d);
      }
      if (c < cw && lane == 0) (final ? chan : first + slot * hop)[c] = s;
    }
    if (!final) return;
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
  });
}

template <typename T, int VB, int ACT, int U>
__device__ void norm_grad_apply(const NormArgs& a, int64_t block) {
  constexpr int EPV = Chunk<T, VB>::EPV;
  const NormTile<EPV> t(a, block);
  const NormLevel& v = a.lv[t.l];
  for (int col = t.tc; col < t.nvc; col += t.tcols) {
    const int c0 = t.g0 * a.cg + col * EPV;
    const float2 st = __ldcg(a.stats + t.segment(a) * a.G + c0 / a.cg);
    const float2 co = __ldcg(a.coef + t.segment(a) * a.G + c0 / a.cg);
    float w[EPV], d[EPV];
#pragma unroll
    for (int i = 0; i < EPV; ++i) {
      const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0 + i;
      w[i] = norm_param(a.weight, a.affine_dtype, at, 1.f);
      if (ACT != MSDA_ACT_NONE) d[i] = norm_param(a.bias, a.affine_dtype, at, 0.f);
    }
    const T* p = reinterpret_cast<const T*>(v.x) + t.b * v.x_batch + (t.row0 + t.tr) * v.x_row + c0;
    const T* g = reinterpret_cast<const T*>(v.gy) + t.b * v.gy_batch + (t.row0 + t.tr) * v.gy_row + c0;
    T* y = reinterpret_cast<T*>(v.out) + t.b * v.out_batch + (t.row0 + t.tr) * v.out_row + c0;
    const int64_t hop = t.trows * v.x_row, ghop = t.trows * v.gy_row, yhop = t.trows * v.out_row;
    const float ra = st.y * co.x, rq = st.y * co.y;
    auto chunk = [&](auto count) {
      constexpr int K = decltype(count)::value;
      Raw<VB> rx[K], rg[K];
#pragma unroll
      for (int u = 0; u < K; ++u) {
        rx[u] = ld_chunk<VB>(p + u * hop);
        rg[u] = ld_chunk<VB>(g + u * ghop);
      }
      p += K * hop;
      g += K * ghop;
#pragma unroll
      for (int u = 0; u < K; ++u) {
        float f[EPV], e[EPV];
        Chunk<T, VB>::unpack(rx[u], f);
        Chunk<T, VB>::unpack(rg[u], e);
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const float h = (f[i] - st.x) * st.y;
          const float dz = ACT == MSDA_ACT_NONE ? e[i] : e[i] * norm_dact<ACT>(h * w[i] + d[i]);
          f[i] = dz * (st.y * w[i]) - ra - h * rq;
        }
        st_chunk<VB>(y + u * yhop, Chunk<T, VB>::pack(f));
      }
      y += K * yhop;
    };
    int r = t.tr;
    for (; r + (U - 1) * t.trows < t.rows; r += U * t.trows) chunk(Count<U>{});
    for (; r < t.rows; r += t.trows) chunk(Count<1>{});
  }
}

template <typename T, int VB, int ACT, int U>
__global__ void __launch_bounds__(kNormThreads, 3)
norm_bwd_kernel(const __grid_constant__ NormArgs a, const NormWave w) {
  norm_let_next_start();
  int64_t block;
  if (norm_applies(w, block)) {
    norm_wait_previous();
    norm_grad_apply<T, VB, ACT, U>(a, block);
  } else {
    norm_grad_stats<T, VB, ACT, U>(a, block);
  }
}

// ------------------------------------------------------------------ launches
template <typename T, int VB, int ACT>
cudaError_t norm_launch(const NormArgs& a, const NormWave& w, bool backward, cudaStream_t st) {
  const unsigned int grid = static_cast<unsigned int>(w.applies + w.stats);
  if (grid == 0) return cudaSuccess;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kNormThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = w.applies > 0 ? 1 : 0;  // the first launch follows other work
  return backward ? cudaLaunchKernelEx(&cfg, norm_bwd_kernel<T, VB, ACT, 2>, a, w)
                  : cudaLaunchKernelEx(&cfg, norm_fwd_kernel<T, VB, ACT, 4>, a, w);
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
