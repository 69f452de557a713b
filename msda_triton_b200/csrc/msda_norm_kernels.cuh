// msda_norm_kernels.cuh -- device code of msda_norm.cuh's items.
#pragma once

#include "msda_b200.h"
#include "msda_f32x2.cuh"
#include "msda_norm.cuh"

// Loads that leave L1 alone, and stores that L2 lets go of first: the forward
// reads each row twice from L2 or DRAM and never its output (647 -> 582 us for
// the 1.23 GB of two 3D xl pyramids).  The backward is slower with such stores
// (1130 -> 1210 us).
namespace msda {

template <int VB> __device__ __forceinline__ Raw<VB> norm_ld(const void* p) {
  if constexpr (VB == 16) {
    Raw<16> r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(p));
    return r;
  } else {
    return ld_chunk<VB>(p);
  }
}
template <int VB> __device__ __forceinline__ void norm_st(void* p, const Raw<VB>& r) {
  if constexpr (VB == 16)
    __stcs(static_cast<uint4*>(p), make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]));
  else
    st_chunk<VB>(p, r);
}

template <int K> struct Count { static constexpr int value = K; };

// -x twice, as a pair (a vector of a single element has no second half), where
// T is fp32; else zeros.  A chunk's mean is taken from what its elements lie off
// its first one: a sum of 32 elements of 31000 is off by several units of its
// last place, and their mean then by as many of its own, 0.004.  Such sums of
// 16-bit elements are exact.
template <typename T, int EPV> __device__ __forceinline__ uint64_t norm_off(uint64_t x) {
  float a, b;
  unpair(x, a, b);
  return sizeof(T) == 2 ? 0 : pair(-a, EPV == 1 ? 0.f : -a);
}
__device__ __forceinline__ float norm_first(uint64_t off) {
  float a, b;
  unpair(off, a, b);
  return -a;
}

// EPV parameters from element i on.
template <int EPV>
__device__ __forceinline__ void norm_params(const void* p, int dtype, int64_t i, float none,
                                            float* f) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < EPV; ++k) f[k] = none;
  } else if (dtype == MSDA_FLOAT32) {
    const float* q = static_cast<const float*>(p) + i;
    if (EPV % 4 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0) {
#pragma unroll
      for (int k = 0; k + 3 < EPV; k += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(q + k));
        f[k] = v.x; f[k + 1] = v.y; f[k + 2] = v.z; f[k + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int k = 0; k < EPV; ++k) f[k] = __ldg(q + k);
    }
  } else if (dtype == MSDA_FLOAT16) {
#pragma unroll
    for (int k = 0; k < EPV; ++k) f[k] = __half2float(__ldg(static_cast<const __half*>(p) + i + k));
  } else {
#pragma unroll
    for (int k = 0; k < EPV; ++k)
      f[k] = __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i + k));
  }
}

// A vector as pairs of fp32; one of a single element has a second one of 0.
template <typename T, int VB> struct Pairs {
  static constexpr int EPV = Chunk<T, VB>::EPV, N = (EPV + 1) / 2;
  static __device__ __forceinline__ void unpack(const Raw<VB>& r, uint64_t* p) {
    float f[2 * N];
    f[2 * N - 1] = 0.f;
    Chunk<T, VB>::unpack(r, f);
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = pair(f[2 * i], f[2 * i + 1]);
  }
  static __device__ __forceinline__ Raw<VB> pack(const uint64_t* p) {
    float f[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) unpair(p[i], f[2 * i], f[2 * i + 1]);
    return Chunk<T, VB>::pack(f);
  }
  static __device__ __forceinline__ void of(const float* f, uint64_t* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = pair(f[2 * i], 2 * i + 1 < EPV ? f[2 * i + 1] : 0.f);
  }
};

// 1 / (1 + exp(-z)); 0 where the exponential overflows.
__device__ __forceinline__ uint64_t norm_sigmoid(uint64_t z) {
  float a, b;
  unpair(mul2(z, pair(-1.4426950409f, -1.4426950409f)), a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  unpair(add2(pair(a, b), pair(1.f, 1.f)), a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return pair(a, b);
}
__device__ __forceinline__ float norm_cdf(float z) { return 0.5f * (1.f + erff(z * 0.70710678f)); }

// act(z) of t = z * norm_arg<ACT>, a factor that the affine map takes in: the
// exponential's and the error function's argument then needs no product of its
// own, and a row no more operations than before its x was centred (580 us for
// the 1.23 GB of two 3D xl pyramids in bf16 with SiLU, 623 with the product).
//   SiLU: t = -z log2 e,      z / (1 + 2^t) = t / (-log2 e (1 + 2^t))
//   GELU: t = z / sqrt 2,     z (1 + erf t) / 2 = h + h erf t,  h = t / sqrt 2
// A NaN stays one.
template <int ACT>
constexpr float norm_arg = ACT == MSDA_ACT_SILU   ? -1.4426950409f
                           : ACT == MSDA_ACT_GELU ? 0.70710678f
                                                  : 1.f;

template <int ACT> __device__ __forceinline__ uint64_t norm_act(uint64_t t) {
  if (ACT == MSDA_ACT_NONE) return t;
  float a, b;
  unpair(t, a, b);
  if (ACT == MSDA_ACT_RELU) return pair(a < 0.f ? 0.f : a, b < 0.f ? 0.f : b);
  if (ACT == MSDA_ACT_SILU) {
    constexpr float k = norm_arg<MSDA_ACT_SILU>;
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    unpair(fma2(pair(a, b), pair(k, k), pair(k, k)), a, b);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
    return mul2(t, pair(a, b));
  }
  const uint64_t h = mul2(t, pair(0.70710678f, 0.70710678f));
  return fma2(h, pair(erff(a), erff(b)), h);
}
// act'(z).
template <int ACT> __device__ __forceinline__ uint64_t norm_dact(uint64_t z) {
  if (ACT == MSDA_ACT_SILU) {  // s (1 + z (1 - s))
    const uint64_t s = norm_sigmoid(z), zs = mul2(z, s);
    return fma2(s, fma2(zs, pair(-1.f, -1.f), z), s);
  }
  float a, b;
  unpair(z, a, b);
  if (ACT == MSDA_ACT_RELU) return pair(a <= 0.f ? 0.f : 1.f, b <= 0.f ? 0.f : 1.f);
  return pair(norm_cdf(a) + a * 0.39894228f * __expf(-0.5f * a * a),
              norm_cdf(b) + b * 0.39894228f * __expf(-0.5f * b * b));
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

// ------------------------------------------------------------------ tiles
struct NormTile {
  int l, b, counter;
  int block, tile, step;  // step: blocks to the unit's next tile
  int groups, g0, rows, nvc, tcols, trows;
  int64_t row0;
};

// A segment's slabs go side by side, tile by tile: neighbouring CTAs read
// neighbouring pieces of the same rows.
template <int EPV, int THREADS = kNormThreads>
__host__ __device__ __forceinline__ NormTile norm_tile(const NormArgs& a, int block) {
  NormTile t;
  t.block = block;
  t.l = a.L - 1;
  while (block < a.lv[t.l].tile0) --t.l;
  const NormLevel& v = a.lv[t.l];
  const int rel = block - v.tile0, seg = v.slabs * v.tiles;
  t.b = rel / seg;
  const int r = rel - t.b * seg;
  t.tile = r / v.slabs;
  t.step = v.slabs;
  const int slab = r - t.tile * v.slabs;
  t.counter = v.done0 + (t.b * v.slabs + slab) * (1 + (v.tiles + kNormFan - 1) / kNormFan);
  t.g0 = slab * v.slab_groups;
  t.groups = min(v.slab_groups, a.G - t.g0);
  t.row0 = static_cast<int64_t>(t.tile) * v.tile_rows;
  t.rows = static_cast<int>(min(static_cast<int64_t>(v.tile_rows), v.rows - t.row0));
  t.nvc = t.groups * a.cg / EPV;
  t.tcols = min(t.nvc, THREADS);
  t.trows = THREADS / t.tcols;
  return t;
}

// A thread's vectors of a tile: column tc (then tc + tcols, ... where one
// group is wider than the CTA), rows tr, tr + trows, ...
struct NormThread {
  int tc, tr;
  int64_t segment, seg_group, seg_chan;
  __device__ __forceinline__ NormThread(const NormArgs& a, const NormTile& t) {
    tr = threadIdx.x / t.tcols;
    tc = threadIdx.x - tr * t.tcols;
    if (tr >= t.trows) tr = t.rows;  // no rows
    segment = static_cast<int64_t>(t.b) * a.L + t.l;
    seg_group = segment * a.G + t.g0;
    seg_chan = segment * a.C + static_cast<int64_t>(t.g0) * a.cg;
  }
};

// Calls chunk(Count<U>) while U rows are left, then chunk(Count<1>).
template <int U, typename Chunk>
__device__ __forceinline__ void norm_rows(const NormTile& t, int tr, Chunk chunk) {
  int r = tr;
  for (; r + (U - 1) * t.trows < t.rows; r += U * t.trows) chunk(Count<U>{});
  for (; r < t.rows; r += t.trows) chunk(Count<1>{});
}

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
__device__ __forceinline__ void norm_join_tiles(const NormArgs& a, const NormTile& t, Join join) {
  const NormLevel& v = a.lv[t.l];
  const int group = t.tile / kNormFan, groups = (v.tiles + kNormFan - 1) / kNormFan;
  const int first = group * kNormFan, count = min(kNormFan, v.tiles - first);
  const int64_t full = v.tile_rows, last = v.rows - (v.tiles - 1) * full;
  if (!norm_last(a.done + t.counter + 1 + group, count)) return;
  join(first, 1, count, full, group + 1 < groups ? full : last, groups == 1);
  if (groups == 1) return;
  if (!norm_last(a.done + t.counter, groups)) return;
  join(0, kNormFan, groups, full * kNormFan, v.rows - (groups - 1) * full * kNormFan, true);
}

// The second launch may start before the first has ended, and waits for it.
__device__ __forceinline__ void norm_let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void norm_wait_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------------ forward
// MIXED, here and below: a vector holds channels of several groups (groups of
// no whole vectors: 320 channels in 32).  Sums are then carried per channel.
// Read in pieces of 4 or 2 bytes, 168 MB of bf16 with 10 channels a group take
// 169 us forward and 392 backward; in such vectors 143 and 219.
template <typename T, int VB, bool DIRECT, bool MIXED, int U>
__device__ void norm_stats(const NormArgs& a, const NormTile& t) {
  using P = Pairs<T, VB>;
  constexpr int EPV = P::EPV;
  // MIXED: each thread's channels' (mean, squared deviations); else (count,
  // mean, squared deviations) of its vectors
  __shared__ float2 channels[MIXED ? kNormThreads * EPV : 1];
  __shared__ float3 part[MIXED ? 1 : kNormThreads];
  const NormLevel& v = a.lv[t.l];
  const NormThread me(a, t);
  const T* x = reinterpret_cast<const T*>(v.x) + v.x_batch * t.b + (t.row0 + me.tr) * v.x_row +
               static_cast<int64_t>(t.g0) * a.cg;
  const int64_t hop = t.trows * v.x_row;
  float n = 0.f, mean = 0.f, m2 = 0.f;
  if constexpr (MIXED) {
    // deviations from the thread's first row, which no outlier elsewhere spoils
    const T* p = x + me.tc * EPV;
    uint64_t minus[P::N], s[P::N], q[P::N];
    if (me.tr < t.rows) P::unpack(norm_ld<VB>(p), minus);
#pragma unroll
    for (int i = 0; i < P::N; ++i) {
      minus[i] = mul2(minus[i], pair(-1.f, -1.f));
      s[i] = q[i] = 0;  // two zeros
    }
    norm_rows<U / 2>(t, me.tr, [&](auto count) {
      constexpr int K = decltype(count)::value;
      Raw<VB> w[K];
#pragma unroll
      for (int u = 0; u < K; ++u) w[u] = norm_ld<VB>(p + u * hop);
      p += K * hop;
#pragma unroll
      for (int u = 0; u < K; ++u) {
        uint64_t f[P::N];
        P::unpack(w[u], f);
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
          const uint64_t d = add2(f[i], minus[i]);
          s[i] = add2(s[i], d);
          q[i] = fma2(d, d, q[i]);
        }
      }
    });
    const float inv = 1.f / static_cast<float>(max(1, (t.rows - me.tr + t.trows - 1) / t.trows));
#pragma unroll
    for (int i = 0; i < P::N; ++i) {
      float m0, m1, s0, s1, q0, q1;
      unpair(minus[i], m0, m1);
      unpair(s[i], s0, s1);
      unpair(q[i], q0, q1);
      channels[threadIdx.x * EPV + 2 * i] =
          make_float2(s0 * inv - m0, fmaxf(q0 - s0 * s0 * inv, 0.f));
      channels[threadIdx.x * EPV + 2 * i + 1] =
          make_float2(s1 * inv - m1, fmaxf(q1 - s1 * s1 * inv, 0.f));
    }
  } else {
    for (int col = me.tc; col < t.nvc; col += t.tcols) {
      const T* p = x + col * EPV;
      norm_rows<U>(t, me.tr, [&](auto count) {
        constexpr int K = decltype(count)::value;
        Raw<VB> w[K];
#pragma unroll
        for (int u = 0; u < K; ++u) w[u] = norm_ld<VB>(p + u * hop);
        p += K * hop;
        uint64_t s = 0, q = 0, off = 0;  // two zeros
#pragma unroll
        for (int u = 0; u < K; ++u) {
          uint64_t f[P::N];
          P::unpack(w[u], f);
          if (u == 0) off = norm_off<T, EPV>(f[0]);
#pragma unroll
          for (int i = 0; i < P::N; ++i)
            s = add2(s, sizeof(T) == 2 ? f[i] : add2(f[i], off));
        }
        float sa, sb;
        unpair(s, sa, sb);
        float cm = (sa + sb) * (1.f / (K * EPV));
        if (sizeof(T) == 4) cm += norm_first(off);
        // a single element's second half is no element
        const uint64_t minus = pair(-cm, EPV == 1 ? 0.f : -cm);
#pragma unroll
        for (int u = 0; u < K; ++u) {
          uint64_t f[P::N];
          P::unpack(w[u], f);
#pragma unroll
          for (int i = 0; i < P::N; ++i) {
            const uint64_t d = add2(f[i], minus);
            q = fma2(d, d, q);
          }
        }
        unpair(q, sa, sb);
        norm_join(n, mean, m2, K * EPV, cm, sa + sb);
      });
    }
    part[threadIdx.x] = make_float3(n, mean, m2);
  }
  __syncthreads();
  // `lanes` threads of a group join its threads' results
  int lanes = 32;
  while (lanes * t.groups > kNormThreads) lanes >>= 1;
  const int g = threadIdx.x / lanes, j = threadIdx.x & (lanes - 1);
  const bool on = g < t.groups;
  const int per = t.groups == 1 ? t.tcols : a.cg / EPV;  // columns of a group
  n = mean = m2 = 0.f;
  if (MIXED && on) {
    for (int k = j; k < a.cg * t.trows; k += lanes) {
      const int row = k / a.cg;
      const float2 o = channels[row * t.tcols * EPV + g * a.cg + (k - row * a.cg)];
      norm_join(n, mean, m2, static_cast<float>(max(0, (t.rows - row + t.trows - 1) / t.trows)),
                o.x, o.y);
    }
  } else if (on) {
    for (int k = j; k < per * t.trows; k += lanes) {
      const float3 o = part[k / per * t.tcols + g * per + k % per];
      norm_join(n, mean, m2, o.x, o.y, o.z);
    }
  }
  for (int d = 1; d < lanes; d <<= 1) {
    const float nb = __shfl_xor_sync(~0u, n, d), mb = __shfl_xor_sync(~0u, mean, d),
                sb = __shfl_xor_sync(~0u, m2, d);
    norm_join(n, mean, m2, nb, mb, sb);
  }
  auto finish = [&](float mu, float var) {
    if (on && j == 0) a.stats[me.seg_group + g] = make_float2(mu, rsqrtf(var + a.eps));
  };
  float2* const mine =
      a.partial + (t.block - static_cast<int64_t>(t.tile) * t.step) * a.partial_stride + g;
  const int64_t next_tile = static_cast<int64_t>(t.step) * a.partial_stride;
  if (on && j == 0) mine[t.tile * next_tile] = make_float2(mean, m2);
  if (DIRECT) return;
  norm_join_tiles(a, t, [&](int slot, int next, int count, int64_t full, int64_t tail,
                            bool final) {
    // the mean of the means, as what they lie off the first, then the deviations
    // from it
    const float nf = static_cast<float>(full) * a.cg, nt = static_cast<float>(tail) * a.cg;
    const float all = nf * (count - 1) + nt;
    const float2* q = mine + slot * next_tile;
    const float near = on ? __ldcg(&q->x) : 0.f;
    float mu = 0.f, dev = 0.f;
    if (on)
      for (int k = j; k < count; k += lanes)
        mu += (__ldcg(&q[k * next * next_tile].x) - near) * ((k + 1 < count ? nf : nt) / all);
    for (int d = 1; d < lanes; d <<= 1) mu += __shfl_xor_sync(~0u, mu, d);
    mu += near;
    if (on)
      for (int k = j; k < count; k += lanes) {
        const float2 o = __ldcg(q + k * next * next_tile);
        dev += o.y + (o.x - mu) * (o.x - mu) * (k + 1 < count ? nf : nt);
      }
    for (int d = 1; d < lanes; d <<= 1) dev += __shfl_xor_sync(~0u, dev, d);
    if (final) finish(mu, dev / all);
    else if (on && j == 0) mine[slot * next_tile] = make_float2(mu, dev);
  });
}

// A group's two values (of `values`, whose first is group g0's) for each of a
// vector's channels c0 ..., as pairs: once, or MIXED for each pair of channels.
enum NormOf { kNormMinusX, kNormMinusBoth };  // (-x, y), (-x, -y)

template <int EPV, bool MIXED, bool SHARED, NormOf OF>
__device__ __forceinline__ void norm_of_groups(const float2* values, int cg, int g0, int c0,
                                               uint64_t* x, uint64_t* y) {
  auto value = [&](int c) {
    // other CTAs' results are read in L2
    float2 p = SHARED ? values[c / cg - g0] : __ldcg(values + (c / cg - g0));
    p.x = -p.x;
    if (OF == kNormMinusBoth) p.y = -p.y;
    return p;
  };
#pragma unroll
  for (int i = 0; i < (MIXED ? EPV : 1); i += 2) {
    const float2 p = value(c0 + i), q = MIXED ? value(c0 + i + 1) : p;
    x[i / 2] = pair(p.x, q.x);
    y[i / 2] = pair(p.y, q.y);
  }
}

// A product of pairs outside the loop over rows.  A packed one the compiler moves
// into the loop (the xl backward's application 582 -> 655 us).
__device__ __forceinline__ uint64_t norm_times(uint64_t x, uint64_t y) {
  float a, b, c, d;
  unpair(x, a, b);
  unpair(y, c, d);
  return pair(a * c, b * d);
}

// A vector's x - mean, as pairs, and its 1 / sqrt(var + eps).  Everything here
// starts from x - mean, which is exact beside a mean of its own size, and takes
// the scale into what it is multiplied by: h = x * scale - (mean * scale) would
// be no fewer instructions and cost the digits of that product, 0.02 of h for
// 16-bit features that are all 1000, whose scale is 316.
template <int EPV, bool MIXED> struct NormCentre {
  static constexpr int N = MIXED ? EPV / 2 : 1;
  uint64_t minus[N], scale[N];
  __device__ __forceinline__ NormCentre(const float2* stats, int cg, int c0) {
    norm_of_groups<EPV, MIXED, false, kNormMinusX>(stats, cg, 0, c0, minus, scale);
  }
  __device__ __forceinline__ uint64_t operator()(uint64_t x, int i) const {
    return add2(x, minus[MIXED ? i : 0]);
  }
  // of a pair's values, times the scale
  __device__ __forceinline__ uint64_t scaled(uint64_t x, int i) const {
    return norm_times(x, scale[MIXED ? i : 0]);
  }
};

// The statistics of a tile's groups from its unit's partial results (direct):
// the mean of the means, as what they lie off the first, then the deviations
// from it.
__device__ __forceinline__ void norm_join_here(const NormArgs& a, const NormTile& t,
                                               const NormThread& me, float2* st) {
  const NormLevel& v = a.lv[t.l];
  int lanes = 32;
  while (lanes * t.groups > kNormThreads) lanes >>= 1;
  const int g = threadIdx.x / lanes, j = threadIdx.x & (lanes - 1);
  const bool on = g < t.groups;
  const float2* q =
      a.partial + (t.block - static_cast<int64_t>(t.tile) * t.step) * a.partial_stride + g;
  const int64_t next = static_cast<int64_t>(t.step) * a.partial_stride;
  const float full = static_cast<float>(v.tile_rows) * a.cg;
  const float tail =
      static_cast<float>(v.rows - static_cast<int64_t>(v.tiles - 1) * v.tile_rows) * a.cg;
  const float all = static_cast<float>(v.rows) * a.cg;
  const float near = on ? __ldcg(&q->x) : 0.f;
  float mu = 0.f, dev = 0.f;
  if (on) {
#pragma unroll 4
    for (int k = j; k < v.tiles; k += lanes)
      mu += (__ldcg(&q[k * next].x) - near) * ((k + 1 < v.tiles ? full : tail) / all);
  }
  for (int d = 1; d < lanes; d <<= 1) mu += __shfl_xor_sync(~0u, mu, d);
  mu += near;
  if (on) {
#pragma unroll 4
    for (int k = j; k < v.tiles; k += lanes) {
      const float2 o = __ldcg(q + k * next);
      dev += o.y + (o.x - mu) * (o.x - mu) * (k + 1 < v.tiles ? full : tail);
    }
  }
  for (int d = 1; d < lanes; d <<= 1) dev += __shfl_xor_sync(~0u, dev, d);
  if (on && j == 0) {
    st[g] = make_float2(mu, rsqrtf(dev / all + a.eps));
    if (t.tile == 0) a.stats[me.seg_group + g] = st[g];  // for the backward
  }
  __syncthreads();
}

template <typename T, int VB, int ACT, bool DIRECT, bool MIXED, int U>
__device__ void norm_apply(const NormArgs& a, const NormTile& t) {
  using P = Pairs<T, VB>;
  constexpr int EPV = P::EPV;
  __shared__ float2 joined[DIRECT ? kNormMaxSlab : 1];
  const NormLevel& v = a.lv[t.l];
  const NormThread me(a, t);
  if (DIRECT) norm_join_here(a, t, me, joined);
  const int64_t hop = t.trows * v.x_row, yhop = t.trows * v.out_row;
  for (int col = me.tc; col < t.nvc; col += t.tcols) {
    const int c0 = t.g0 * a.cg + col * EPV;
    constexpr int M = MIXED ? P::N : 1;  // pairs with statistics of their own
    uint64_t minus[M], r2[M];
    if (DIRECT)
      norm_of_groups<EPV, MIXED, true, kNormMinusX>(joined, a.cg, t.g0, c0, minus, r2);
    else
      norm_of_groups<EPV, MIXED, false, kNormMinusX>(a.stats + me.segment * a.G, a.cg, 0, c0,
                                                     minus, r2);
    float f[EPV];
    uint64_t w[P::N], d[P::N];
    const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0;
    norm_params<EPV>(a.weight, a.affine_dtype, at, 1.f, f);
    P::of(f, w);
    norm_params<EPV>(a.bias, a.affine_dtype, at, 0.f, f);
    P::of(f, d);
#pragma unroll
    for (int i = 0; i < P::N; ++i) {
      constexpr float k = norm_arg<ACT>;
      w[i] = norm_times(norm_times(w[i], r2[MIXED ? i : 0]), pair(k, k));
      d[i] = norm_times(d[i], pair(k, k));
    }
    const T* p =
        reinterpret_cast<const T*>(v.x) + v.x_batch * t.b + (t.row0 + me.tr) * v.x_row + c0;
    T* y = reinterpret_cast<T*>(v.out) + v.out_batch * t.b + (t.row0 + me.tr) * v.out_row + c0;
    norm_rows<U>(t, me.tr, [&](auto count) {
      constexpr int K = decltype(count)::value;
      Raw<VB> raw[K];
#pragma unroll
      for (int u = 0; u < K; ++u) raw[u] = norm_ld<VB>(p + u * hop);
      p += K * hop;
#pragma unroll
      for (int u = 0; u < K; ++u) {
        uint64_t e[P::N];
        P::unpack(raw[u], e);
#pragma unroll
        for (int i = 0; i < P::N; ++i)
          e[i] = norm_act<ACT>(fma2(add2(e[i], minus[MIXED ? i : 0]), w[i], d[i]));
        norm_st<VB>(y + u * yhop, P::pack(e));
      }
      y += K * yhop;
    });
  }
}

// A unit that is one tile, and no more than kNormOnceVectors vectors a thread.
// Of a pyramid of 1 360 x 256 in fp32, 7.0 us where two launches end after 10.5;
// a call takes 7.7 us of the host instead of 10.3.
template <typename T, int VB, int ACT>
__global__ void __launch_bounds__(kNormOnceThreads, 2)
norm_once_kernel(const __grid_constant__ NormArgs a) {
  using P = Pairs<T, VB>;
  constexpr int EPV = P::EPV, K = kNormOnceVectors;
  __shared__ float3 part[kNormOnceThreads];
  __shared__ float2 joined[kNormMaxSlab];
  const NormTile t = norm_tile<EPV, kNormOnceThreads>(a, blockIdx.x);
  const NormLevel& v = a.lv[t.l];
  const NormThread me(a, t);
  const int c0 = t.g0 * a.cg + me.tc * EPV;
  const T* p = reinterpret_cast<const T*>(v.x) + v.x_batch * t.b + me.tr * v.x_row + c0;
  const int64_t hop = t.trows * v.x_row, yhop = t.trows * v.out_row;
  const int mine = me.tr < t.rows ? (t.rows - me.tr + t.trows - 1) / t.trows : 0;
  Raw<VB> w[K];
#pragma unroll
  for (int u = 0; u < K; ++u)
    if (u < mine) w[u] = norm_ld<VB>(p + u * hop);
  float n = static_cast<float>(mine * EPV), mean = 0.f, m2 = 0.f;
  if (mine > 0) {
    uint64_t s = 0, q = 0, off = 0;  // two zeros
#pragma unroll
    for (int u = 0; u < K; ++u)
      if (u < mine) {
        uint64_t f[P::N];
        P::unpack(w[u], f);
        if (u == 0) off = norm_off<T, EPV>(f[0]);
#pragma unroll
        for (int i = 0; i < P::N; ++i) s = add2(s, sizeof(T) == 2 ? f[i] : add2(f[i], off));
      }
    float sa, sb;
    unpair(s, sa, sb);
    mean = (sa + sb) / n;
    if (sizeof(T) == 4) mean += norm_first(off);
    const uint64_t minus = pair(-mean, EPV == 1 ? 0.f : -mean);
#pragma unroll
    for (int u = 0; u < K; ++u)
      if (u < mine) {
        uint64_t f[P::N];
        P::unpack(w[u], f);
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
          const uint64_t d = add2(f[i], minus);
          q = fma2(d, d, q);
        }
      }
    unpair(q, sa, sb);
    m2 = sa + sb;
  }
  part[threadIdx.x] = make_float3(n, mean, m2);
  __syncthreads();
  int lanes = 32;
  while (lanes * t.groups > kNormOnceThreads) lanes >>= 1;
  const int g = threadIdx.x / lanes, j = threadIdx.x & (lanes - 1);
  const bool on = g < t.groups;
  const int per = a.cg / EPV;  // columns of a group
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
  if (on && j == 0) {
    joined[g] = make_float2(mean, rsqrtf(m2 / n + a.eps));
    a.stats[me.seg_group + g] = joined[g];
  }
  __syncthreads();
  if (mine == 0) return;
  const float2 st = joined[c0 / a.cg - t.g0];
  float f[EPV];
  uint64_t sc[P::N], d[P::N];
  const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0;
  norm_params<EPV>(a.weight, a.affine_dtype, at, 1.f, f);
  P::of(f, sc);
  norm_params<EPV>(a.bias, a.affine_dtype, at, 0.f, f);
  P::of(f, d);
  const uint64_t minus = pair(-st.x, -st.x), r2 = pair(st.y, st.y);
#pragma unroll
  for (int i = 0; i < P::N; ++i) {  // as norm_apply
    constexpr float k = norm_arg<ACT>;
    sc[i] = norm_times(norm_times(sc[i], r2), pair(k, k));
    d[i] = norm_times(d[i], pair(k, k));
  }
  T* y = reinterpret_cast<T*>(v.out) + v.out_batch * t.b + me.tr * v.out_row + c0;
#pragma unroll
  for (int u = 0; u < K; ++u)
    if (u < mine) {
      uint64_t e[P::N];
      P::unpack(w[u], e);
#pragma unroll
      for (int i = 0; i < P::N; ++i)
        e[i] = norm_act<ACT>(fma2(add2(e[i], minus), sc[i], d[i]));
      norm_st<VB>(y + u * yhop, P::pack(e));
    }
}

// ------------------------------------------------------------------ backward
// Rows of the sums' pass that a thread has on their way, in shared memory that
// it alone uses.  Two rows in registers, at three CTAs an SM, kept 49 KB in
// flight (566 us for the 2.45 GB of two 3D xl pyramids); this way four CTAs
// fit, with 96 KB: 418 us, 5.9 TB/s.  Then issue is the bound (16 instructions
// an element with SiLU).
constexpr int kNormStages = 4;

template <int AT> __device__ __forceinline__ void norm_copy(uint32_t shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1], 16;" ::"r"(shared), "l"(global), "n"(AT)
               : "memory");
}
template <int AT> __device__ __forceinline__ Raw<16> norm_staged(uint32_t shared) {
  Raw<16> r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
               : "r"(shared), "n"(AT) : "memory");
  return r;
}
// f(Count<0>) ... f(Count<N - 1>) until one returns false.
template <int I, int N, typename F> __device__ __forceinline__ bool norm_each(F f) {
  if constexpr (I == N) return true;
  else return f(Count<I>{}) && norm_each<I + 1, N>(f);
}
__device__ __forceinline__ void norm_copies_end() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void norm_copies_wait() {  // for all but the last kNormStages - 2
  asm volatile("cp.async.wait_group %0;" ::"n"(kNormStages - 2) : "memory");
}

// Sums s1, s2 per channel of one tile, and the groups' coefficients a, q of the unit.
template <typename T, int VB, int ACT, bool DIRECT, bool MIXED, int U>
__device__ void norm_grad_stats(const NormArgs& a, const NormTile& t) {
  using P = Pairs<T, VB>;
  constexpr int EPV = P::EPV;
  constexpr bool kStaged = VB == 16;
  __shared__ __align__(16) char space[kStaged ? kNormStages * 2 * kNormThreads * 16
                                              : kNormThreads * EPV * 8];
  float2* const part = reinterpret_cast<float2*>(space);
  const NormLevel& v = a.lv[t.l];
  const NormThread me(a, t);
  const int64_t hop = t.trows * v.x_row, ghop = t.trows * v.gy_row;
  float2* const mine = a.partial + static_cast<int64_t>(t.block) * a.partial_stride;
  for (int col0 = 0; col0 < t.nvc; col0 += t.tcols) {
    const int col = col0 + me.tc;
    uint64_t s1[P::N], s2[P::N];
#pragma unroll
    for (int i = 0; i < P::N; ++i) s1[i] = s2[i] = 0;  // two zeros
    if (kStaged && col0 > 0) __syncthreads();  // the sums before are read
    if (col < t.nvc) {
      const int c0 = t.g0 * a.cg + col * EPV;
      const NormCentre<EPV, MIXED> centre(a.stats + me.segment * a.G, a.cg, c0);
      uint64_t w[P::N], d[P::N];
      if (ACT != MSDA_ACT_NONE) {
        float f[EPV];
        const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0;
        norm_params<EPV>(a.weight, a.affine_dtype, at, 1.f, f);
        P::of(f, w);
#pragma unroll
        for (int i = 0; i < P::N; ++i) w[i] = centre.scaled(w[i], i);
        norm_params<EPV>(a.bias, a.affine_dtype, at, 0.f, f);
        P::of(f, d);
      }
      const T* p =
          reinterpret_cast<const T*>(v.x) + v.x_batch * t.b + (t.row0 + me.tr) * v.x_row + c0;
      const T* g =
          reinterpret_cast<const T*>(v.gy) + v.gy_batch * t.b + (t.row0 + me.tr) * v.gy_row + c0;
      auto add = [&](const Raw<VB>& rx, const Raw<VB>& rg) {
        uint64_t f[P::N], e[P::N];
        P::unpack(rx, f);
        P::unpack(rg, e);
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
          const uint64_t off = centre(f[i], i);
          const uint64_t dz =
              ACT == MSDA_ACT_NONE ? e[i] : mul2(e[i], norm_dact<ACT>(fma2(off, w[i], d[i])));
          s1[i] = add2(s1[i], dz);
          s2[i] = fma2(dz, off, s2[i]);  // scaled below
        }
      };
      if constexpr (kStaged) {
        constexpr int kStage = 2 * kNormThreads * 16;
        const uint32_t slot =
            static_cast<uint32_t>(__cvta_generic_to_shared(space)) + threadIdx.x * 16;
        int ahead = me.tr, r = me.tr;  // the rows to copy and to add next
        auto copy = [&](auto stage) {
          constexpr int kAt = decltype(stage)::value * kStage;
          if (ahead < t.rows) {
            norm_copy<kAt>(slot, p);
            norm_copy<kAt + kStage / 2>(slot, g);
            p += hop;
            g += ghop;
            ahead += t.trows;
          }
          norm_copies_end();
          return true;
        };
        norm_each<0, kNormStages - 1>(copy);
        while (norm_each<0, kNormStages>([&](auto stage) {
          constexpr int kNow = decltype(stage)::value;
          if (r >= t.rows) return false;
          norm_copies_wait();
          const Raw<16> rx = norm_staged<kNow * kStage>(slot);
          const Raw<16> rg = norm_staged<kNow * kStage + kStage / 2>(slot);
          copy(Count<(kNow + kNormStages - 1) % kNormStages>{});
          add(rx, rg);
          r += t.trows;
          return true;
        })) {
        }
      } else {
        norm_rows<U>(t, me.tr, [&](auto count) {
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
          for (int u = 0; u < K; ++u) add(rx[u], rg[u]);
        });
      }
#pragma unroll
      for (int i = 0; i < P::N; ++i) s2[i] = centre.scaled(s2[i], i);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P::N; ++i) {
      float a0, a1, b0, b1;
      unpair(s1[i], a0, a1);
      unpair(s2[i], b0, b1);
      part[threadIdx.x * EPV + 2 * i] = make_float2(a0, b0);
      if (2 * i + 1 < EPV) part[threadIdx.x * EPV + 2 * i + 1] = make_float2(a1, b1);
    }
    __syncthreads();
    const int cols = min(t.tcols, t.nvc - col0), row = t.tcols * EPV;
    for (int c = threadIdx.x; c < cols * EPV; c += kNormThreads) {
      float2 s = make_float2(0.f, 0.f);
      for (int k = 0; k < t.trows; ++k) {
        const float2 o = part[k * row + c];
        s.x += o.x;
        s.y += o.y;
      }
      mine[col0 * EPV + c] = s;
    }
  }
  const int cw = t.groups * a.cg, c0 = t.g0 * a.cg;
  // sums of a group's channels, from `s`, weighted
  auto group = [&](const float2* s, int g) {
    float2 sum = make_float2(0.f, 0.f);
    for (int i = 0; i < a.cg; ++i) {
      const int c = g * a.cg + i;
      float w;
      norm_params<1>(a.weight, a.affine_dtype,
                     static_cast<int64_t>(t.l) * a.affine_level + c0 + c, 1.f, &w);
      sum.x += w * s[c].x;
      sum.y += w * s[c].y;
    }
    return sum;
  };
  if (DIRECT) {
    __syncthreads();  // `mine` is written
    const int stride = a.lv[0].slab_groups;
    for (int g = threadIdx.x; g < t.groups; g += kNormThreads)
      a.weighted[static_cast<int64_t>(t.block) * stride + g] = group(mine, g);
    return;
  }
  float2* const first =
      a.partial + (t.block - static_cast<int64_t>(t.tile) * t.step) * a.partial_stride;
  const int64_t next_tile = static_cast<int64_t>(t.step) * a.partial_stride;
  float2* const chan = a.chan + me.seg_chan;
  norm_join_tiles(a, t, [&](int slot, int next, int count, int64_t, int64_t, bool final) {
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
          const float2 o = __ldcg(first + (slot + k * next) * next_tile + c);
          s.x += o.x;
          s.y += o.y;
        }
      }
      for (int d = 1; d < lanes; d <<= 1) {
        s.x += __shfl_xor_sync(~0u, s.x, d);
        s.y += __shfl_xor_sync(~0u, s.y, d);
      }
      if (c < cw && lane == 0) (final ? chan : first + slot * next_tile)[c] = s;
    }
    if (!final) return;
    __syncthreads();
    const float n = static_cast<float>(v.rows) * a.cg;
    for (int g = threadIdx.x; g < t.groups; g += kNormThreads) {
      const float2 sum = group(chan, g);
      a.coef[me.seg_group + g] = make_float2(sum.x / n, sum.y / n);
    }
  });
}

// The coefficients of a tile's groups from its unit's weighted sums (direct).
__device__ __forceinline__ void norm_grad_join_here(const NormArgs& a, const NormTile& t,
                                                    float2* co) {
  const NormLevel& v = a.lv[t.l];
  int lanes = 32;
  while (lanes * t.groups > kNormThreads) lanes >>= 1;
  const int g = threadIdx.x / lanes, j = threadIdx.x & (lanes - 1);
  const bool on = g < t.groups;
  const int stride = a.lv[0].slab_groups;
  const float2* q = a.weighted + (t.block - static_cast<int64_t>(t.tile) * t.step) * stride + g;
  const int64_t next = static_cast<int64_t>(t.step) * stride;
  float2 s = make_float2(0.f, 0.f);
  if (on) {
#pragma unroll 4
    for (int k = j; k < v.tiles; k += lanes) {
      const float2 o = __ldcg(q + k * next);
      s.x += o.x;
      s.y += o.y;
    }
  }
  for (int d = 1; d < lanes; d <<= 1) {
    s.x += __shfl_xor_sync(~0u, s.x, d);
    s.y += __shfl_xor_sync(~0u, s.y, d);
  }
  const float n = static_cast<float>(v.rows) * a.cg;
  if (on && j == 0) co[g] = make_float2(s.x / n, s.y / n);
  __syncthreads();
}

// Gradients of kNormParamChannels channels of the affine map, of one level or
// of all: a warp's worth of lanes a channel takes the batch entries' (direct:
// their tiles') sums in turn.
__device__ __forceinline__ void norm_param_grad(const NormArgs& a, int cta) {
  const int per_row = (a.C + kNormParamChannels - 1) / kNormParamChannels;
  const int row = cta / per_row;
  const int c =
      (cta - row * per_row) * kNormParamChannels + (threadIdx.x & (kNormParamChannels - 1));
  const int lane = threadIdx.x / kNormParamChannels;
  constexpr int kLanes = kNormThreads / kNormParamChannels;
  __shared__ float2 sums[kNormThreads];
  float2 s = make_float2(0.f, 0.f);
  auto add = [&](const float2& o) {
    s.x += o.x;
    s.y += o.y;
  };
  const int l0 = a.affine_level ? row : 0, l1 = a.affine_level ? row + 1 : a.L;
  if (c < a.C)
    for (int l = l0; l < l1; ++l) {
      const NormLevel& v = a.lv[l];
      if (v.rows == 0) continue;
      if (a.direct) {
        const int wide = v.slab_groups * a.cg, slab = c / wide, n = a.B * v.tiles;
        const float2* q = a.partial + static_cast<int64_t>(v.tile0 + slab) * a.partial_stride +
                          (c - slab * wide);
#pragma unroll 8
        for (int k = lane; k < n; k += kLanes)
          add(__ldcg(q + static_cast<int64_t>(k) * v.slabs * a.partial_stride));
      } else {
#pragma unroll 4
        for (int b = lane; b < a.B; b += kLanes)
          add(__ldcg(a.chan + (static_cast<int64_t>(b) * a.L + l) * a.C + c));
      }
    }
  sums[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x >= kNormParamChannels || c >= a.C) return;
  for (int k = 1; k < kLanes; ++k) add(sums[k * kNormParamChannels + threadIdx.x]);
  auto put = [&](void* out, float x) {
    const int64_t i = static_cast<int64_t>(row) * a.C + c;
    if (out == nullptr) return;
    if (a.affine_dtype == MSDA_FLOAT32) static_cast<float*>(out)[i] = x;
    else if (a.affine_dtype == MSDA_FLOAT16) static_cast<__half*>(out)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(x);
  };
  put(a.gweight, s.y);
  put(a.gbias, s.x);
}

template <typename T, int VB, int ACT, bool DIRECT, bool MIXED, int U>
__device__ void norm_grad_apply(const NormArgs& a, const NormTile& t) {
  using P = Pairs<T, VB>;
  constexpr int EPV = P::EPV;
  __shared__ float2 joined[DIRECT ? kNormMaxSlab : 1];
  const NormLevel& v = a.lv[t.l];
  const NormThread me(a, t);
  if (DIRECT) norm_grad_join_here(a, t, joined);
  const int64_t hop = t.trows * v.x_row, ghop = t.trows * v.gy_row, yhop = t.trows * v.out_row;
  for (int col = me.tc; col < t.nvc; col += t.tcols) {
    const int c0 = t.g0 * a.cg + col * EPV;
    const NormCentre<EPV, MIXED> centre(a.stats + me.segment * a.G, a.cg, c0);
    constexpr int M = MIXED ? P::N : 1;
    uint64_t ma[M], mq[M];
    if (DIRECT)
      norm_of_groups<EPV, MIXED, true, kNormMinusBoth>(joined, a.cg, t.g0, c0, ma, mq);
    else
      norm_of_groups<EPV, MIXED, false, kNormMinusBoth>(a.coef + me.segment * a.G, a.cg, 0, c0, ma,
                                                        mq);
    float f[EPV];
    uint64_t w[P::N], d[P::N];
    const int64_t at = static_cast<int64_t>(t.l) * a.affine_level + c0;
    norm_params<EPV>(a.weight, a.affine_dtype, at, 1.f, f);
    P::of(f, w);
#pragma unroll
    for (int i = 0; i < P::N; ++i) w[i] = centre.scaled(w[i], i);
#pragma unroll
    for (int k = 0; k < M; ++k) {
      ma[k] = centre.scaled(ma[k], k);
      mq[k] = centre.scaled(mq[k], k);
    }
    if (ACT != MSDA_ACT_NONE) {
      norm_params<EPV>(a.bias, a.affine_dtype, at, 0.f, f);
      P::of(f, d);
    }
    const T* p =
        reinterpret_cast<const T*>(v.x) + v.x_batch * t.b + (t.row0 + me.tr) * v.x_row + c0;
    const T* g =
        reinterpret_cast<const T*>(v.gy) + v.gy_batch * t.b + (t.row0 + me.tr) * v.gy_row + c0;
    T* y = reinterpret_cast<T*>(v.out) + v.out_batch * t.b + (t.row0 + me.tr) * v.out_row + c0;
    norm_rows<U>(t, me.tr, [&](auto count) {
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
        uint64_t x[P::N], e[P::N];
        P::unpack(rx[u], x);
        P::unpack(rg[u], e);
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
          const uint64_t off = centre(x[i], i);
          const uint64_t dz =
              ACT == MSDA_ACT_NONE ? e[i] : mul2(e[i], norm_dact<ACT>(fma2(off, w[i], d[i])));
          const int k = MIXED ? i : 0;
          const uint64_t h = mul2(off, centre.scale[k]);
          x[i] = fma2(dz, w[i], fma2(h, mq[k], ma[k]));
        }
        st_chunk<VB>(y + u * yhop, P::pack(x));
      }
      y += K * yhop;
    });
  }
}

// ------------------------------------------------------------------ the launches
// CTAs per SM and vectors in flight per thread: of the combinations that were
// timed (3 to 6 CTAs, 2 to 8 vectors) the fastest.  Two 3D xl pyramids, 1.23 GB
// of bf16 with SiLU: statistics 202 us (6.1 TB/s) and application 382 us
// (6.4 TB/s) forward, 418 us (5.9) and 585 us (6.3) backward.
template <typename T, int VB, int ACT, bool BWD, bool DIRECT, bool MIXED>
__global__ void __launch_bounds__(kNormThreads, BWD && (MIXED || VB < 16) ? 3 : 4)
norm_stats_kernel(const __grid_constant__ NormArgs a) {
  norm_let_next_start();
  const NormTile t = norm_tile<Chunk<T, VB>::EPV>(a, blockIdx.x);
  if (BWD) norm_grad_stats<T, VB, ACT, DIRECT, MIXED, 2>(a, t);
  else norm_stats<T, VB, DIRECT, MIXED, 8>(a, t);
}

template <typename T, int VB, int ACT, bool BWD, bool DIRECT, bool MIXED>
__global__ void __launch_bounds__(kNormThreads, (BWD ? 3 : 4) - MIXED)
norm_apply_kernel(const __grid_constant__ NormArgs a) {
  const int block = static_cast<int>(blockIdx.x) - a.param_ctas;
  if (BWD && block < 0) {
    norm_wait_previous();
    norm_param_grad(a, blockIdx.x);
    return;
  }
  const NormTile t = norm_tile<Chunk<T, VB>::EPV>(a, a.tiles - 1 - block);
  norm_wait_previous();
  if (BWD) norm_grad_apply<T, VB, ACT, DIRECT, MIXED, 2>(a, t);
  else norm_apply<T, VB, ACT, DIRECT, MIXED, 4>(a, t);
}

template <typename T, int VB, int ACT, bool BWD, bool DIRECT, bool MIXED>
cudaError_t norm_launch_one(const NormArgs& a, cudaStream_t st) {
  // the forward's statistics are the same for every activation
  constexpr int kAct = BWD ? ACT : MSDA_ACT_NONE;
  if (a.tiles > 0) {
    norm_stats_kernel<T, VB, kAct, BWD, DIRECT, MIXED><<<a.tiles, kNormThreads, 0, st>>>(a);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return err;
  }
  if (a.tiles + a.param_ctas == 0) return cudaSuccess;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.tiles + a.param_ctas);
  cfg.blockDim = dim3(kNormThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = a.tiles > 0 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, norm_apply_kernel<T, VB, ACT, BWD, DIRECT, MIXED>, a);
}

template <typename T, int VB, bool MIXED>
cudaError_t norm_launch_act(const NormArgs& a, int act, bool backward, bool once,
                            cudaStream_t st) {
  switch (act) {
#define MSDA_NORM_ACT(ACT)                                                              \
  case ACT:                                                                             \
    if constexpr (!MIXED)                                                               \
      if (once) {                                                                       \
        norm_once_kernel<T, VB, ACT><<<a.tiles, kNormOnceThreads, 0, st>>>(a);          \
        return cudaGetLastError();                                                      \
      }                                                                                 \
    if (a.direct)                                                                       \
      return backward ? norm_launch_one<T, VB, ACT, true, true, MIXED>(a, st)           \
                      : norm_launch_one<T, VB, ACT, false, true, MIXED>(a, st);         \
    return backward ? norm_launch_one<T, VB, ACT, true, false, MIXED>(a, st)            \
                    : norm_launch_one<T, VB, ACT, false, false, MIXED>(a, st);
    MSDA_NORM_ACT(MSDA_ACT_RELU)
    MSDA_NORM_ACT(MSDA_ACT_SILU)
    MSDA_NORM_ACT(MSDA_ACT_GELU)
    MSDA_NORM_ACT(MSDA_ACT_NONE)
#undef MSDA_NORM_ACT
  }
  return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t norm_launch(const NormArgs& a, int vb, bool mixed, int act, bool backward, bool once,
                        cudaStream_t st) {
  if (mixed) return norm_launch_act<T, 16, true>(a, act, backward, once, st);
  switch (vb) {
    case 16: return norm_launch_act<T, 16, false>(a, act, backward, once, st);
    case 8: return norm_launch_act<T, 8, false>(a, act, backward, once, st);
    case 4: return norm_launch_act<T, 4, false>(a, act, backward, once, st);
    default:
      if constexpr (sizeof(T) == 2)
        return norm_launch_act<T, 2, false>(a, act, backward, once, st);
      return cudaErrorInvalidValue;
  }
}

}  // namespace msda
