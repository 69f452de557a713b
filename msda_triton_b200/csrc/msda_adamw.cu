// msda_adamw.cu -- one AdamW step over many tensors in one launch, with the
// two moments in fp32 or in 8 bits.
//
//   g' = s g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32, the parameter rounded once to its type (from an fp32 master copy,
// if there is one).  With fp32 moments it is bound by memory: 28 bytes a
// parameter in fp32 (22 in bf16), 335 M of them in 1.35 ms (1.07 ms), 6.9 TB/s.
// With 8-bit moments and bf16 parameters, 10 bytes a parameter, the coding is:
// about 73 instructions a parameter, half of them on the integer units that are
// 74 % busy, 0.82 ms for 335 M (4.1 TB/s; fp32 parameters 1.00 ms, 5.4 TB/s).
//
// States of all tensors lie in one array each; tensor i's elements start at
// the sum of the earlier tensors' sizes, each rounded up to kBlock.
//
// 8-bit moments.  A block of kBlock = 128 elements shares an exponent byte E.
// With the fp32 bits b of a magnitude, its code is (b >> 20) - 8 (E - top): a
// float of 3 mantissa bits whose exponent counts down from the block's. The
// second moment takes 5 exponent bits (top = 31, a range of 2^31), the first
// its sign and 4 (top = 15).  E is the largest magnitude's exponent after it
// is rounded up by one code more than it can be, so the highest code is never
// reached by rounding; it stands for a value that is not finite.
//
// Moments are rounded at random, up with the probability of the part cut off:
// a change of 0.1 % a step (b2 = 0.999) is far below the spacing of 12.5 %, and
// rounding to the nearest code would freeze the second moment where it is.
// The random bits are a mixed counter of the element's index, the seed and the
// step, so a step can be repeated.
//
// Below the lowest code, 1.125 x 2^-15 or 2^-31 of the power of two that holds
// the block's largest, rounding is not random.  A first moment becomes zero: an
// element whose gradients stay that far below a neighbour's keeps no momentum,
// and its update is about 1 - b1 of what it would be.  A second moment above
// zero takes the lowest code: decoded as zero it would divide by eps alone.
//
// A warp takes a block, a lane four neighbouring elements: 16-byte (8-byte)
// accesses of fp32 (16-bit) parameters and whole 128-byte lines of codes, and
// the block's maximum is one redux instruction.  Tensors are listed in the
// kernel's own parameters: no copy to the device precedes the launch.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "msda_common.cuh"
#include "msda_f32x2.cuh"
#include "msda_status.cuh"

namespace msda {
namespace {

constexpr int kAdamThreads = 256;
constexpr int kBlock = 128;                                 // elements per exponent
constexpr int kAdamUnroll = 4;                              // blocks per warp
constexpr int kChunk = kAdamThreads / 32 * kBlock * kAdamUnroll;  // elements per CTA
constexpr int kFewTensors = 64, kManyTensors = 640;  // per launch: 4 KB, 32 KB of parameters

struct AdamTensor {
  void* p;
  const void* g;
  int64_t n;
  float step_size, inv_sqrt_bc2;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  uint32_t key;
  uint32_t offset;  // of its states, in blocks
  uint32_t cta0;    // first CTA of the launch
};

struct AdamArgs {
  // m = k m + c (g - l m): with l = k = 1 (b >= 1/2), only c's share of the
  // rounding of c and of the difference reaches m; with a small b that share is
  // most of m, and l = 0, k = b
  float c1, k1, l1, c2, k2, l2;  // c = 1 - b; l negated
  float eps, decay;              // decay = 1 - lr wd
  const float* grad_scale;
  void *m, *v;
  uint8_t *me, *ve;
  float* master;
};

// A CTA looks for its tensor among those of its part of the grid.  By a search
// over all tensors this cost seven instructions an element, which two rounds of
// elements a CTA would have halved; the loop over rounds then cost more than the
// search (335 M bf16 parameters, 8 bits: 875 us against 818).
constexpr int kAdamParts = 64;

template <int N> struct AdamTable {
  AdamArgs a;
  int32_t part_shift;              // of a CTA's index
  uint16_t first[kAdamParts + 1];  // tensor of each part's first CTA
  AdamTensor t[N];
};

constexpr uint32_t kMaxFinite = 0x7f7fffffu;

// A lane's four first and four second moments.  Zero stays zero.  The highest
// code, which is no number, is rare: whether there is one is tested for all
// eight codes at once.
__device__ __forceinline__ void adam_decode(uint32_t wm, uint32_t wv, uint32_t em, uint32_t ev,
                                            float* m, float* v) {
  const uint32_t sm = (em - 15u) << 23, sv = (ev - 31u) << 23;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t top = wm << (24 - 8 * i);
    uint32_t x = top >> 4 & 0x07f00000u;
    if (x != 0u) x += sm;
    m[i] = __uint_as_float(x | (top & 0x80000000u));
    uint32_t y = (i < 3 ? wv << (20 - 8 * i) : wv >> 4) & 0x0ff00000u;
    if (y != 0u) y += sv;
    v[i] = __uint_as_float(y);
  }
  constexpr uint32_t kOnes = 0x01010101u;
  const uint32_t odd = ((wm & 0x7f7f7f7fu) + kOnes) | (~(wv + kOnes) & wv);
  if ((odd & 0x80808080u) == 0u) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((wm >> (8 * i) & 127u) == 127u) m[i] = __uint_as_float(0x7fc00000u);
    if ((wv >> (8 * i) & 255u) == 255u) v[i] = __uint_as_float(0x7fc00000u);
  }
}

// Four values as codes where some are not finite, or at the end of the range.
template <uint32_t TOP, bool SIGNED>
__device__ __noinline__ uint32_t adam_encode_odd(float4 x, uint4 r, uint32_t& e) {
  constexpr uint32_t kTopCode = SIGNED ? 127u : 255u;
  const float f[4] = {x.x, x.y, x.z, x.w};
  const uint32_t rnd[4] = {r.x, r.y, r.z, r.w};
  uint32_t most = 0u;
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
    if (b <= kMaxFinite) most = max(most, b);
  }
  most = __reduce_max_sync(~0u, most);
  e = max((most + 0x1fffffu) >> 23, TOP);
  const int base = static_cast<int>(e - TOP) << 3;
  uint32_t word = 0u;
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __float_as_uint(f[i]) & 0x7fffffffu;
    int c = static_cast<int>(min(b + rnd[i] * 16u + 8u, kMaxFinite) >> 20) - base;
    c = max(c, !SIGNED && b != 0u ? 1 : 0);
    if (b > kMaxFinite) c = kTopCode;
    if (SIGNED) c |= __float_as_uint(f[i]) >> 24 & 128u;
    word |= static_cast<uint32_t>(c) << (8 * i);
  }
  return word;
}

// The codes of four values per lane; `r` holds 16 random bits each, which with
// a set bit below them are the upper 17 of the 20 that are added.
template <uint32_t TOP, bool SIGNED>
__device__ __forceinline__ uint32_t adam_encode(const float* x, const uint32_t* r, uint32_t& e) {
  uint32_t b[4], most = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    b[i] = __float_as_uint(x[i]);
    if (SIGNED) b[i] &= 0x7fffffffu;
    most = max(most, b[i]);
  }
  most = __reduce_max_sync(~0u, most);
  if (most > kMaxFinite - 0x1fffffu)
    return adam_encode_odd<TOP, SIGNED>(make_float4(x[0], x[1], x[2], x[3]),
                                        make_uint4(r[0], r[1], r[2], r[3]), e);
  e = max((most + 0x1fffffu) >> 23, TOP);
  const int less = 8 - static_cast<int>((e - TOP) << 23);
  uint32_t c[4];  // a code's byte on top
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int least = SIGNED ? 0 : static_cast<int>(min(b[i], 1u) << 20);
    c[i] = static_cast<uint32_t>(max(static_cast<int>(r[i] * 16u + b[i]) + less, least)) << 4;
    if (SIGNED) c[i] = (c[i] & 0x7fffffffu) | (__float_as_uint(x[i]) & 0x80000000u);
  }
  return __byte_perm(__byte_perm(c[0], c[1], 0x73), __byte_perm(c[2], c[3], 0x73), 0x5410);
}

// A counter times an odd constant, mixed by shifts and products.  The constants
// are the first three primes of the published 32-bit hash xxHash (Y. Collet).
__device__ __forceinline__ uint32_t adam_random(uint32_t index, uint32_t key) {
  uint32_t x = index * 0x9e3779b1u + key;
  x = (x ^ (x >> 16)) * 0x85ebca77u;
  x = (x ^ (x >> 13)) * 0xc2b2ae3du;
  return x ^ (x >> 16);
}

// Four elements; those of index `valid` and up are not there.
template <typename T>
__device__ __forceinline__ Raw<4 * sizeof(T)> adam_load(const T* p, int valid, bool vec) {
  Raw<4 * sizeof(T)> w;
  if (vec && valid == 4) {
    if constexpr (sizeof(T) == 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(p);
      w.w[0] = q.x; w.w[1] = q.y; w.w[2] = q.z; w.w[3] = q.w;
    } else {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      w.w[0] = q.x; w.w[1] = q.y;
    }
  } else {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = i < valid ? Elem<T>::to_f(p[i]) : 0.f;
    w = Chunk<T, 4 * sizeof(T)>::pack(f);
  }
  return w;
}
template <typename T>
__device__ __forceinline__ void adam_store(T* p, int valid, bool vec, const float* f) {
  if (vec && valid == 4) {
    st_chunk<4 * sizeof(T)>(p, Chunk<T, 4 * sizeof(T)>::pack(f));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) p[i] = Elem<T>::from_f(f[i]);
  }
}

// The root of at least the smallest normal number (below it the unit's result
// would be zero), and a NaN's.
__device__ __forceinline__ float adam_sqrt(float x) {
  float y;
  asm("{\n .reg .f32 t;\n max.NaN.f32 t, %1, 0f00800000;\n sqrt.approx.ftz.f32 %0, t;\n}"
      : "=f"(y) : "f"(x));
  return y;
}
// x is no less than such a root times a factor above 1/2: never subnormal.
__device__ __forceinline__ float adam_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T, bool SMALL, bool MASTER, int N>
__global__ void __launch_bounds__(kAdamThreads)
adamw_kernel(const __grid_constant__ AdamTable<N> tab) {
  constexpr int U = kAdamUnroll;
  const AdamArgs& a = tab.a;
  // the last tensor whose first CTA is not after this one
  const int part = blockIdx.x >> tab.part_shift;
  int lo = tab.first[part], hi = tab.first[part + 1] + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].cta0 <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const AdamTensor& t = tab.t[lo];
  const int lane = threadIdx.x & 31;
  const float scale = a.grad_scale == nullptr ? 1.f : __ldg(a.grad_scale);
  const uint64_t gs = pair(scale, scale), c1 = pair(a.c1, a.c1), k1 = pair(a.k1, a.k1),
                 l1 = pair(a.l1, a.l1), c2 = pair(a.c2, a.c2), k2 = pair(a.k2, a.k2),
                 l2 = pair(a.l2, a.l2), bc = pair(t.inv_sqrt_bc2, t.inv_sqrt_bc2),
                 eps = pair(a.eps, a.eps), decay = pair(a.decay, a.decay),
                 size = pair(-t.step_size, -t.step_size);
  const bool vec = (reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g)) %
                       (4 * sizeof(T)) == 0;

  const int64_t first =
      static_cast<int64_t>(blockIdx.x - t.cta0) * kChunk +
      (threadIdx.x >> 5) * (kBlock * U) + lane * 4;
  // elements from this lane's first one to the tensor's end
  const int left = static_cast<int>(max(min(t.n - first, static_cast<int64_t>(kChunk)),
                                        -static_cast<int64_t>(kChunk)));
  if (left + lane * 4 <= 0) return;  // the whole warp
  T* p = static_cast<T*>(t.p) + first;
  const T* g = static_cast<const T*>(t.g) + first;
  const int64_t s0 = static_cast<int64_t>(t.offset) * kBlock + first;
  float* const master = a.master + s0;
  uint8_t* const m8 = static_cast<uint8_t*>(a.m) + s0;
  uint8_t* const v8 = static_cast<uint8_t*>(a.v) + s0;
  uint8_t *const me = a.me + s0 / kBlock, *const ve = a.ve + s0 / kBlock;
  float *const m32 = static_cast<float*>(a.m) + s0, *const v32 = static_cast<float*>(a.v) + s0;

  // everything is on its way before the first use
  Raw<4 * sizeof(T)> rg[U], rp[U];
  Raw<16> rx[U], rm[U], rv[U];
  uint32_t cm[U], cv[U], em[U], ev[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int valid = left - u * kBlock;
    if (valid + lane * 4 <= 0) continue;  // the whole warp: a block that is not there
    rg[u] = adam_load(g + u * kBlock, min(valid, 4), vec);
    if (MASTER) rx[u] = adam_load(master + u * kBlock, 4, true);
    else rp[u] = adam_load(p + u * kBlock, min(valid, 4), vec);
    if (SMALL) {
      cm[u] = *reinterpret_cast<const uint32_t*>(m8 + u * kBlock);
      cv[u] = *reinterpret_cast<const uint32_t*>(v8 + u * kBlock);
      em[u] = me[u];
      ev[u] = ve[u];
    } else {
      rm[u] = adam_load(m32 + u * kBlock, 4, true);
      rv[u] = adam_load(v32 + u * kBlock, 4, true);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int valid = left - u * kBlock;
    if (valid + lane * 4 <= 0) return;
    float x[4], d[4], m[4], v[4];
    Chunk<T, 4 * sizeof(T)>::unpack(rg[u], d);
    if (MASTER) Chunk<float, 16>::unpack(rx[u], x);
    else Chunk<T, 4 * sizeof(T)>::unpack(rp[u], x);
    if (SMALL) {
      adam_decode(cm[u], cv[u], em[u], ev[u], m, v);
    } else {
      Chunk<float, 16>::unpack(rm[u], m);
      Chunk<float, 16>::unpack(rv[u], v);
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      uint64_t e = mul2(pair(d[i], d[i + 1]), gs);
      uint64_t mm = pair(m[i], m[i + 1]), vv = pair(v[i], v[i + 1]);
      mm = fma2(c1, fma2(l1, mm, e), mul2(k1, mm));
      e = mul2(e, e);
      vv = fma2(c2, fma2(l2, vv, e), mul2(k2, vv));
      unpair(mm, m[i], m[i + 1]);
      unpair(vv, v[i], v[i + 1]);
      float den[2];
      unpair(fma2(pair(adam_sqrt(v[i]), adam_sqrt(v[i + 1])), bc, eps), den[0], den[1]);
      const uint64_t q = mul2(mm, pair(adam_rcp(den[0]), adam_rcp(den[1])));
      unpair(fma2(size, q, mul2(decay, pair(x[i], x[i + 1]))), x[i], x[i + 1]);
    }
    if (valid < 4) {  // between tensors
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i >= valid) m[i] = v[i] = x[i] = 0.f;
    }
    adam_store(p + u * kBlock, min(valid, 4), vec, x);
    if (MASTER) adam_store(master + u * kBlock, 4, true, x);
    if (SMALL) {
      uint32_t qm[4], qv[4], nm, nv;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t r = adam_random(static_cast<uint32_t>(s0) + u * kBlock + i, t.key);
        qm[i] = r & 0xffffu;
        qv[i] = r >> 16;
      }
      const uint32_t wm = adam_encode<15u, true>(m, qm, nm);
      const uint32_t wv = adam_encode<31u, false>(v, qv, nv);
      *reinterpret_cast<uint32_t*>(m8 + u * kBlock) = wm;
      *reinterpret_cast<uint32_t*>(v8 + u * kBlock) = wv;
      if (lane == 0) {
        me[u] = static_cast<uint8_t>(nm);
        ve[u] = static_cast<uint8_t>(nv);
      }
    } else {
      adam_store(m32 + u * kBlock, 4, true, m);
      adam_store(v32 + u * kBlock, 4, true, v);
    }
  }
}

// The values that 8-bit moments stand for; bf16 holds them exactly.
__global__ void __launch_bounds__(kAdamThreads)
adamw_values_kernel(const uint8_t* m, const uint8_t* me, const uint8_t* v, const uint8_t* ve,
                    int64_t n, __nv_bfloat16* mo, __nv_bfloat16* vo) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * kAdamThreads + threadIdx.x) * 8;
  if (i >= n) return;
  const uint2 cm = __ldg(reinterpret_cast<const uint2*>(m + i));
  const uint2 cv = __ldg(reinterpret_cast<const uint2*>(v + i));
  const uint32_t em = __ldg(me + i / kBlock), ev = __ldg(ve + i / kBlock);
  float fm[8], fv[8];
  adam_decode(cm.x, cv.x, em, ev, fm, fv);
  adam_decode(cm.y, cv.y, em, ev, fm + 4, fv + 4);
  st_chunk<16>(mo + i, Chunk<__nv_bfloat16, 16>::pack(fm));
  st_chunk<16>(vo + i, Chunk<__nv_bfloat16, 16>::pack(fv));
}

template <typename T, int N>
cudaError_t adamw_launch(const AdamTable<N>& tab, bool small, unsigned int grid, cudaStream_t st) {
  if (tab.a.master != nullptr) {
    if constexpr (sizeof(T) == 2) {
      if (small) adamw_kernel<T, true, true, N><<<grid, kAdamThreads, 0, st>>>(tab);
      else adamw_kernel<T, false, true, N><<<grid, kAdamThreads, 0, st>>>(tab);
    }
  } else {
    if (small) adamw_kernel<T, true, false, N><<<grid, kAdamThreads, 0, st>>>(tab);
    else adamw_kernel<T, false, false, N><<<grid, kAdamThreads, 0, st>>>(tab);
  }
  return cudaGetLastError();
}

struct Step {
  int dtype;
  bool small;
  int64_t tensors;
  void* const* params;
  const void* const* grads;
  const int64_t *counts, *steps;
  double lr, b1, b2;
  uint32_t seed;
};

template <int N> cudaError_t adamw_all(const Step& s, const AdamArgs& args, cudaStream_t st) {
  AdamTable<N> tab;
  tab.a = args;
  int used = 0;
  int64_t chunks = 0, offset = 0, known = -1;
  float step_size = 0.f, inv_sqrt_bc2 = 0.f;
  auto flush = [&]() {
    if (used == 0) return cudaSuccess;
    const unsigned int grid = static_cast<unsigned int>(chunks);
    tab.part_shift = 0;
    while ((grid - 1) >> tab.part_shift >= kAdamParts) ++tab.part_shift;
    for (int part = 0, i = 0; part <= kAdamParts; ++part) {
      while (i + 1 < used && tab.t[i + 1].cta0 <= static_cast<uint64_t>(part) << tab.part_shift)
        ++i;
      tab.first[part] = static_cast<uint16_t>(i);
    }
    used = 0;
    chunks = 0;
    if (s.dtype == MSDA_FLOAT32) return adamw_launch<float, N>(tab, s.small, grid, st);
    if (s.dtype == MSDA_FLOAT16) return adamw_launch<__half, N>(tab, s.small, grid, st);
    return adamw_launch<__nv_bfloat16, N>(tab, s.small, grid, st);
  };
  for (int64_t i = 0; i < s.tensors; ++i) {
    const int64_t n = s.counts[i], at = offset;
    offset += (n + kBlock - 1) / kBlock * kBlock;
    if (n == 0 || s.grads[i] == nullptr) continue;
    if (s.steps[i] != known) {
      known = s.steps[i];
      const double t = static_cast<double>(known);
      step_size = static_cast<float>(s.lr / (1.0 - std::pow(s.b1, t)));
      inv_sqrt_bc2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(s.b2, t)));
    }
    const int64_t own = (n + kChunk - 1) / kChunk;
    if (used == N || chunks + own > 0x7fffffff) {
      const cudaError_t err = flush();
      if (err != cudaSuccess) return err;
    }
    tab.t[used++] = AdamTensor{s.params[i], s.grads[i], n, step_size, inv_sqrt_bc2,
                               s.seed + static_cast<uint32_t>(known) * 0x632be5abu,
                               static_cast<uint32_t>(at / kBlock), static_cast<uint32_t>(chunks)};
    chunks += own;
  }
  return flush();
}

}  // namespace
}  // namespace msda

using namespace msda;

int msda_adamw_step(int dtype, int state_bits, int64_t num_tensors, void* const* params,
                    const void* const* grads, const int64_t* counts, const int64_t* steps,
                    double lr, double beta1, double beta2, double eps, double weight_decay,
                    uint32_t seed, const float* grad_scale, void* exp_avg, void* exp_avg_sq,
                    uint8_t* exp_avg_exponent, uint8_t* exp_avg_sq_exponent, float* master,
                    int64_t state_elements, void* stream) {
  const int64_t es = elem_bytes(dtype);
  if (es == 0) return report(MSDA_ERROR_UNSUPPORTED_DTYPE, "AdamW supports fp32, fp16 and bf16");
  if (state_bits != 32 && state_bits != 8)
    return report(MSDA_ERROR_INVALID_ARGUMENT, "states of 32 or 8 bits expected, got %d",
                  state_bits);
  if (master != nullptr && dtype == MSDA_FLOAT32)
    return report(MSDA_ERROR_INVALID_ARGUMENT, "fp32 parameters take no master copy");
  if (num_tensors < 0 || (num_tensors > 0 && (params == nullptr || grads == nullptr ||
                                              counts == nullptr || steps == nullptr)))
    return report(MSDA_ERROR_INVALID_ARGUMENT, "NULL tensor table");
  if (!(lr >= 0) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) ||
      !(weight_decay >= 0))
    return report(MSDA_ERROR_INVALID_ARGUMENT,
                  "lr, eps and weight_decay must not be negative, betas lie in [0, 1)");
  int64_t total = 0;
  for (int64_t i = 0; i < num_tensors; ++i) {
    if (counts[i] < 0 || counts[i] > (int64_t{1} << 40) || steps[i] < 1)
      return report(MSDA_ERROR_INVALID_ARGUMENT, "tensor %lld: bad size or step (from 1)",
                    static_cast<long long>(i));
    total += (counts[i] + kBlock - 1) / kBlock * kBlock;
    if (counts[i] > 0 && grads[i] != nullptr &&
        (params[i] == nullptr || !is_aligned(params[i], es) || !is_aligned(grads[i], es)))
      return report(MSDA_ERROR_MISALIGNED, "tensor %lld: NULL or unaligned",
                    static_cast<long long>(i));
  }
  if (state_elements < total)
    return report(MSDA_ERROR_SHAPE_MISMATCH, "states of %lld elements where %lld are needed",
                  static_cast<long long>(state_elements), static_cast<long long>(total));
  if (total == 0) return report_ok();
  const bool small = state_bits == 8;
  if (exp_avg == nullptr || exp_avg_sq == nullptr || !is_aligned(exp_avg, 16) ||
      !is_aligned(exp_avg_sq, 16) || !is_aligned(master, 16) || !is_aligned(grad_scale, 4) ||
      (small && (exp_avg_exponent == nullptr || exp_avg_sq_exponent == nullptr)))
    return report(MSDA_ERROR_MISALIGNED, "NULL or unaligned state");
  AdamArgs a{};
  a.c1 = static_cast<float>(1.0 - beta1);
  a.k1 = beta1 < 0.5 ? static_cast<float>(beta1) : 1.f;
  a.l1 = beta1 < 0.5 ? 0.f : -1.f;
  a.c2 = static_cast<float>(1.0 - beta2);
  a.k2 = beta2 < 0.5 ? static_cast<float>(beta2) : 1.f;
  a.l2 = beta2 < 0.5 ? 0.f : -1.f;
  a.eps = static_cast<float>(eps);
  a.decay = static_cast<float>(1.0 - lr * weight_decay);
  a.grad_scale = grad_scale;
  a.m = exp_avg;
  a.v = exp_avg_sq;
  a.me = exp_avg_exponent;
  a.ve = exp_avg_sq_exponent;
  a.master = master;
  const Step s{dtype, small, num_tensors, params, grads, counts, steps, lr, beta1, beta2, seed};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // a launch copies its parameters: the short table where it is enough
  return report_cuda(num_tensors <= kFewTensors ? adamw_all<kFewTensors>(s, a, st)
                                                : adamw_all<kManyTensors>(s, a, st),
                     "AdamW launch");
}

int msda_adamw_values(const uint8_t* exp_avg, const uint8_t* exp_avg_exponent,
                      const uint8_t* exp_avg_sq, const uint8_t* exp_avg_sq_exponent,
                      int64_t state_elements, void* exp_avg_values, void* exp_avg_sq_values,
                      void* stream) {
  if (state_elements < 0 || state_elements % kBlock != 0)
    return report(MSDA_ERROR_INVALID_ARGUMENT, "state_elements must be a multiple of %d", kBlock);
  if (state_elements == 0) return report_ok();
  if (exp_avg_exponent == nullptr || exp_avg_sq_exponent == nullptr)
    return report(MSDA_ERROR_MISALIGNED, "NULL state");
  for (const void* p : {static_cast<const void*>(exp_avg), static_cast<const void*>(exp_avg_sq),
                        static_cast<const void*>(exp_avg_values),
                        static_cast<const void*>(exp_avg_sq_values)})
    if (p == nullptr || !is_aligned(p, 16))
      return report(MSDA_ERROR_MISALIGNED, "NULL or unaligned state");
  const int64_t grid = (state_elements / 8 + kAdamThreads - 1) / kAdamThreads;
  if (grid > 0x7fffffff)
    return report(MSDA_ERROR_INT32_OVERFLOW, "too many elements for one launch");
  adamw_values_kernel<<<static_cast<unsigned int>(grid), kAdamThreads, 0,
                        static_cast<cudaStream_t>(stream)>>>(
      exp_avg, exp_avg_exponent, exp_avg_sq, exp_avg_sq_exponent, state_elements,
      static_cast<__nv_bfloat16*>(exp_avg_values), static_cast<__nv_bfloat16*>(exp_avg_sq_values));
  return report_cuda(cudaGetLastError(), "AdamW values launch");
}
