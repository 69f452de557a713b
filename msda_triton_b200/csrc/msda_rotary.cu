// msda_rotary.cu -- rotary positions on several axes, applied to one or two
// tensors of heads (queries and keys) in one launch; the same kernel turns the
// output gradients back, and can form the positions' gradient on the way.
//
// Pair j of a head's first 2P channels -- (j, j + P), or (2j, 2j + 1) with
// interleaved pairs -- turns by the angle  th_j = position[axis_j] * f_j:
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin
// and the gradient by its negative.  d y / d th is y turned by a quarter, so
//   gpos[a] = sum over heads and the pairs on axis a of  f_j (x1 gx2 - x2 gx1).
//
// Bound by memory: 2 bytes moved per byte of input, 6 flops a pair.  The
// angles are the same for every head, so a CTA takes some tokens, turns their
// P angles into (cos, sin) in shared memory once, and its threads then walk
// all heads' vectors in memory order.  The first vectors are loaded before the
// angles are computed.
//
// The angle is formed in half turns as a pair of floats, th / pi = u + v, and
// reduced by the nearest even integer, which is exact; cospi and sinpi take
// the rest.  An angle of 10^5 radians is then as exact as a small one, where
// an fp32 product alone would be 0.004 off.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "msda_common.cuh"
#include "msda_status.cuh"

namespace msda {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotPairs = 2048;  // (token, pair) angles of a CTA
constexpr int kRotUnits = 1024;  // vectors of a CTA's tokens, unless one has more
constexpr int kRotAxes = 4;

// n / d for 0 <= n < 2^31 as a multiply and shift: with m = ceil(2^(31+l) / d)
// and l = ceil(log2 d) the error stays below 1/d.
struct Divider {
  uint32_t m, s, d;
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> s);
  }
};
Divider divider(uint32_t d) {
  if (d == 0) d = 1;
  uint32_t l = 0;
  while ((uint64_t{1} << l) < d) ++l;
  return Divider{static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + d - 1) / d), 31 + l, d};
}

// Strides in elements: token, head, and what a batch entry's first token lies
// off the token behind the entry before.
struct RotTensor {
  const char* x;  // what is turned: the input, or the output's gradient
  char* y;
  const char* in; // with a gradient for the positions: the input
  int64_t xb, xq, xh, yb, yq, yh, ib, iq, ih;
};

struct RotArgs {
  RotTensor t[2];
  int32_t heads0, heads;   // of the first tensor, of both
  int32_t P, units;        // pairs; vectors per head (turned, then copied)
  int32_t turned;          // vectors per head that are turned
  int32_t tokens;          // per CTA
  int32_t total;           // B * Q
  int32_t hop;             // tokens between a thread's vectors if a token's are no more than a
                           // CTA's threads (then head and pair stay the same), else 0
  int32_t step;            // vectors between a thread's; the threads that take any
  int32_t flat;            // no tensor has a gap between batch entries
  Divider dq, dunit, dhead, dpair;
  const void* pos;
  int64_t pos_batch;       // elements between batch entries' positions: 0 if shared
  int32_t pos_dtype, axes;
  const float* inv_freq;
  const int32_t* axis;
  float sign;              // -1 turns back
  float* gpos;             // (B, Q, axes)
};

__device__ __forceinline__ float rot_position(const RotArgs& a, int64_t i) {
  if (a.pos_dtype == MSDA_POSITION_INT32)
    return static_cast<float>(__ldg(static_cast<const int32_t*>(a.pos) + i));
  if (a.pos_dtype == MSDA_POSITION_INT64)
    return static_cast<float>(__ldg(static_cast<const long long*>(a.pos) + i));
  return __ldg(static_cast<const float*>(a.pos) + i);
}

__device__ __forceinline__ float2 rot_angle(float p, float f, float sign) {
  const float kHi = 0.318309873f, kLo = 1.28412765e-8f;  // 1 / pi in two floats
  const float t = __fmul_rn(p, f), tl = __fmaf_rn(p, f, -t);
  const float u = __fmul_rn(t, kHi);
  const float v = __fmaf_rn(t, kHi, -u) + __fmaf_rn(t, kLo, tl * kHi);
  const float r = __fsub_rn(u, 2.f * rintf(0.5f * u)) + v;
  float s, c;
  sincospif(r, &s, &c);
  return make_float2(c, s * sign);
}

// Loads that may be of memory that this thread writes later (in place).
template <int VB> __device__ __forceinline__ Raw<VB> rot_load(const void* p) {
  Raw<VB> r;
  if constexpr (VB == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
  } else if constexpr (VB == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r.w[0] = v.x; r.w[1] = v.y;
  } else if constexpr (VB == 4) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    r.h = *reinterpret_cast<const uint16_t*>(p);
  }
  return r;
}

// Shared memory of a CTA: the angles' (cos, sin) of its tokens, with room after
// each vector's N pairs so that lanes with different vectors meet different
// banks; for the positions' gradient each pair's frequency at its axis, spaced
// likewise, and the sums of each vector's pairs per axis.
template <int N> struct RotShared {
  static constexpr int kPad = N >= 4 ? 2 : 0;
  static __host__ __device__ int turns(int P) { return P + P / N * kPad; }  // per token
  static __host__ __device__ int weights(int P) { return P + P / N; }
  static __host__ __device__ int turn_bytes(int P, int tokens) {
    return (turns(P) * tokens * 8 + 15) / 16 * 16;
  }
};

// A thread has one vector of 16 bytes (two, of both halves) in flight; six CTAs
// an SM were faster than three with four each (762 us against 925 for 4.9 GB,
// 6.4 TB/s).  Of smaller vectors, which pairs of an odd number leave, it has two,
// and what bounds it is their instructions (20 of 24 channels in 16 bits, 0.69 GB:
// 233 us; 286 with one, and with 256 threads of which each finds its head anew).
template <typename T, int VB, bool PAIRS, bool GPOS>
__global__ void __launch_bounds__(kRotThreads, GPOS ? 4 : 6)
rotary_kernel(const __grid_constant__ RotArgs a) {
  constexpr int N = Chunk<T, VB>::EPV;  // pairs that a thread turns at a time
  // It loads vectors j of the turned channels' two halves.  They hold N pairs
  // in either order of channels, but for single interleaved elements, which are
  // a pair side by side.
  constexpr bool kAdjacent = PAIRS && N == 1;
  using S = RotShared<N>;
  extern __shared__ __align__(16) char shared[];
  const int token0 = blockIdx.x * a.tokens;
  const int tokens = min(a.tokens, a.total - token0);
  const int per_token = a.heads * a.units;
  const int count = tokens * per_token;
  const int row = S::turns(a.P);
  float2* const turn = reinterpret_cast<float2*>(shared);
  float4* const weight = reinterpret_cast<float4*>(shared + S::turn_bytes(a.P, a.tokens));
  float4* const sums = weight + S::weights(a.P);

  constexpr int U = VB == 16 ? 1 : 2;
  Raw<VB> va[U], vb[U], ia[U], ib[U];
  T* out[U];
  int t[U], j[U];
  int tt = 0, jj = 0, gap = 0;
  bool second = false;
  const T *px = nullptr, *pi = nullptr;
  T* py = nullptr;
  auto load = [&](int u, int k) {
    if (u >= count) return;
    if (u < a.step || a.hop == 0) {
      tt = a.dhead(u);
      const int rest = u - tt * per_token;
      int h = a.dunit(rest);
      jj = rest - h * a.units;
      second = h >= a.heads0;
      const RotTensor& x = a.t[second];
      if (second) h -= a.heads0;
      int c = kAdjacent ? 2 * jj : N * jj;
      gap = kAdjacent ? 1 : a.P;
      if (jj >= a.turned) {
        c = 2 * a.P + (jj - a.turned) * N;
        gap = 0;
      }
      px = reinterpret_cast<const T*>(x.x) + h * x.xh + c;
      py = reinterpret_cast<T*>(x.y) + h * x.yh + c;
      if (GPOS) pi = reinterpret_cast<const T*>(x.in) + h * x.ih + c;
    } else {
      tt += a.hop;
    }
    t[k] = tt;
    j[k] = jj;
    const RotTensor& x = a.t[second];
    const int64_t n = token0 + tt;
    int64_t ox = n * x.xq, oy = n * x.yq, oi = GPOS ? n * x.iq : 0;
    if (!a.flat) {
      const int64_t b = a.dq(static_cast<uint32_t>(n));
      ox += b * x.xb;
      oy += b * x.yb;
      if (GPOS) oi += b * x.ib;
    }
    va[k] = rot_load<VB>(px + ox);
    vb[k] = rot_load<VB>(px + ox + gap);
    out[k] = py + oy;
    if (GPOS) {
      ia[k] = rot_load<VB>(pi + oi);
      ib[k] = rot_load<VB>(pi + oi + gap);
    }
  };
  auto load_all = [&](int u) {
#pragma unroll
    for (int k = 0; k < U; ++k) load(u + k * a.step, k);
  };

  // first those before the angles' latency; threads past the step have none
  const int u0 = static_cast<int>(threadIdx.x) < a.step ? threadIdx.x : count;
  load_all(u0);
  for (int i = threadIdx.x; i < tokens * a.P; i += blockDim.x) {
    const int k = a.dpair(i), p = i - k * a.P;
    const uint32_t n = token0 + k, b = a.dq(n), q = n - b * a.dq.d;
    const int on = __ldg(a.axis + p);
    const float x = static_cast<unsigned int>(on) < static_cast<unsigned int>(a.axes)
                        ? rot_position(a, b * a.pos_batch + static_cast<int64_t>(q) * a.axes + on)
                        : __uint_as_float(0x7fc00000u);  // no such axis
    turn[k * row + p + p / N * S::kPad] = rot_angle(x, __ldg(a.inv_freq + p), a.sign);
  }
  if (GPOS)
    for (int p = threadIdx.x; p < a.P; p += blockDim.x) {
      const float f = __ldg(a.inv_freq + p);
      const int on = __ldg(a.axis + p);
      weight[p + p / N] = make_float4(on == 0 ? f : 0.f, on == 1 ? f : 0.f, on == 2 ? f : 0.f,
                                      on == 3 ? f : 0.f);
    }
  __syncthreads();

  auto turn_one = [&](int u, int k) {
    float4 ax = make_float4(0.f, 0.f, 0.f, 0.f);
    const int jk = j[k];
    if (jk >= a.turned) {
      st_chunk<VB>(out[k], va[k]);
    } else {
      // the first of N pairs, or of N / 2 in each half
      constexpr bool kSplit = PAIRS && N > 1;
      const int j2 = a.turned + jk;
      const float2* const angles = turn + t[k] * row;
      const float2* const angle =
          angles + (kSplit ? jk * N / 2 + jk / 2 * S::kPad : jk * (N + S::kPad));
      const float2* const angle2 = angles + j2 * N / 2 + j2 / 2 * S::kPad;
      const int w1 = kSplit ? jk * N / 2 + jk / 2 : jk * (N + 1), w2 = j2 * N / 2 + j2 / 2;
      float f[2 * N], s[2 * N];
      Chunk<T, VB>::unpack(va[k], f);
      Chunk<T, VB>::unpack(vb[k], f + N);
      if (GPOS) {
        Chunk<T, VB>::unpack(ia[k], s);
        Chunk<T, VB>::unpack(ib[k], s + N);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool upper = kSplit && i >= N / 2;
        const int ii = upper ? i - N / 2 : i;
        const float2 cs = upper ? angle2[ii] : angle[ii];
        const int x1 = kSplit ? 2 * i : i, x2 = kSplit ? 2 * i + 1 : i + N;
        const float y1 = f[x1] * cs.x - f[x2] * cs.y, y2 = f[x2] * cs.x + f[x1] * cs.y;
        f[x1] = y1;
        f[x2] = y2;
        if (GPOS) {
          const float g = s[x1] * y2 - s[x2] * y1;
          const float4 w = weight[(upper ? w2 : w1) + ii];
          ax.x += g * w.x;
          ax.y += g * w.y;
          ax.z += g * w.z;
          ax.w += g * w.w;
        }
      }
      st_chunk<VB>(out[k], Chunk<T, VB>::pack(f));
      st_chunk<VB>(out[k] + (kAdjacent ? 1 : a.P), Chunk<T, VB>::pack(f + N));
    }
    if (GPOS) {
      // one token's vectors may take several passes over the same slots
      float4& slot = sums[u & (kRotUnits - 1)];
      if (u >= kRotUnits) {
        const float4 o = slot;
        ax = make_float4(ax.x + o.x, ax.y + o.y, ax.z + o.z, ax.w + o.w);
      }
      slot = ax;
    }
  };
  for (int u = u0; u < count; u += a.step * U) {
    if (u >= a.step * U) load_all(u);
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (u + k * a.step < count) turn_one(u + k * a.step, k);
  }
  if (GPOS) {
    __syncthreads();
    // a warp per token, in the same order every time
    const int slots = min(per_token, kRotUnits);
    for (int k = threadIdx.x >> 5; k < tokens; k += blockDim.x >> 5) {
      float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i = threadIdx.x & 31; i < slots; i += 32) {
        const float4 o = sums[k * slots + i];
        g = make_float4(g.x + o.x, g.y + o.y, g.z + o.z, g.w + o.w);
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) {
        g.x += __shfl_xor_sync(~0u, g.x, s);
        g.y += __shfl_xor_sync(~0u, g.y, s);
        g.z += __shfl_xor_sync(~0u, g.z, s);
        g.w += __shfl_xor_sync(~0u, g.w, s);
      }
      const int d = threadIdx.x & 31;
      if (d < a.axes)
        a.gpos[static_cast<int64_t>(token0 + k) * a.axes + d] =
            d == 0 ? g.x : d == 1 ? g.y : d == 2 ? g.z : g.w;
    }
  }
}

template <typename T, int VB>
cudaError_t rotary_launch(const RotArgs& a, bool pairs, cudaStream_t st) {
  using S = RotShared<Chunk<T, VB>::EPV>;
  const unsigned int grid = (a.total + a.tokens - 1) / a.tokens;
  const int threads = (a.step + 31) / 32 * 32;
  int bytes = S::turn_bytes(a.P, a.tokens);
  if (a.gpos != nullptr) {
    bytes += (S::weights(a.P) + std::min(a.tokens * a.heads * a.units, kRotUnits)) *
             static_cast<int>(sizeof(float4));
    auto* kernel = pairs ? rotary_kernel<T, VB, true, true> : rotary_kernel<T, VB, false, true>;
    if (bytes > 48 << 10) {
      const cudaError_t err =
          cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (err != cudaSuccess) return err;
    }
    kernel<<<grid, threads, bytes, st>>>(a);
  } else {
    auto* kernel = pairs ? rotary_kernel<T, VB, true, false> : rotary_kernel<T, VB, false, false>;
    kernel<<<grid, threads, bytes, st>>>(a);
  }
  return cudaGetLastError();
}

template <typename T>
cudaError_t rotary_dispatch(const RotArgs& a, int vb, bool pairs, cudaStream_t st) {
  switch (vb) {
    case 16: return rotary_launch<T, 16>(a, pairs, st);
    case 8: return rotary_launch<T, 8>(a, pairs, st);
    case 4: return rotary_launch<T, 4>(a, pairs, st);
    default:
      if constexpr (sizeof(T) == 2) return rotary_launch<T, 2>(a, pairs, st);
      return cudaErrorInvalidValue;
  }
}

}  // namespace
}  // namespace msda

using namespace msda;

int msda_rotary(int dtype, int64_t batch, int64_t num_tokens, int64_t channels, int num_tensors,
                const int64_t* heads, const void* const* x, const int64_t* x_strides,
                void* const* y, const int64_t* y_strides, const void* positions,
                int position_dtype, int64_t position_batch, int64_t num_axes,
                const float* inv_freq, const int32_t* axis_index, int64_t num_pairs,
                int interleaved, int inverse, const void* const* inputs,
                const int64_t* input_strides, float* grad_positions, void* stream) {
  const int64_t es = elem_bytes(dtype);
  if (es == 0) return report(MSDA_ERROR_UNSUPPORTED_DTYPE, "rotary supports fp32, fp16 and bf16");
  if (num_tensors < 1 || num_tensors > 2 || batch < 0 || num_tokens < 0 || channels < 0)
    return report(MSDA_ERROR_INVALID_ARGUMENT, "one or two tensors of non-negative sizes expected");
  if (num_axes < 1 || num_axes > kRotAxes)
    return report(MSDA_ERROR_INVALID_ARGUMENT, "num_axes must be 1 to %d", kRotAxes);
  if (num_pairs < 0 || 2 * num_pairs > channels || num_pairs > kRotPairs)
    return report(MSDA_ERROR_INVALID_ARGUMENT,
                  "num_pairs (%lld) must fit the channels (%lld) and be at most %d",
                  static_cast<long long>(num_pairs), static_cast<long long>(channels), kRotPairs);
  if (position_dtype < MSDA_POSITION_FLOAT32 || position_dtype > MSDA_POSITION_INT64)
    return report(MSDA_ERROR_UNSUPPORTED_DTYPE, "positions must be fp32, int32 or int64");
  if (heads == nullptr || x == nullptr || y == nullptr || x_strides == nullptr ||
      y_strides == nullptr)
    return report(MSDA_ERROR_INVALID_ARGUMENT, "NULL tensor table");
  if (grad_positions != nullptr && (inputs == nullptr || input_strides == nullptr))
    return report(MSDA_ERROR_INVALID_ARGUMENT, "the positions' gradient needs the inputs");
  int64_t all_heads = 0;
  for (int i = 0; i < num_tensors; ++i) {
    if (heads[i] < 0) return report(MSDA_ERROR_INVALID_ARGUMENT, "negative number of heads");
    all_heads += heads[i];
  }
  constexpr int64_t kMost = 0x7fffffff;
  if (batch > kMost || num_tokens > kMost || batch * num_tokens > kMost - kRotUnits ||
      channels > kMost || all_heads > kMost || all_heads * channels > kMost / 2)
    return report(MSDA_ERROR_INT32_OVERFLOW, "batch * tokens or heads * channels exceeds int32");
  if (batch * num_tokens == 0) return report_ok();
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (all_heads * channels == 0) {
    return grad_positions == nullptr
               ? report_ok()
               : report_cuda(cudaMemsetAsync(grad_positions, 0,
                                             batch * num_tokens * num_axes * 4, st),
                             "rotary launch");
  }
  const int64_t ps = position_dtype == MSDA_POSITION_INT64 ? 8 : 4;
  if (positions == nullptr || !is_aligned(positions, ps) || !is_aligned(grad_positions, 4) ||
      (num_pairs > 0 && (inv_freq == nullptr || axis_index == nullptr ||
                         !is_aligned(inv_freq, 4) || !is_aligned(axis_index, 4))))
    return report(MSDA_ERROR_MISALIGNED, "NULL or unaligned positions or frequencies");
  RotArgs a{};
  // the largest vector that divides both halves, the rest, every stride and address
  int64_t vb = 16;
  auto fit = [&](int64_t bytes) {
    while (vb > es && bytes % vb != 0) vb >>= 1;
  };
  fit(num_pairs * es);
  bool in_place = true;
  for (int i = 0; i < num_tensors; ++i) {
    RotTensor& t = a.t[i];
    t.x = static_cast<const char*>(x[i]);
    t.y = static_cast<char*>(y[i]);
    t.in = grad_positions == nullptr ? nullptr : static_cast<const char*>(inputs[i]);
    const int64_t *xs = x_strides + 3 * i, *ys = y_strides + 3 * i;
    t.xb = xs[0]; t.xq = xs[1]; t.xh = xs[2];
    t.yb = ys[0]; t.yq = ys[1]; t.yh = ys[2];
    if (heads[i] == 0) continue;
    if (t.x == nullptr || t.y == nullptr || !is_aligned(t.x, es) || !is_aligned(t.y, es))
      return report(MSDA_ERROR_MISALIGNED, "NULL or unaligned tensor");
    in_place = in_place && t.x == t.y && t.xb == t.yb && t.xq == t.yq && t.xh == t.yh;
    for (int64_t s : {t.xb, t.xq, t.xh, t.yb, t.yq, t.yh}) fit(s * es);
    fit(static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.x) % 16));
    fit(static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.y) % 16));
    if (t.in != nullptr || grad_positions != nullptr) {
      if (t.in == nullptr || !is_aligned(t.in, es))
        return report(MSDA_ERROR_MISALIGNED, "NULL or unaligned input");
      const int64_t* is = input_strides + 3 * i;
      t.ib = is[0]; t.iq = is[1]; t.ih = is[2];
      for (int64_t s : {t.ib, t.iq, t.ih}) fit(s * es);
      fit(static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.in) % 16));
    }
  }
  const int64_t rest = in_place ? 0 : channels - 2 * num_pairs;
  fit(rest * es);
  const int64_t n = vb / es;
  a.heads0 = static_cast<int32_t>(heads[0]);
  a.heads = static_cast<int32_t>(all_heads);
  a.P = static_cast<int32_t>(num_pairs);
  a.turned = static_cast<int32_t>(num_pairs / n);
  a.units = a.turned + static_cast<int32_t>(rest / n);
  a.total = static_cast<int32_t>(batch * num_tokens);
  if (a.units == 0 && grad_positions == nullptr) return report_ok();
  const int64_t per_token = std::max<int64_t>(1, all_heads * a.units);
  a.tokens = static_cast<int32_t>(std::max<int64_t>(
      1, std::min(kRotUnits / per_token, kRotPairs / std::max<int64_t>(num_pairs, 1))));
  a.dq = divider(static_cast<uint32_t>(num_tokens));
  a.dunit = divider(static_cast<uint32_t>(a.units));
  a.dhead = divider(static_cast<uint32_t>(per_token));
  a.dpair = divider(static_cast<uint32_t>(num_pairs));
  a.pos = positions;
  a.pos_batch = position_batch;
  a.pos_dtype = position_dtype;
  a.axes = static_cast<int32_t>(num_axes);
  a.inv_freq = inv_freq;
  a.axis = axis_index;
  a.sign = inverse ? -1.f : 1.f;
  a.gpos = grad_positions;
  a.hop = static_cast<int32_t>(kRotThreads / per_token);
  a.step = a.hop == 0 ? kRotThreads : a.hop * static_cast<int32_t>(per_token);
  a.flat = 1;
  for (int i = 0; i < num_tensors; ++i) {
    RotTensor& t = a.t[i];
    t.xb -= num_tokens * t.xq;
    t.yb -= num_tokens * t.yq;
    t.ib -= num_tokens * t.iq;
    if (batch > 1 && heads[i] > 0 && (t.xb != 0 || t.yb != 0 || (t.in != nullptr && t.ib != 0)))
      a.flat = 0;
  }
  cudaError_t err;
  if (dtype == MSDA_FLOAT32) err = rotary_dispatch<float>(a, static_cast<int>(vb), interleaved, st);
  else if (dtype == MSDA_FLOAT16)
    err = rotary_dispatch<__half>(a, static_cast<int>(vb), interleaved, st);
  else err = rotary_dispatch<__nv_bfloat16>(a, static_cast<int>(vb), interleaved, st);
  return report_cuda(err, "rotary launch");
}
