// msda_norm.cu -- msda_group_norm_{fwd,bwd}: checks, the plan of units, tiles
// and waves, the launches, and the reduction of the parameters' gradients.
#include <algorithm>

#include "msda_norm.cuh"
#include "msda_status.cuh"

namespace msda {
namespace {

// Bytes of input per wave, and of the largest unit that counts as one that L2 holds.
constexpr int64_t kWaveBytes = int64_t{1} << 30;
constexpr int64_t kFitBytes = 72 << 20;
// Row pieces that a segment is cut to: as wide as this, narrower (whole lines
// still) where a unit only then fits; and the input bytes of a tile.
constexpr int64_t kSlabBytes = 256;
constexpr int64_t kMinPiece = 128;
constexpr int64_t kTileBytes = 128 << 10;
// CTAs that a pass over everything should have at least.
constexpr int64_t kMinTiles = 148 * 4;

struct Plan {
  NormLevel lv[kMaxLevels];
  int64_t tiles;    // over all levels
  int64_t counters;
  int32_t partial_stride;
  int64_t partial, done, chan, coef, bytes;  // offsets into the workspace, and its size
  int64_t zero, zero_bytes;                  // the part that starts as zeros
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Depends on sizes alone, not on pointers or strides.
int make_plan(int dtype, int64_t B, int64_t C, int64_t G, int64_t L, const int64_t* rows,
              bool backward, Plan& p) {
  const int64_t es = elem_bytes(dtype), cg = C / G;
  const int64_t streams = backward ? 2 : 1, row_bytes = C * es * streams;
  int64_t total = 0;
  for (int64_t l = 0; l < L; ++l) total += B * rows[l] * row_bytes;
  p.tiles = p.counters = 0;
  int64_t slab_groups_max = 1;
  for (int64_t l = 0; l < L; ++l) {
    NormLevel& v = p.lv[l];
    v.rows = rows[l];
    v.block0 = p.tiles;
    v.done0 = static_cast<int32_t>(p.counters);
    // Slabs of whole lines; narrower ones where a wave only then holds a slab.
    int64_t piece_bytes = kSlabBytes, sg = 1;
    for (;; piece_bytes /= 2) {
      sg = std::min(G, std::max<int64_t>(1, std::min(ceil_div(piece_bytes, cg * es), kNormMaxSlab / cg)));
      if (rows[l] * sg * cg * es * streams <= kFitBytes || piece_bytes <= kMinPiece) break;
    }
    const int64_t unit = std::max<int64_t>(1, rows[l] * sg * cg * es * streams);
    const int64_t slabs = ceil_div(G, sg);
    v.run = static_cast<int32_t>(unit > kFitBytes ? slabs : std::min(slabs, std::max<int64_t>(1, kWaveBytes / unit)));
    if (unit > kFitBytes) {  // no residency
      sg = std::min(G, std::max<int64_t>(1, std::min(ceil_div(kSlabBytes, cg * es), kNormMaxSlab / cg)));
      v.run = static_cast<int32_t>(ceil_div(G, sg));
    }
    v.slab_groups = static_cast<int32_t>(sg);
    v.slabs = static_cast<int32_t>(ceil_div(G, sg));
    slab_groups_max = std::max(slab_groups_max, sg);
    const int64_t piece = sg * cg * es * (backward ? 2 : 1);
    const int64_t tile = std::min(kTileBytes, std::max<int64_t>(total / kMinTiles, 16384));
    v.tile_rows = static_cast<int32_t>(std::max<int64_t>(
        1, std::min<int64_t>({rows[l], tile / piece, int64_t{1} << 30})));
    v.tiles = static_cast<int32_t>(ceil_div(rows[l], v.tile_rows));
    const int64_t units = rows[l] > 0 ? B * v.slabs : 0;
    p.counters += units * (1 + ceil_div(v.tiles, kNormFan));
    p.tiles += units * v.tiles;
    if (rows[l] > (int64_t{1} << 30) || p.counters > (int64_t{1} << 30))
      return report(MSDA_ERROR_INT32_OVERFLOW, "level %lld: too many rows",
                    static_cast<long long>(l));
  }
  p.partial_stride = static_cast<int32_t>(slab_groups_max * (backward ? cg : 1));
  int64_t at = 0;
  p.partial = at;
  at += round_up(p.tiles * p.partial_stride * 8, 256);
  p.coef = at;
  at += backward ? round_up(B * L * G * 8, 256) : 0;
  p.zero = p.done = at;
  at += round_up(p.counters * 4, 256);
  p.chan = at;
  at += backward ? round_up(B * L * C * 8, 256) : 0;
  p.zero_bytes = at - p.zero;
  p.bytes = at;
  return MSDA_SUCCESS;
}

int check_sizes(int dtype, int64_t B, int64_t C, int64_t G, int64_t L, const int64_t* rows) {
  if (elem_bytes(dtype) == 0)
    return report(MSDA_ERROR_UNSUPPORTED_DTYPE, "group norm supports fp32, fp16 and bf16");
  if (L < 0 || L > MSDA_MAX_LEVELS)
    return report(MSDA_ERROR_TOO_MANY_LEVELS, "num_levels=%lld exceeds the supported maximum %d",
                  static_cast<long long>(L), MSDA_MAX_LEVELS);
  if (B < 0 || C < 1 || G < 1 || C % G != 0 || C > (1 << 20))
    return report(MSDA_ERROR_INVALID_ARGUMENT,
                  "channels (%lld) must be a positive multiple of num_groups (%lld), at most 2^20",
                  static_cast<long long>(C), static_cast<long long>(G));
  if (L > 0 && rows == nullptr) return report(MSDA_ERROR_INVALID_ARGUMENT, "rows is NULL");
  for (int64_t l = 0; l < L; ++l)
    if (rows[l] < 0)
      return report(MSDA_ERROR_INVALID_ARGUMENT, "negative size at level %lld",
                    static_cast<long long>(l));
  return MSDA_SUCCESS;
}

// The largest vector that divides a group, every stride and every address.
int vector_bytes(const Plan& p, int64_t L, int64_t cg, int64_t es, bool backward) {
  int64_t vb = 16;
  auto fit = [&](int64_t bytes) {
    while (vb > es && bytes % vb != 0) vb >>= 1;
  };
  fit(cg * es);
  for (int64_t l = 0; l < L; ++l) {
    const NormLevel& v = p.lv[l];
    if (v.rows == 0) continue;
    fit(static_cast<int64_t>(reinterpret_cast<uintptr_t>(v.x) % 16));
    fit(static_cast<int64_t>(reinterpret_cast<uintptr_t>(v.out) % 16));
    for (int64_t s : {v.x_batch, v.x_row, v.out_batch, v.out_row}) fit(s * es);
    if (backward) {
      fit(static_cast<int64_t>(reinterpret_cast<uintptr_t>(v.gy) % 16));
      for (int64_t s : {v.gy_batch, v.gy_row}) fit(s * es);
    }
  }
  return static_cast<int>(vb);
}

// Waves of whole units, each of kWaveBytes of input if units are that small.
cudaError_t launch_waves(const NormArgs& a, const Plan& p, int64_t B, int dtype, int vb, int act,
                         bool backward, cudaStream_t st) {
  NormWave w{0, 0, 0, 0, 1};
  const int64_t es = elem_bytes(dtype) * (backward ? 2 : 1);
  int64_t in_wave = 0;
  auto flush = [&]() {
    const cudaError_t err = norm_wave(a, w, dtype, vb, act, backward, st);
    w = NormWave{w.stats0, w.stats0 + w.stats, w.stats, 0, w.order};
    in_wave = 0;
    return err;
  };
  for (int l = 0; l < a.L; ++l) {
    const NormLevel& v = a.lv[l];
    if (v.rows == 0) continue;
    for (int64_t b = 0; b < B; ++b)
      for (int32_t s0 = 0; s0 < v.slabs; s0 += v.run) {
        const int32_t width = std::min(v.run, v.slabs - s0);
        const int64_t bytes = v.rows * es *
                              (std::min<int64_t>((s0 + width) * v.slab_groups * a.cg, a.C) -
                               static_cast<int64_t>(s0) * v.slab_groups * a.cg);
        // a launch's tiles are counted in 32 bits
        if (w.stats > 0 && (in_wave + bytes > kWaveBytes || w.stats > (1 << 28))) {
          const cudaError_t err = flush();
          if (err != cudaSuccess) return err;
        }
        w.stats += width * v.tiles;
        in_wave += bytes;
      }
  }
  cudaError_t err = flush();
  if (err == cudaSuccess && w.applies > 0) err = flush();
  return err;
}

void fill(NormArgs& a, const Plan& p, int64_t C, int64_t G, int64_t L, const void* weight,
         const void* bias, int affine_dtype, int affine_per_level, void* workspace) {
  std::copy(p.lv, p.lv + L, a.lv);
  a.L = static_cast<int32_t>(L);
  a.C = static_cast<int32_t>(C);
  a.G = static_cast<int32_t>(G);
  a.cg = static_cast<int32_t>(C / G);
  a.weight = weight;
  a.bias = bias;
  a.affine_dtype = affine_dtype;
  a.affine_level = affine_per_level ? a.C : 0;
  char* ws = static_cast<char*>(workspace);
  a.partial = reinterpret_cast<float2*>(ws + p.partial);
  a.partial_stride = p.partial_stride;
  a.done = reinterpret_cast<unsigned int*>(ws + p.done);
  a.chan = reinterpret_cast<float2*>(ws + p.chan);
  a.coef = reinterpret_cast<float2*>(ws + p.coef);
}

int check_common(const Plan& p, int64_t L, int64_t es, const void* weight, const void* bias,
                 int affine_dtype, int act, const void* stats, const void* workspace,
                 size_t workspace_bytes, bool backward) {
  if (act < MSDA_ACT_NONE || act > MSDA_ACT_GELU)
    return report(MSDA_ERROR_INVALID_ARGUMENT, "unknown activation %d", act);
  const int64_t as = elem_bytes(affine_dtype);
  if (as == 0)
    return report(MSDA_ERROR_UNSUPPORTED_DTYPE, "the affine map must be fp32, fp16 or bf16");
  if (!is_aligned(weight, as) || !is_aligned(bias, as))
    return report(MSDA_ERROR_MISALIGNED, "unaligned affine map");
  for (int64_t l = 0; l < L; ++l) {
    const NormLevel& v = p.lv[l];
    if (v.rows == 0) continue;
    if (v.x == nullptr || v.out == nullptr || !is_aligned(v.x, es) || !is_aligned(v.out, es) ||
        (backward && (v.gy == nullptr || !is_aligned(v.gy, es))))
      return report(MSDA_ERROR_MISALIGNED, "NULL or unaligned feature buffer");
    if (stats == nullptr || !is_aligned(stats, 8))
      return report(MSDA_ERROR_MISALIGNED, "NULL or unaligned statistics");
  }
  if (p.bytes > 0 && (workspace == nullptr || !is_aligned(workspace, 256) ||
                      workspace_bytes < static_cast<size_t>(p.bytes)))
    return report(MSDA_ERROR_WORKSPACE, "workspace needs %lld bytes, 256-byte aligned",
                  static_cast<long long>(p.bytes));
  return MSDA_SUCCESS;
}

__global__ void norm_param_grad_kernel(const NormParamGrad p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int levels = p.per_level ? 1 : p.L;
  if (i >= static_cast<int64_t>(p.per_level ? p.L : 1) * p.C) return;
  const int64_t l0 = p.per_level ? i / p.C : 0, c = p.per_level ? i % p.C : i;
  float sw = 0.f, sb = 0.f;
  for (int b = 0; b < p.B; ++b)
    for (int l = 0; l < levels; ++l) {
      const float2 s = __ldg(p.chan + (static_cast<int64_t>(b) * p.L + l0 + l) * p.C + c);
      sb += s.x;
      sw += s.y;
    }
  auto put = [&](void* out, float v) {
    if (out == nullptr) return;
    if (p.dtype == MSDA_FLOAT32) static_cast<float*>(out)[i] = v;
    else if (p.dtype == MSDA_FLOAT16) static_cast<__half*>(out)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  };
  put(p.gweight, sw);
  put(p.gbias, sb);
}

}  // namespace

cudaError_t norm_wave(const NormArgs& a, const NormWave& w, int dtype, int vb, int act,
                      bool backward, cudaStream_t st) {
  if (dtype == MSDA_FLOAT32) return norm_wave_t<float>(a, w, vb, act, backward, st);
  if (dtype == MSDA_FLOAT16) return norm_wave_t<__half>(a, w, vb, act, backward, st);
  return norm_wave_t<__nv_bfloat16>(a, w, vb, act, backward, st);
}

cudaError_t norm_param_grad(const NormParamGrad& p, cudaStream_t st) {
  const int64_t n = static_cast<int64_t>(p.per_level ? p.L : 1) * p.C;
  if (n == 0) return cudaSuccess;
  norm_param_grad_kernel<<<static_cast<unsigned int>(ceil_div(n, 128)), 128, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace msda

using namespace msda;

size_t msda_group_norm_workspace_bytes(int dtype, int64_t batch, int64_t channels,
                                       int64_t num_groups, int64_t num_levels,
                                       const int64_t* rows, int backward) {
  Plan p;
  if (check_sizes(dtype, batch, channels, num_groups, num_levels, rows) != MSDA_SUCCESS ||
      make_plan(dtype, batch, channels, num_groups, num_levels, rows, backward != 0, p) !=
          MSDA_SUCCESS)
    return 0;
  return static_cast<size_t>(p.bytes);
}

int msda_group_norm_fwd(int dtype, int64_t batch, int64_t channels, int64_t num_groups,
                        int64_t num_levels, const int64_t* rows, const void* const* x,
                        const int64_t* x_strides, const void* weight, const void* bias,
                        int affine_dtype, int affine_per_level, double eps, int activation,
                        void* y, float* stats, void* workspace, size_t workspace_bytes,
                        void* stream) {
  Plan p;
  int rc = check_sizes(dtype, batch, channels, num_groups, num_levels, rows);
  if (rc != MSDA_SUCCESS) return rc;
  rc = make_plan(dtype, batch, channels, num_groups, num_levels, rows, false, p);
  if (rc != MSDA_SUCCESS) return rc;
  if (!(eps >= 0)) return report(MSDA_ERROR_INVALID_ARGUMENT, "eps must not be negative");
  const int64_t es = elem_bytes(dtype);
  int64_t keys = 0, at = 0;
  for (int64_t l = 0; l < num_levels; ++l) keys += rows[l];
  if (batch == 0 || keys == 0) return report_ok();
  if (x == nullptr || x_strides == nullptr || y == nullptr)
    return report(MSDA_ERROR_INVALID_ARGUMENT, "NULL feature table");
  for (int64_t l = 0; l < num_levels; ++l) {
    NormLevel& v = p.lv[l];
    v.x = static_cast<const char*>(x[l]);
    v.out = static_cast<char*>(y) + at * channels * es;
    v.gy = nullptr;
    v.x_batch = x_strides[2 * l];
    v.x_row = x_strides[2 * l + 1];
    v.out_batch = keys * channels;
    v.out_row = channels;
    v.gy_batch = v.gy_row = 0;
    at += rows[l];
  }
  rc = check_common(p, num_levels, es, weight, bias, affine_dtype, activation, stats, workspace,
                    workspace_bytes, false);
  if (rc != MSDA_SUCCESS) return rc;
  NormArgs a{};
  fill(a, p, channels, num_groups, num_levels, weight, bias, affine_dtype, affine_per_level,
       workspace);
  a.eps = static_cast<float>(eps);
  a.stats = reinterpret_cast<float2*>(stats);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t err = cudaMemsetAsync(static_cast<char*>(workspace) + p.zero, 0,
                                    static_cast<size_t>(p.zero_bytes), st);
  if (err == cudaSuccess)
    err = launch_waves(a, p, batch, dtype, vector_bytes(p, num_levels, a.cg, es, false),
                       activation, false, st);
  return report_cuda(err, "group norm forward launch");
}

int msda_group_norm_bwd(int dtype, int64_t batch, int64_t channels, int64_t num_groups,
                        int64_t num_levels, const int64_t* rows, const void* const* x,
                        const int64_t* x_strides, const void* weight, const void* bias,
                        int affine_dtype, int affine_per_level, int activation,
                        const float* stats, const void* grad_y, void* const* grad_x,
                        const int64_t* grad_x_strides, void* grad_weight, void* grad_bias,
                        void* workspace, size_t workspace_bytes, void* stream) {
  Plan p;
  int rc = check_sizes(dtype, batch, channels, num_groups, num_levels, rows);
  if (rc != MSDA_SUCCESS) return rc;
  rc = make_plan(dtype, batch, channels, num_groups, num_levels, rows, true, p);
  if (rc != MSDA_SUCCESS) return rc;
  const int64_t es = elem_bytes(dtype);
  int64_t keys = 0, at = 0;
  for (int64_t l = 0; l < num_levels; ++l) keys += rows[l];
  if (batch == 0) keys = 0;
  if (keys > 0 && (x == nullptr || x_strides == nullptr || grad_y == nullptr ||
                   grad_x == nullptr || grad_x_strides == nullptr))
    return report(MSDA_ERROR_INVALID_ARGUMENT, "NULL feature table");
  for (int64_t l = 0; l < num_levels; ++l) {
    NormLevel& v = p.lv[l];
    if (keys == 0) {
      v.rows = 0;
      continue;
    }
    v.x = static_cast<const char*>(x[l]);
    v.out = static_cast<char*>(grad_x[l]);
    v.gy = static_cast<const char*>(grad_y) + at * channels * es;
    v.x_batch = x_strides[2 * l];
    v.x_row = x_strides[2 * l + 1];
    v.out_batch = grad_x_strides[2 * l];
    v.out_row = grad_x_strides[2 * l + 1];
    v.gy_batch = keys * channels;
    v.gy_row = channels;
    at += rows[l];
  }
  rc = check_common(p, num_levels, es, weight, bias, affine_dtype, activation, stats, workspace,
                    workspace_bytes, true);
  if (rc != MSDA_SUCCESS) return rc;
  const int64_t as = elem_bytes(affine_dtype);
  if (!is_aligned(grad_weight, as) || !is_aligned(grad_bias, as))
    return report(MSDA_ERROR_MISALIGNED, "unaligned gradient of the affine map");
  NormArgs a{};
  fill(a, p, channels, num_groups, num_levels, weight, bias, affine_dtype, affine_per_level,
       workspace);
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t err = p.zero_bytes == 0
                        ? cudaSuccess
                        : cudaMemsetAsync(static_cast<char*>(workspace) + p.zero, 0,
                                          static_cast<size_t>(p.zero_bytes), st);
  if (err == cudaSuccess)
    err = launch_waves(a, p, batch, dtype, vector_bytes(p, num_levels, a.cg, es, true),
                       activation, true, st);
  if (err == cudaSuccess && (grad_weight != nullptr || grad_bias != nullptr))
    err = norm_param_grad(NormParamGrad{a.chan, static_cast<int32_t>(batch), a.L, a.C,
                                        affine_per_level, affine_dtype, grad_weight, grad_bias},
                          st);
  return report_cuda(err, "group norm backward launch");
}
