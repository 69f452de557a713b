// msda_norm.cu -- msda_group_norm_{fwd,bwd}: checks, and the plan of units
// and tiles.
#include <algorithm>
#include <numeric>

#include "msda_norm.cuh"
#include "msda_status.cuh"

namespace msda {
namespace {

constexpr int64_t kSMs = 148;
// Row pieces that a slab takes, direct or not (of 64 bytes, DRAM was read in
// 128: 336 MB a pass where 200 were wanted).
constexpr int64_t kDirectPiece = 128, kPiece = 256;
// Bytes of x in a tile.  Direct: as many tiles as CTAs run at once, nearly (of
// the 2D encoder's 41 MB, 632 tiles where 592 run took 32 us forward, 576 take
// 27), but no fewer bytes than the first.  Else the third, or the second where
// there would be few tiles.  At once: four CTAs an SM forward and, as its
// application has, three backward.
constexpr int64_t kSmallTile = 16 << 10, kMediumTile = 64 << 10, kTile = 128 << 10;
// The one launch: the narrowest piece of a row, and from where on whole lines.
constexpr int64_t kOncePiece = 32, kOnceMuch = 32 << 20;
// Direct: at most so many tiles a unit, and (for the affine map's gradients) in
// all batch entries' and levels' units of a slab.
constexpr int64_t kDirectTiles = 64, kDirectSum = 2048;

struct Plan {
  NormLevel lv[kMaxLevels];
  int64_t tiles;  // over all levels
  int64_t counters;
  bool direct;
  int32_t partial_stride;
  int64_t partial, weighted, done, chan, coef, bytes;  // offsets into the workspace, and its size
  int64_t zero_bytes;                                  // from `done` on: starts as zeros
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Depends on sizes alone, not on pointers or strides.  Sizes in bytes are of x;
// the backward reads as much of gy.
int make_plan(int dtype, int64_t B, int64_t C, int64_t G, int64_t L, const int64_t* rows,
              bool backward, Plan& p) {
  const int64_t es = elem_bytes(dtype), cg = C / G;
  int64_t total = 0, sg = 1;
  for (int64_t l = 0; l < L; ++l) {
    if (rows[l] > (int64_t{1} << 30) || B * rows[l] > (int64_t{1} << 40) / C)
      return report(MSDA_ERROR_INT32_OVERFLOW, "level %lld: too many rows",
                    static_cast<long long>(l));
    total += B * rows[l] * C * es;
  }
  for (int attempt = 0; attempt < 2; ++attempt) {
    p.direct = attempt == 0;
    const int64_t at_once = kSMs * (backward ? 3 : 4);
    const int64_t tile = p.direct ? std::max(kSmallTile, total * 12 / (11 * at_once))
                                  : std::min(kTile, std::max(total / at_once, kMediumTile));
    const int64_t piece = p.direct ? kDirectPiece : kPiece;
    sg = std::min(G, std::max<int64_t>(1, std::min(ceil_div(piece, cg * es), kNormMaxSlab / cg)));
    // of whole vectors, for those that hold several groups
    const int64_t whole = std::min(G, round_up(sg, 16 / es / std::gcd(cg, 16 / es)));
    if (whole * cg <= kNormMaxSlab) sg = whole;
    p.tiles = p.counters = 0;
    int64_t most = 0, sum = 0;
    for (int64_t l = 0; l < L; ++l) {
      NormLevel& v = p.lv[l];
      v.rows = rows[l];
      v.tile0 = static_cast<int32_t>(p.tiles);
      v.done0 = static_cast<int32_t>(p.counters);
      v.slab_groups = static_cast<int32_t>(sg);
      v.slabs = static_cast<int32_t>(ceil_div(G, sg));
      v.tile_rows =
          static_cast<int32_t>(std::max<int64_t>(1, std::min(rows[l], tile / (sg * cg * es))));
      v.tiles = static_cast<int32_t>(ceil_div(rows[l], v.tile_rows));
      const int64_t units = rows[l] > 0 ? B * v.slabs : 0;
      p.counters += units * (1 + ceil_div(v.tiles, kNormFan));
      p.tiles += units * v.tiles;
      most = std::max<int64_t>(most, v.tiles);
      sum += B * v.tiles;
      if (p.counters > (1 << 29) || p.tiles > (1 << 29))
        return report(MSDA_ERROR_INT32_OVERFLOW, "too many tiles of work");
    }
    if (p.direct && tile <= kTile && most <= kDirectTiles && (!backward || sum <= kDirectSum))
      break;
  }
  p.partial_stride = static_cast<int32_t>(sg * (backward ? cg : 1));
  int64_t at = 0;
  p.partial = at;
  at += round_up(p.tiles * p.partial_stride * 8, 256);
  p.weighted = at;
  at += backward && p.direct ? round_up(p.tiles * sg * 8, 256) : 0;
  p.coef = at;
  at += backward && !p.direct ? round_up(B * L * G * 8, 256) : 0;
  p.chan = at;
  at += backward && !p.direct ? round_up(B * L * C * 8, 256) : 0;
  p.done = at;
  at += p.direct ? 0 : round_up(p.counters * 4, 256);
  p.zero_bytes = at - p.done;
  p.bytes = std::max<int64_t>(at, 256);
  return MSDA_SUCCESS;
}

int check_sizes(int dtype, int64_t B, int64_t C, int64_t G, int64_t L, const int64_t* rows) {
  if (elem_bytes(dtype) == 0)
    return report(MSDA_ERROR_UNSUPPORTED_DTYPE, "group norm supports fp32, fp16 and bf16");
  if (L < 0 || L > MSDA_MAX_LEVELS)
    return report(MSDA_ERROR_TOO_MANY_LEVELS, "num_levels=%lld exceeds the supported maximum %d",
                  static_cast<long long>(L), MSDA_MAX_LEVELS);
  if (B < 0 || B > 0x7fffffff || C < 1 || G < 1 || C % G != 0 || C > (1 << 20))
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

// The largest vector that divides every stride and every address.
int vector_bytes(const NormArgs& a, int64_t es, bool backward) {
  int64_t vb = 16;
  auto fit = [&](int64_t bytes) {
    while (vb > es && bytes % vb != 0) vb >>= 1;
  };
  for (int64_t l = 0; l < a.L; ++l) {
    const NormLevel& v = a.lv[l];
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

void fill(NormArgs& a, const Plan& p, int64_t B, int64_t C, int64_t G, int64_t L,
          const void* weight, const void* bias, int affine_dtype, int affine_per_level,
          void* workspace) {
  std::copy(p.lv, p.lv + L, a.lv);
  a.L = static_cast<int32_t>(L);
  a.C = static_cast<int32_t>(C);
  a.G = static_cast<int32_t>(G);
  a.cg = static_cast<int32_t>(C / G);
  a.B = static_cast<int32_t>(B);
  a.weight = weight;
  a.bias = bias;
  a.affine_dtype = affine_dtype;
  a.affine_level = affine_per_level ? a.C : 0;
  char* ws = static_cast<char*>(workspace);
  a.partial = reinterpret_cast<float2*>(ws + p.partial);
  a.partial_stride = p.partial_stride;
  a.tiles = static_cast<int32_t>(p.tiles);
  a.direct = p.direct;
  a.weighted = reinterpret_cast<float2*>(ws + p.weighted);
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

// The one launch's units, if a CTA's registers hold each: as wide pieces of
// rows as that allows, down to kOncePiece, or to whole lines where much is read.
bool make_once(NormArgs& a, int vb, int64_t es) {
  const int64_t epv = vb / es;
  int64_t total = 0, tiles = 0;
  for (int l = 0; l < a.L; ++l) total += a.B * a.lv[l].rows * a.C * es;
  const int64_t least = total > kOnceMuch ? kDirectPiece : kOncePiece;
  NormLevel lv[kMaxLevels];
  for (int l = 0; l < a.L; ++l) {
    NormLevel& v = lv[l] = a.lv[l];
    int64_t groups = std::min<int64_t>(
        {a.G, kNormMaxSlab, std::max<int64_t>(1, kDirectPiece / (a.cg * es))});
    for (;; groups = (groups + 1) / 2) {
      const int64_t columns = groups * a.cg / epv;
      if (columns <= kNormOnceThreads &&
          v.rows <= kNormOnceThreads / columns * kNormOnceVectors)
        break;
      if (groups == 1 || groups * a.cg * es <= least) return false;
    }
    v.tile0 = static_cast<int32_t>(tiles);
    v.slab_groups = static_cast<int32_t>(groups);
    v.slabs = static_cast<int32_t>(ceil_div(a.G, groups));
    v.tiles = 1;
    v.tile_rows = static_cast<int32_t>(v.rows);
    tiles += v.rows > 0 ? static_cast<int64_t>(a.B) * v.slabs : 0;
    if (tiles > (1 << 29)) return false;
  }
  std::copy(lv, lv + a.L, a.lv);
  a.tiles = static_cast<int32_t>(tiles);
  return true;
}

// Zeroes what starts as zeros, then both launches; or the one.
cudaError_t run(NormArgs& a, const Plan& p, int dtype, int act, bool backward, void* workspace,
                cudaStream_t st) {
  const int64_t es = elem_bytes(dtype);
  const int wide = vector_bytes(a, es, backward);
  int vb = wide;  // dividing a group too
  while (a.cg * es % vb != 0) vb >>= 1;
  const bool once = !backward && make_once(a, vb, es);
  // slabs of whole vectors, where those hold several groups
  const bool mixed = !once && wide == 16 && vb < 16 && a.C * es % 16 == 0 &&
                     (a.lv[0].slab_groups == a.G || a.lv[0].slab_groups * a.cg * es % 16 == 0) &&
                     a.lv[0].slab_groups * a.cg <= kNormMaxSlab;
  if (p.zero_bytes > 0 && !once) {
    const cudaError_t err = cudaMemsetAsync(static_cast<char*>(workspace) + p.done, 0,
                                            static_cast<size_t>(p.zero_bytes), st);
    if (err != cudaSuccess) return err;
  }
  if (dtype == MSDA_FLOAT32) return norm_launch<float>(a, vb, mixed, act, backward, once, st);
  if (dtype == MSDA_FLOAT16) return norm_launch<__half>(a, vb, mixed, act, backward, once, st);
  return norm_launch<__nv_bfloat16>(a, vb, mixed, act, backward, once, st);
}

}  // namespace
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
  fill(a, p, batch, channels, num_groups, num_levels, weight, bias, affine_dtype, affine_per_level,
       workspace);
  a.eps = static_cast<float>(eps);
  a.stats = reinterpret_cast<float2*>(stats);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t err = run(a, p, dtype, activation, false, workspace, st);
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
  fill(a, p, batch, channels, num_groups, num_levels, weight, bias, affine_dtype, affine_per_level,
       workspace);
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (grad_weight != nullptr || grad_bias != nullptr) {
    a.gweight = grad_weight;
    a.gbias = grad_bias;
    a.param_ctas = static_cast<int32_t>((affine_per_level ? num_levels : 1) *
                                        ceil_div(channels, kNormParamChannels));
  }
  const cudaError_t err = run(a, p, dtype, activation, true, workspace, st);
  return report_cuda(err, "group norm backward launch");
}
