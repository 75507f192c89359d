// disco_residual.hip -- C entries of the join between two residual blocks, and the end of its parameter gradients.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "disco_residual.h"

namespace disco {

__device__ __forceinline__ float param_at(const void* p, int type, int64_t i) {
  if (type == DISCO_F32) return static_cast<const float*>(p)[i];
  if (type == DISCO_F16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void param_put(void* p, int type, int64_t i, double v) {
  if (type == DISCO_F32) static_cast<float*>(p)[i] = (float)v;
  else if (type == DISCO_F16) static_cast<_Float16*>(p)[i] = (_Float16)(float)v;
  else static_cast<__bf16*>(p)[i] = (__bf16)(float)v;
}

struct FinishArgs {
  const float* partial;
  int64_t groups;
  int width, partials, param_type, channel, act;
  float scale;
  const void *w1, *b1, *lam, *g;
  void *dw1, *db1, *dw2, *db2, *dlam, *dg;
};

// Parameter gradients from the workgroups' column sums: 16 columns per workgroup, 64 lanes down each column, sums in
// float64 in a fixed order.  With c = act(channel gate) and s the scale, z = u1 * w1 + b1 gives
//   dw1 = s c P1,  db1 = s c P2,  ds = c (w1 P1 + b1 P2),  dgate = s c' (w1 P1 + b1 P2),  dw2 = P3,  db2 = P4.
__global__ __launch_bounds__(1024) void k_residual_finish(const FinishArgs a) {
  __shared__ double part[4][16][16];
  const int cl = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + cl;
  double w = 1.0, b = 0.0, scale = (double)a.scale, g = 0.0;      // read while the sums come in
  if (slice == 0 && c < a.width) {
    if (a.w1) w = (double)param_at(a.w1, a.param_type, c);
    if (a.b1) b = (double)param_at(a.b1, a.param_type, c);
    if (a.lam) scale *= (double)param_at(a.lam, a.param_type, c);
    if (a.channel) g = (double)param_at(a.g, a.param_type, c);
  }
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  if (c < a.width) {
    // four groups of all sums in flight: each load waits for memory that another workgroup wrote
    const float* p = a.partial + (int64_t)slice * 4 * a.width + c;
    const int64_t step = 64 * 4 * (int64_t)a.width;
    for (int64_t g = slice; g < a.groups; g += 64 * 4, p += 4 * step) {
      float v[4][4] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (a.partials >> k & 1)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[k][i] = p[(g + 64 * i < a.groups ? i * step : 0) + (int64_t)k * a.width];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[k] += g + 64 * i < a.groups ? (double)v[k][i] : 0.0;
    }
  }
  // the four slices of a wave, then the 16 waves: lane 16 k + column of the first wave ends with sum k of its column
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    s[k] += __shfl_xor(s[k], 16, 64);
    s[k] += __shfl_xor(s[k], 32, 64);
    if ((threadIdx.x & 63) < 16) part[k][threadIdx.x >> 6][cl] = s[k];
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += part[threadIdx.x >> 4][i][cl];
  const double P1 = __shfl(sum, cl, 64), P2 = __shfl(sum, 16 + cl, 64), P3 = __shfl(sum, 32 + cl, 64), P4 = __shfl(sum, 48 + cl, 64);
  if (slice != 0 || c >= a.width) return;
  double gate = 1.0, slope = 0.0;
  if (a.channel) {
    // slopes from the exponential: 1 - gate would cancel
    if (a.act == DISCO_ACT_SIGMOID) {
      const double e = exp(-fabs(g)), r = 1.0 / (1.0 + e);
      gate = g < 0.0 ? e * r : r;
      slope = e * r * r;
    } else if (a.act == DISCO_ACT_TANH) {
      const double e = exp(-2.0 * fabs(g)), r = 1.0 / (1.0 + e);
      gate = tanh(g);
      slope = 4.0 * e * r * r;
    } else {
      gate = g;
      slope = 1.0;
    }
  }
  if (a.dw1) param_put(a.dw1, a.param_type, c, scale * gate * P1);
  if (a.db1) param_put(a.db1, a.param_type, c, scale * gate * P2);
  const double T = w * P1 + b * P2;
  if (a.dlam) param_put(a.dlam, a.param_type, c, (double)a.scale * gate * T);
  if (a.channel && a.dg) param_put(a.dg, a.param_type, c, scale * slope * T);
  if (a.dw2) param_put(a.dw2, a.param_type, c, P3);
  if (a.db2) param_put(a.db2, a.param_type, c, P4);
}

// Zeros into rows of `width` elements, for a gradient that nothing flows into.
template <typename T>
__global__ __launch_bounds__(256) void k_residual_zero(T* p, int64_t rows, int64_t width, int64_t ld) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * width; i += (int64_t)gridDim.x * 256) p[i / width * ld + i % width] = (T)0.0f;
}

static int pair_of(int stream_type, int block_type) {
  if (stream_type == block_type) return stream_type == DISCO_F32 ? kPairF32 : stream_type == DISCO_F16 ? kPairF16 : stream_type == DISCO_BF16 ? kPairBF16 : -1;
  if (stream_type == DISCO_F32) return block_type == DISCO_F16 ? kPairF32F16 : block_type == DISCO_BF16 ? kPairF32BF16 : -1;
  return -1;
}

static int check_desc(const disco_residual_norm* d) {
  if (!d || d->rows < 0 || d->width < 1 || !(d->eps > 0.0f) || !isfinite(d->eps) || !isfinite(d->scale)) return DISCO_EINVAL;
  if (d->param_type < DISCO_F32 || d->param_type > DISCO_BF16 || pair_of(d->stream_type, d->block_type) < 0) return DISCO_EINVAL;
  if (d->post_norm < DISCO_NORM_NONE || d->post_norm > DISCO_NORM_LAYER || d->pre_norm < DISCO_NORM_NONE || d->pre_norm > DISCO_NORM_LAYER)
    return DISCO_EINVAL;
  if (d->gate_kind < DISCO_GATE_NONE || d->gate_kind > DISCO_GATE_CHANNEL || d->gate_act < DISCO_ACT_NONE || d->gate_act > DISCO_ACT_TANH)
    return DISCO_EINVAL;
  if (!d->has_block && (d->post_norm || d->gate_kind || d->scale_vector || d->post_weight || d->post_bias || !d->pre_norm)) return DISCO_EINVAL;
  if (!d->post_norm && (d->post_weight || d->post_bias)) return DISCO_EINVAL;
  if (!d->pre_norm && (d->pre_weight || d->pre_bias)) return DISCO_EINVAL;
  if (d->gate_kind == DISCO_GATE_CHANNEL && !d->gate) return DISCO_EINVAL;
  if (d->width > DISCO_RESIDUAL_MAX_WIDTH) return DISCO_EUNSUPPORTED;
  return DISCO_OK;
}

static void fill(const disco_residual_norm* d, ResidualArgs* a) {
  *a = ResidualArgs{};
  a->rows = d->rows; a->width = (int)d->width;
  a->ldx = d->ldx; a->ldy = d->ldy; a->ldg = d->ld_gate;
  a->param_type = d->param_type; a->post = d->post_norm; a->pre = d->pre_norm; a->gate = d->gate_kind; a->act = d->gate_act;
  a->scale = d->scale; a->eps = d->eps; a->inv_width = 1.0f / (float)d->width;
  a->x = d->x; a->y = d->has_block ? d->y : nullptr; a->g = d->gate;
  a->w1 = d->post_weight; a->b1 = d->post_bias; a->w2 = d->pre_weight; a->b2 = d->pre_bias; a->lam = d->scale_vector;
}

// Workgroups of a launch: about what the 256 compute units hold at once, each walks its share of the rows.
static unsigned groups(int64_t rows, int threads, int lanes, int64_t most) {
  const int64_t at_a_time = threads / lanes, want = (rows + at_a_time - 1) / at_a_time;
  return (unsigned)(want < most ? want : most);
}
// The forward's waves: as many as keep FETCHED bytes of rows on their way to a compute unit (HBM answers after about a
// microsecond at 20 GB/s for each), and no more: each further wave is one more place that memory is read and written at.
// Joins of 100 M float32 or 200 M half values, float32 rows of 256: 287 us with 8 waves, 308 with 16, 343 with 32; half rows:
// 297, 322, 351; norms, with half the bytes a wave, need 16: 179 us with 8, 141 with 16, 150 with 32.  Rows that several waves share
// wait for each other, and want more (half rows of 5000: 383 us with 8, 304 with 16); so do gates for each element, whose
// arithmetic shows (169343 x 256: 180 us with 8, 157 with 12).
static unsigned forward_grid(int64_t rows, int64_t width, const ResidualShape& s, int mode, bool wide_stream, bool halves) {
  const int threads = residual_threads(s.lanes), y = halves ? 2 : 4, x = wide_stream ? 4 : 2;
  const int bytes = (int)(64 * width / s.lanes) * (x + (mode == kNormOnly ? 0 : mode == kJoin ? y : 2 * y));
  const int fetched = (mode == kJoinGated ? 2 : 1) * (s.lanes <= 64 ? 16384 : s.lanes <= 256 ? 24576 : 32768);
  const int waves = std::max(8, std::min(32, (fetched + bytes - 1) / bytes));
  return groups(rows, threads, s.lanes, 256 * std::max(1, (waves * 64 + threads - 1) / threads));
}

// The backward's number is also the number of partial sums that the finish reads again.
static unsigned backward_grid(int64_t rows, const ResidualShape& s, int mode) {
  const int threads = residual_back_threads(s.lanes, s.elems, mode);
  return groups(rows, threads, s.lanes, (int64_t)residual_back_waves(s.lanes, s.elems, mode) * 256 * 256 / threads);
}

static bool strided(int64_t ld, int64_t rows, int64_t width) { return rows <= 1 || ld >= width; }

}  // namespace disco

using namespace disco;

extern "C" int disco_residual_norm_forward(const disco_residual_norm* d, void* out, int64_t ld_out, void* h, int64_t ld_h,
                                           float* stats, void* stream_) {
  const int rc = check_desc(d);
  if (rc != DISCO_OK) return rc;
  const int64_t n = d->rows, F = d->width;
  if (!strided(ld_out, n, F) && d->has_block) return DISCO_EINVAL;
  if (!strided(ld_h, n, F) && d->pre_norm) return DISCO_EINVAL;
  if (n == 0) return DISCO_OK;
  if (d->ldx < 0 || d->ldy < 0 || d->ld_gate < 0) return DISCO_EINVAL;
  if (!d->x || (d->has_block && (!d->y || !out)) || (d->pre_norm && !h) || (d->gate_kind && !d->gate)) return DISCO_EINVAL;
  ResidualArgs a;
  fill(d, &a);
  a.out = out; a.ldo = ld_out; a.h = h; a.ldh = ld_h; a.stats = stats;
  const ResidualShape s = residual_shape(F, d->block_type != DISCO_F32);
  const unsigned grid = forward_grid(n, F, s, residual_mode(d->has_block, d->gate_kind), d->stream_type == DISCO_F32, d->block_type != DISCO_F32);
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  switch (pair_of(d->stream_type, d->block_type)) {
    case kPairF32: return residual_forward<kPairF32>(a, grid, stream);
    case kPairF16: return residual_forward<kPairF16>(a, grid, stream);
    case kPairBF16: return residual_forward<kPairBF16>(a, grid, stream);
    case kPairF32F16: return residual_forward<kPairF32F16>(a, grid, stream);
    default: return residual_forward<kPairF32BF16>(a, grid, stream);
  }
}

extern "C" size_t disco_residual_norm_workspace_bytes(int64_t rows, int64_t width) {
  if (rows < 0 || width < 1 || width > DISCO_RESIDUAL_MAX_WIDTH) return 0;
  unsigned most = 0;      // of any type and gate
  for (const bool halves : {false, true})
    for (const int mode : {kNormOnly, kJoin, kJoinGated}) most = std::max(most, backward_grid(rows, residual_shape(width, halves), mode));
  return (size_t)most * 4 * (size_t)width * sizeof(float);
}

extern "C" int disco_residual_norm_backward(const disco_residual_norm* d, const float* stats, const disco_residual_norm_grads* g,
                                            void* workspace, size_t workspace_bytes, void* stream_) {
  const int rc = check_desc(d);
  if (rc != DISCO_OK) return rc;
  if (!g) return DISCO_EINVAL;
  const int64_t n = d->rows, F = d->width;
  if (!d->has_block && (g->dy || g->dgate || g->dscale || g->dpost_weight || g->dpost_bias || g->dout)) return DISCO_EINVAL;
  if ((g->dpost_weight && !d->post_weight) || (g->dpost_bias && !d->post_bias) || (g->dpre_weight && !d->pre_weight) ||
      (g->dpre_bias && !d->pre_bias) || (g->dscale && !d->scale_vector) || (g->dgate && !d->gate_kind) || (g->dh && !d->pre_norm))
    return DISCO_EINVAL;
  // out = x + scale * y: the gradient of y is that of out, scaled
  const bool reads_y = d->post_norm || d->gate_kind || d->scale_vector || g->dh;
  ResidualArgs a;
  fill(d, &a);
  const bool channel = d->gate_kind == DISCO_GATE_CHANNEL;
  const bool branch = g->dscale || (channel && g->dgate);
  a.partials = (g->dpost_weight || branch ? 1 : 0) | (g->dpost_bias || (branch && d->post_bias) ? 2 : 0) | (g->dpre_weight ? 4 : 0) |
               (g->dpre_bias ? 8 : 0);
  if (n > 0) {
    if ((g->dx && !strided(g->ld_dx, n, F)) || (g->dy && !strided(g->ld_dy, n, F)) || (d->gate_kind == DISCO_GATE_FULL && g->dgate && !strided(g->ld_dgate, n, F)) ||
        (d->gate_kind == DISCO_GATE_ROW && g->dgate && g->ld_dgate < 1 && n > 1))
      return DISCO_EINVAL;
    if (d->ldx < 0 || d->ldy < 0 || d->ld_gate < 0 || g->ld_dout < 0 || g->ld_dh < 0) return DISCO_EINVAL;
    if ((d->has_block && !d->y && (reads_y || !g->dout)) || (g->dh && !d->x) || (d->gate_kind && !d->gate) || ((d->post_norm || g->dh) && !stats)) return DISCO_EINVAL;
  }
  const ResidualShape s = residual_shape(F, d->block_type != DISCO_F32);
  const unsigned grid = backward_grid(n, s, residual_mode(d->has_block, d->gate_kind));
  const size_t need = (size_t)grid * 4 * (size_t)F * sizeof(float);
  // The norm alone without a gradient of h: every gradient is zero, and neither x nor the statistics are there to be read.
  const bool nothing = !d->has_block && !g->dh;
  const int64_t summed = nothing ? 0 : n;
  if (a.partials && summed > 0 && (!workspace || workspace_bytes < need)) return DISCO_EWORKSPACE;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  a.stats = const_cast<float*>(stats);
  if (d->has_block && !a.y) {      // a row that is there, in place of one whose values go nowhere
    a.y = g->dout;
    a.ldy = 0;
  }
  a.dout = g->dout; a.lddo = g->ld_dout; a.dh = g->dh; a.lddh = g->ld_dh;
  a.dx = g->dx; a.lddx = g->ld_dx; a.dy = g->dy; a.lddy = g->ld_dy; a.dg = channel ? nullptr : g->dgate; a.lddg = g->ld_dgate;
  a.partial = a.partials ? static_cast<float*>(workspace) : nullptr;
  if (nothing && a.dx && n > 0) {
    const dim3 blocks((unsigned)std::min<int64_t>((n * F + 255) / 256, 4096));
    if (d->stream_type == DISCO_F32) hipLaunchKernelGGL(k_residual_zero<float>, blocks, dim3(256), 0, stream, static_cast<float*>(a.dx), n, F, a.lddx);
    else hipLaunchKernelGGL(k_residual_zero<_Float16>, blocks, dim3(256), 0, stream, static_cast<_Float16*>(a.dx), n, F, a.lddx);      // bfloat16 too
    DISCO_CHECK_LAUNCH();
  }
  if (summed > 0 && (a.dx || a.dy || a.dg || a.partials)) {
    int r;
    switch (pair_of(d->stream_type, d->block_type)) {
      case kPairF32: r = residual_backward<kPairF32>(a, grid, stream); break;
      case kPairF16: r = residual_backward<kPairF16>(a, grid, stream); break;
      case kPairBF16: r = residual_backward<kPairBF16>(a, grid, stream); break;
      case kPairF32F16: r = residual_backward<kPairF32F16>(a, grid, stream); break;
      default: r = residual_backward<kPairF32BF16>(a, grid, stream);
    }
    if (r != DISCO_OK) return r;
  }
  if (!a.partials) return DISCO_OK;
  FinishArgs f{};
  f.partial = a.partial; f.groups = summed > 0 ? grid : 0; f.width = (int)F; f.partials = a.partials; f.param_type = d->param_type;
  f.channel = channel; f.act = d->gate_act; f.scale = d->scale;
  f.w1 = d->post_weight; f.b1 = d->post_bias; f.lam = d->scale_vector; f.g = channel ? d->gate : nullptr;
  f.dw1 = g->dpost_weight; f.db1 = g->dpost_bias; f.dw2 = g->dpre_weight; f.db2 = g->dpre_bias; f.dlam = g->dscale;
  f.dg = channel ? g->dgate : nullptr;
  hipLaunchKernelGGL(k_residual_finish, dim3((unsigned)((F + 15) / 16)), dim3(1024), 0, stream, f);
  DISCO_CHECK_LAUNCH();
  return DISCO_OK;
}
