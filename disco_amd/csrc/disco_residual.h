// Kernels of the join between two residual blocks (forward and backward), one instantiation unit per pair of types.
//
//   z   = u1 * w1 + b1,  u1 = standardised row of y           (post norm: rms, layer or none -> z = y)
//   out = x + lam * a * z,  lam = scale (* channel gate),  a = act(gate) per element or per row
//   h   = u2 * w2 + b2,  u2 = standardised row of out         (pre norm of the next block: rms, layer or none)
//
// Backward, with q = dh * w2 and m(.) the mean over the row:
//   dO = dout + r2 * (q - m(q) - u2 * m(q * u2))              (rms: without the m(q) term)
//   dx = dO,  p = dO * a * lam * w1,  dy = r1 * (p - m(p) - u1 * m(p * u1)),  dgate = dO * lam * z * a'
//   Every parameter gradient is a column sum, and four of them are enough:
//   P1 = sum dO * a * u1,  P2 = sum dO * a,  P3 = sum dh * u2,  P4 = sum dh   (k_residual_finish derives the rest).
//
// Both directions are bound by memory (about 20 and 40 operations for 20 to 40 bytes): a row is read once into registers,
// all its reductions run there, and each output is written once.  Statistics and sums are float32 whatever the types;
// values are rounded once, when they are stored.  The next block's norm reads the unrounded sum, not the stored one: its
// only rounding is then its own, and the backward, which rebuilds the sum from x and y, sees the same values.
#ifndef DISCO_RESIDUAL_H
#define DISCO_RESIDUAL_H

#include <type_traits>

#include "disco_internal.h"

namespace disco {

struct ResidualArgs {
  int64_t rows, ldx, ldy, ldg, ldo, ldh;
  int64_t lddo, lddh, lddx, lddy, lddg;
  int width, param_type, post, pre, gate, act;
  float scale, eps, inv_width;
  const void *x, *y, *g, *w1, *b1, *w2, *b2, *lam;
  void *out, *h;
  float* stats;                     // [4, rows]: mean and 1 / deviation of y, then of the sum; NULL: not kept
  const void *dout, *dh;
  void *dx, *dy, *dg;
  float* partial;                   // [workgroups, 4, width]: column sums of each workgroup; NULL: no parameter gradient
  int partials;                     // bit k: sum P(k+1) is wanted
};

enum ResidualPair { kPairF32 = 0, kPairF16 = 1, kPairBF16 = 2, kPairF32F16 = 3, kPairF32BF16 = 4 };

// A kernel variant: lanes per row and elements a lane holds.  A row takes the first variant that holds it.  Blocks of 16
// bits take eight elements a lane where float32 takes four, and half the lanes: the same bytes in flight for each wave
// (HALVES).
struct ResidualShape { int lanes, elems; };
constexpr ResidualShape kResidualShapes[] = {{4, 4}, {8, 4}, {16, 4}, {32, 4}, {64, 4}, {64, 8}, {64, 12}, {64, 16}, {128, 12},
                                             {256, 8}, {256, 12}, {256, 16}, {512, 12}, {512, 16}, {1024, 16}};
constexpr ResidualShape residual_shape(int64_t width, bool halves) {
  for (const ResidualShape& s : kResidualShapes)
    if (width <= (int64_t)s.lanes * s.elems) return halves && s.elems == 4 ? ResidualShape{s.lanes / 2, 8} : s;
  return {0, 0};
}
// the smallest width of a variant: vectors inside it need no check
constexpr int residual_least(int lanes, int elems) {
  int least = 1;
  for (const ResidualShape& s : kResidualShapes) {
    if ((s.lanes == lanes && s.elems == elems) || (s.elems == 4 && s.lanes == 2 * lanes && elems == 8)) break;
    least = s.lanes * s.elems + 1;
  }
  return least;
}

// lanes of a workgroup: four rows of a wave or more of less, or one row that takes several waves
constexpr int residual_threads(int lanes) { return lanes > 64 ? lanes : 256; }
// What a launch is for: the norm of x alone, the join, or the join with a gate for each element.  (One kernel for all three
// would hold the registers of the last: the norm needs half of them.)
enum ResidualMode { kNormOnly = 0, kJoin = 1, kJoinGated = 2 };
inline int residual_mode(bool block, int gate) { return !block ? kNormOnly : gate == DISCO_GATE_FULL ? kJoinGated : kJoin; }
// ... of the backward: waves of a SIMD, which share its 512 registers.  An element of a lane needs 10 to 15 of them in the join and
// 12 to 16 with a gate of its own, beside some 25 that every variant needs: four waves at 4 elements, four at 8 (three gated),
// three at 12 (two gated, two where a row's sums pass through LDS of four waves and more), two at 16.  The norm alone needs 7 an
// element and has room for four; from 12 on it measured faster with fewer, but for rows of eight waves (512 lanes).  One call's gradients over 60 M elements, us, with the number taken | with its neighbour:
//   norm   float32 rows of 602 (12 elements) 151 with 3 | 162 with 4, of 1000 (16) 155 with 2 | 161 with 3;
//          half rows of 1433 (128 lanes, 12) 99 with 2 | 110 with 3, of 5000 (512 lanes, 12) 88 with 4 | 130 with 2
//   join   float32 rows of 2500 (256 lanes, 12) 295 with 2 | 385 with 3, of 602 307 with 3 | 301 with 2; half rows of 602 169 with 3 |
//          182 with 2, of 4096 (16) 165 with 2 | 223 with 1; a float32 stream with bfloat16 blocks of 1200 281 with 3 | 230 with 2
//   gated  float32 rows of 602 392 with 2 | 459 with 3, of 1800 (256 lanes, 8) 408 with 3 | 412 with 4, of 4096 379 with 2 | 440 with 1
// Where a neighbour is ahead here it spills less: 12 elements in three waves put 1 to 24 registers into scratch in most types,
// rows of up to 32 half values (8 elements, three or four waves) 13 to 32, 1024 lanes up to 311; no other variant more than 10.
constexpr int residual_back_waves(int lanes, int elems, int mode) {
  return lanes == 1024 || elems <= 4 ? 4
         : mode == kNormOnly ? (elems <= 8 ? 4 : elems > 12 || lanes == 128 ? 2 : lanes == 512 ? 4 : 3)
         : lanes == 512 || elems > 12 ? 2 : elems <= 8 ? 4 - (mode == kJoinGated) : 3 - (lanes == 256 || mode == kJoinGated);
}
constexpr int residual_back_threads(int lanes, int elems, int mode) { return lanes > 64 ? lanes : 256 * residual_back_waves(lanes, elems, mode); }

// grid: workgroups; a workgroup takes rows / (its rows at a time * grid) turns
template <int PAIR> int residual_forward(const ResidualArgs& a, unsigned grid, hipStream_t stream);
template <int PAIR> int residual_backward(const ResidualArgs& a, unsigned grid, hipStream_t stream);

#if defined(DISCO_RESIDUAL_KERNELS)

__device__ __forceinline__ float activate(float g, int act) {
  // the reciprocal instruction (1 ulp) rather than a division: a gate for each element is arithmetic that shows
  if (act == DISCO_ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + expf(-g));
  if (act == DISCO_ACT_TANH) return tanhf(g);
  return g;
}
// A gate as the backward keeps it: in one register, from which the activation a and its slope both come without cancellation.
// Sigmoid: the smaller of a and 1 - a, which is e / (1 + e) with e = exp(-|g|), its sign bit set where a is the larger; the
// slope is their product.  (From a alone, 1 - a has lost 4 digits at g = 8 and everything at 18.)  Tanh keeps its value, and
// 1 - a * a what that leaves, as torch's does.
__device__ __forceinline__ float gate_code(float g, int act) {
  if (act == DISCO_ACT_SIGMOID) {
    const float e = expf(-fabsf(g));
    return __uint_as_float(__float_as_uint(-e * __builtin_amdgcn_rcpf(1.0f + e)) ^ (__float_as_uint(g) & 0x80000000u));
  }
  return act == DISCO_ACT_TANH ? tanhf(g) : g;
}
// `one`: the bits of 1.0 for a sigmoid, 0 otherwise
__device__ __forceinline__ float gate_value(float c, int one) { return c + __int_as_float((__float_as_int(c) >> 31) & one); }
__device__ __forceinline__ float gate_slope(float c, int act) {
  if (act == DISCO_ACT_SIGMOID) return fabsf(c) * (1.0f - fabsf(c));
  if (act == DISCO_ACT_TANH) return 1.0f - c * c;
  return 1.0f;
}

// One lane's part of a row: vectors of four elements, `lanes` vectors apart.  Rows may start at any element: the vector
// type asks for the element's alignment only, which global memory instructions allow.  ODD: the width is no multiple of
// four, so the row's last vector is partial.
template <typename T, int LANES, int E, bool ODD>
struct RowPart {
  static constexpr int LEAST = residual_least(LANES, E);
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  // No branch around a load, so that all of a row's are in flight together (behind branches half rows of 1434 moved
  // 2.9 TB/s, of 1436 4.1): a vector that reaches behind the row is read from the row's end instead and shifted down;
  // elements behind the width are zero.
  struct Raw { vec v[E / 4]; };
  __device__ static __forceinline__ Raw fetch(const T* p, int lane, int width) {
    Raw r;
    if (LEAST == 1 && ODD && width < 4) {
      const int c = lane * 4;
#pragma unroll
      for (int k = 0; k < E / 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[k][e] = k == 0 && c + e < width ? p[c + e] : (T)0.0f;
      return r;
    }
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      const int c = (k * LANES + lane) * 4;
      r.v[k] = *reinterpret_cast<const vec*>(p + ((k + 1) * LANES * 4 <= LEAST ? c : min(c, width - 4)));
    }
    return r;
  }
  __device__ static __forceinline__ void expand(const Raw& raw, float (&r)[E], int lane, int width) {
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      float t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = (float)raw.v[k][e];
      if ((k + 1) * LANES * 4 > LEAST && !(LEAST == 1 && ODD && width < 4)) {
        const int over = (k * LANES + lane) * 4 + 4 - width;      // elements of this vector behind the row, if positive
        if (ODD) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float u = over <= 0 ? t[e] : 0.0f;
            if (e < 3) u = over == 1 ? t[e < 3 ? e + 1 : 3] : u;
            if (e < 2) u = over == 2 ? t[e < 2 ? e + 2 : 3] : u;
            if (e < 1) u = over == 3 ? t[3] : u;
            t[e] = u;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) t[e] = over <= 0 ? t[e] : 0.0f;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) r[4 * k + e] = t[e];
    }
  }
  __device__ static __forceinline__ void load(float (&r)[E], const T* p, int lane, int width) { expand(fetch(p, lane, width), r, lane, width); }
  __device__ static __forceinline__ void store(const float (&r)[E], T* p, int lane, int width) {
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      const int c = (k * LANES + lane) * 4;
      vec v;
      v.x = (T)r[4 * k]; v.y = (T)r[4 * k + 1]; v.z = (T)r[4 * k + 2]; v.w = (T)r[4 * k + 3];
      if (c + 4 <= width) {
        *reinterpret_cast<vec*>(p + c) = v;
      } else if (ODD && c < width) {
        p[c] = v.x;
        if (c + 1 < width) p[c + 1] = v.y;
        if (c + 2 < width) p[c + 2] = v.z;
      }
    }
  }
};

// Adds the value of a partner lane: within 16 lanes through the adder's own lane permutations, beyond through the row and
// half swaps (both results of a swap of a value with itself add up to the pair's sum).  Every lane of a pair adds the same
// two numbers, so all lanes of a row end with the same bits.  (Shuffles through LDS cost about 100 cycles a step, six steps a
// sum and up to three sums a row: with them the trained join of 25000 x 602 took 216 us instead of 165 us.)
template <int CTRL> __device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float add_swap16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_swap32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sums R values over the lanes of a row, the same in every lane.  The order is fixed: results do not vary from run to run.
template <int LANES, int R>
__device__ __forceinline__ void row_sum(float (&v)[R], float4* lds, int& turn) {
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = add_dpp<0xB1>(v[r]);       // quad_perm [1, 0, 3, 2]
  if constexpr (LANES >= 4)
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = add_dpp<0x4E>(v[r]);     // quad_perm [2, 3, 0, 1]
  if constexpr (LANES >= 8)
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = add_dpp<0x141>(v[r]);    // row_half_mirror
  if constexpr (LANES >= 16)
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = add_dpp<0x140>(v[r]);    // row_mirror
  if constexpr (LANES >= 32)
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = add_swap16(v[r]);
  if constexpr (LANES >= 64)
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = add_swap32(v[r]);
  if constexpr (LANES > 64) {
    constexpr int WAVES = LANES / 64;
    // two buffers in turn: a wave that is ahead by one reduction writes the other one, and cannot be ahead by two
    float4* part = lds + turn * WAVES;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = make_float4(v[0], R > 1 ? v[R > 1 ? 1 : 0] : 0.0f, R > 2 ? v[R > 2 ? 2 : 0] : 0.0f, 0.0f);
    __syncthreads();
    float4 s = part[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const float4 t = part[w];
      s.x += t.x; s.y += t.y; s.z += t.z;
    }
    v[0] = s.x;
    if constexpr (R > 1) v[1] = s.y;
    if constexpr (R > 2) v[2] = s.z;
  }
}

template <int E, int LANES>
__device__ __forceinline__ bool in_row(int e, int lane, int width) { return ((e >> 2) * LANES + lane) * 4 + (e & 3) < width; }

// Standardises a row in place and returns (mean, 1 / deviation).  The variance is summed from the deviations, after the
// mean: subtracting two large sums would lose it.  Elements behind the width stay zero.
template <int LANES, int E>
__device__ __forceinline__ void standardise(float (&v)[E], int kind, float eps, float inv_width, int lane, int width, float4* lds,
                                            int& turn, float& mean, float& rstd) {
  float s[1] = {0.0f};
  mean = 0.0f;
  if (kind == DISCO_NORM_LAYER) {
#pragma unroll
    for (int e = 0; e < E; ++e) s[0] += v[e];
    row_sum<LANES, 1>(s, lds, turn);
    mean = s[0] * inv_width;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = in_row<E, LANES>(e, lane, width) ? v[e] - mean : 0.0f;
    s[0] = 0.0f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s[0] = fmaf(v[e], v[e], s[0]);
  row_sum<LANES, 1>(s, lds, turn);
  rstd = 1.0f / sqrtf(fmaf(s[0], inv_width, eps));
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] *= rstd;
}

// A parameter vector, `other` where it is absent; zero behind the width.
template <int LANES, int E, bool ODD>
__device__ __forceinline__ void load_vector(const void* p, int type, int lane, int width, float other, float (&v)[E]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = other;
  } else if (type == DISCO_F32) {
    RowPart<float, LANES, E, ODD>::load(v, static_cast<const float*>(p), lane, width);
  } else if (type == DISCO_F16) {
    RowPart<_Float16, LANES, E, ODD>::load(v, static_cast<const _Float16*>(p), lane, width);
  } else {
    RowPart<__bf16, LANES, E, ODD>::load(v, static_cast<const __bf16*>(p), lane, width);
  }
}

// z = u1 * A + B with the residual scale and a channel gate folded in (A = lam * w1, B = lam * b1): loaded once per workgroup.
template <int LANES, int E, bool ODD>
__device__ __forceinline__ void load_branch(const ResidualArgs& a, int lane, float (&A)[E], float (&B)[E]) {
  float g[E], lam[E];
  load_vector<LANES, E, ODD>(a.w1, a.param_type, lane, a.width, 1.0f, A);
  load_vector<LANES, E, ODD>(a.b1, a.param_type, lane, a.width, 0.0f, B);
  load_vector<LANES, E, ODD>(a.lam, a.param_type, lane, a.width, 1.0f, lam);
  load_vector<LANES, E, ODD>(a.gate == DISCO_GATE_CHANNEL ? a.g : nullptr, a.param_type, lane, a.width, 1.0f, g);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float l = a.scale * lam[e];
    if (a.gate == DISCO_GATE_CHANNEL) l *= activate(g[e], a.act);
    A[e] *= l;
    B[e] *= l;
  }
}

template <typename TX, typename TY, int MODE, int LANES, int E, bool ODD>
__global__ __launch_bounds__(residual_threads(LANES)) void k_residual_forward(const ResidualArgs a) {
  constexpr int THREADS = residual_threads(LANES), ROWS = THREADS / LANES;
  constexpr bool BLOCK = MODE != kNormOnly, FULL = MODE == kJoinGated;
  typedef RowPart<TX, LANES, E, ODD> PX;
  typedef RowPart<TY, LANES, E, ODD> PY;
  __shared__ float4 lds[LANES > 64 ? 2 * (LANES / 64) : 1];
  const int lane = threadIdx.x % LANES;
  int turn = 0;
  float A[E], B[E], W2[E], B2[E];
  if constexpr (BLOCK) load_branch<LANES, E, ODD>(a, lane, A, B);
  if (!BLOCK || a.pre) {
    load_vector<LANES, E, ODD>(a.w2, a.param_type, lane, a.width, 1.0f, W2);
    load_vector<LANES, E, ODD>(a.b2, a.param_type, lane, a.width, 0.0f, B2);
  }
  for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
    // all of the row's loads, before any of them is waited for
    typename PY::Raw ry, rg;
    float o[E], z[E], g[E], grow = 1.0f;
    const typename PX::Raw rx = PX::fetch(static_cast<const TX*>(a.x) + row * a.ldx, lane, a.width);
    if constexpr (BLOCK) {
      ry = PY::fetch(static_cast<const TY*>(a.y) + row * a.ldy, lane, a.width);
      if constexpr (FULL) rg = PY::fetch(static_cast<const TY*>(a.g) + row * a.ldg, lane, a.width);
      else if (a.gate == DISCO_GATE_ROW) grow = (float)static_cast<const TY*>(a.g)[row * a.ldg];
    }
    PX::expand(rx, o, lane, a.width);
    if constexpr (BLOCK) {
      PY::expand(ry, z, lane, a.width);
      if constexpr (FULL) PY::expand(rg, g, lane, a.width);
      if (!FULL && a.gate == DISCO_GATE_ROW) grow = activate(grow, a.act);
      if (a.post) {
        float mean, rstd;
        standardise<LANES, E>(z, a.post, a.eps, a.inv_width, lane, a.width, lds, turn, mean, rstd);
        if (a.stats && lane == 0) { a.stats[row] = mean; a.stats[a.rows + row] = rstd; }
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float t = fmaf(z[e], A[e], B[e]);
        if constexpr (FULL) t *= activate(g[e], a.act);
        else t *= grow;
        o[e] += t;
      }
      PX::store(o, static_cast<TX*>(a.out) + row * a.ldo, lane, a.width);
    }
    if (!BLOCK || a.pre) {
      float mean, rstd;
      standardise<LANES, E>(o, a.pre, a.eps, a.inv_width, lane, a.width, lds, turn, mean, rstd);
      if (a.stats && lane == 0) { a.stats[2 * a.rows + row] = mean; a.stats[3 * a.rows + row] = rstd; }
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], W2[e], B2[e]);
      PY::store(o, static_cast<TY*>(a.h) + row * a.ldh, lane, a.width);
    }
  }
}

// The backward holds a row's x, y, gate and both gradients and four running column sums per element.  The three parameter
// vectors that every row needs again stay in LDS (12 bytes an element beside the 20 to 32 that the row moves through memory):
// in registers they cost a third of the waves that a compute unit can hold.  Rows of a wave or less share a workgroup as
// large as the registers allow, since each workgroup leaves one partial row per sum behind for the finish to read.
template <typename TX, typename TY, int MODE, int LANES, int E, bool ODD>
__global__ __launch_bounds__(residual_back_threads(LANES, E, MODE), residual_back_waves(LANES, E, MODE)) void k_residual_backward(const ResidualArgs a) {
  constexpr bool BLOCK = MODE != kNormOnly, FULL = MODE == kJoinGated;
  constexpr int THREADS = residual_back_threads(LANES, E, MODE), ROWS = THREADS / LANES, W = LANES * E;
  __shared__ float4 lds[LANES > 64 ? 2 * (LANES / 64) : 1];
  // the vectors; after the last row, for rows of a wave or less, the column sums of the workgroup's row groups
  __shared__ float4 store[(W <= 8192 ? (ROWS > 3 ? ROWS : 3) * W : 4) / 4];
  // The code of a row's gate in a scalar register, decoded where it is used: the join has no vector register to spare (float32 rows
  // of 602: 262 us with code and value in vector registers, 252 so and before).  1024 lanes spill either way, and less without.
  constexpr bool SCALAR = MODE == kJoin && LANES >= 64 && LANES < 1024;
  const int one = a.act == DISCO_ACT_SIGMOID ? 0x3f800000 : 0;
  constexpr bool IN_LDS = W <= 8192, AHEAD = LANES == 512 && MODE == kJoin && (E == 12 || sizeof(TX) == 2);
  typedef RowPart<TX, LANES, E, ODD> PX;
  typedef RowPart<TY, LANES, E, ODD> PY;
  const int lane = threadIdx.x % LANES;
  int turn = 0;
  float regs[IN_LDS ? 1 : 3][E], P1[E], P2[E], P3[E], P4[E];
  {
    float A[E], B[E], W2[E];
    if (!IN_LDS || threadIdx.x < LANES) {
      if constexpr (BLOCK) load_branch<LANES, E, ODD>(a, lane, A, B);
      load_vector<LANES, E, ODD>(a.w2, a.param_type, lane, a.width, 1.0f, W2);
    }
    if constexpr (IN_LDS) {
      if (threadIdx.x < LANES)
#pragma unroll
        for (int k = 0; k < E / 4; ++k) {
          if constexpr (BLOCK) {
            store[k * LANES + lane] = make_float4(A[4 * k], A[4 * k + 1], A[4 * k + 2], A[4 * k + 3]);
            store[W / 4 + k * LANES + lane] = make_float4(B[4 * k], B[4 * k + 1], B[4 * k + 2], B[4 * k + 3]);
          }
          store[W / 2 + k * LANES + lane] = make_float4(W2[4 * k], W2[4 * k + 1], W2[4 * k + 2], W2[4 * k + 3]);
        }
      __syncthreads();
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (BLOCK) { regs[0][e] = A[e]; regs[1][e] = B[e]; }
        regs[2][e] = W2[e];
      }
    }
  }
  const auto vector = [&](int which, float (&v)[E]) {
    if constexpr (IN_LDS) {
#pragma unroll
      for (int k = 0; k < E / 4; ++k) {
        const float4 t = store[which * (W / 4) + k * LANES + lane];
        v[4 * k] = t.x; v[4 * k + 1] = t.y; v[4 * k + 2] = t.z; v[4 * k + 3] = t.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = regs[which][e];
    }
  };
#pragma unroll
  for (int e = 0; e < E; ++e) P1[e] = P2[e] = P3[e] = P4[e] = 0.0f;
  typename PX::Raw rx, rdo;
  typename PY::Raw ry, rg, rdh;
  float m1 = 0.0f, r1 = 1.0f, m2 = 0.0f, r2 = 1.0f, grow = 1.0f;
  // A row's loads, all before any of them is waited for; with a gate for each element in two parts, which takes fewer
  // registers (169343 x 256: 267 us, 281 in one).  AHEAD: the next row's are under way during this one's work -- for rows of
  // eight waves, of which a compute unit holds one (60 M elements in half rows of 5000: 186 us, 214 without; of 8192 160 and 178; a
  // float32 stream with bfloat16 blocks of 5000 212 and 246).
  const auto fetch = [&](int64_t row) {
    if constexpr (BLOCK) {
      ry = PY::fetch(static_cast<const TY*>(a.y) + row * a.ldy, lane, a.width);
      if constexpr (FULL) rg = PY::fetch(static_cast<const TY*>(a.g) + row * a.ldg, lane, a.width);
      else if (a.gate == DISCO_GATE_ROW) grow = (float)static_cast<const TY*>(a.g)[row * a.ldg];
      if (a.post) {
        m1 = a.stats[row];
        r1 = a.stats[a.rows + row];
      }
    }
  };
  const auto fetch_sum = [&](int64_t row) {
    if (!BLOCK || a.dh) {
      rx = PX::fetch(static_cast<const TX*>(a.x) + row * a.ldx, lane, a.width);
      rdh = PY::fetch(static_cast<const TY*>(a.dh) + row * a.lddh, lane, a.width);
      m2 = a.stats[2 * a.rows + row];
      r2 = a.stats[3 * a.rows + row];
    }
    if (BLOCK && a.dout) rdo = PX::fetch(static_cast<const TX*>(a.dout) + row * a.lddo, lane, a.width);
  };
  int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (AHEAD && row < a.rows) { fetch(row); fetch_sum(row); }
  while (row < a.rows) {
    if constexpr (IN_LDS) asm volatile("" ::: "memory");      // the vectors are read again, not kept in registers
    const int64_t next = row + (int64_t)gridDim.x * ROWS;
    if (!AHEAD) { fetch(row); if (!FULL) fetch_sum(row); }
    const typename PY::Raw cy = ry, cg = rg;
    const float mean1 = m1, rstd1 = r1;
    typename PX::Raw cx = rx, cdo = rdo;
    typename PY::Raw cdh = rdh;
    float mean2 = m2, rstd2 = r2;
    float u1[E], act[FULL ? E : 1], d[E], gate = grow;
    if (AHEAD && next < a.rows) { fetch(next); fetch_sum(next); }
    if constexpr (BLOCK) {
      PY::expand(cy, u1, lane, a.width);
      if (a.post)
#pragma unroll
        for (int e = 0; e < E; ++e) u1[e] = in_row<E, LANES>(e, lane, a.width) ? (u1[e] - mean1) * rstd1 : 0.0f;
      if constexpr (FULL) {
        PY::expand(cg, act, lane, a.width);
#pragma unroll
        for (int e = 0; e < E; ++e) act[e] = gate_code(act[e], a.act);
      } else {
        if (a.gate == DISCO_GATE_ROW) gate = gate_code(gate, a.act);
        if constexpr (SCALAR) gate = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(gate)));
        act[0] = SCALAR ? gate_value(gate, one) : a.act == DISCO_ACT_SIGMOID && signbit(gate) ? 1.0f + gate : gate;
      }
    }
    if (FULL) { fetch_sum(row); cx = rx; cdo = rdo; cdh = rdh; mean2 = m2; rstd2 = r2; }
    const auto gated = [&](int e) { return FULL ? gate_value(act[FULL ? e : 0], one) : act[0]; };
    if (BLOCK && a.dout) {
      PX::expand(cdo, d, lane, a.width);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = 0.0f;
    }
    if (!BLOCK || a.dh) {
      float s[2] = {0.0f, 0.0f}, W2[E], u2[E], q[E];
      PX::expand(cx, u2, lane, a.width);
      PY::expand(cdh, q, lane, a.width);
      vector(2, W2);
      if constexpr (BLOCK) {
        float A[E], B[E];
        vector(0, A);
        vector(1, B);
#pragma unroll
        for (int e = 0; e < E; ++e) u2[e] = fmaf(gated(e), fmaf(u1[e], A[e], B[e]), u2[e]);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        u2[e] = in_row<E, LANES>(e, lane, a.width) ? (u2[e] - mean2) * rstd2 : 0.0f;
        P3[e] = fmaf(q[e], u2[e], P3[e]);
        P4[e] += q[e];
        q[e] *= W2[e];
        s[0] = fmaf(q[e], u2[e], s[0]);
        s[1] += q[e];
      }
      row_sum<LANES, 2>(s, lds, turn);
      const float mq = a.pre == DISCO_NORM_LAYER ? s[1] * a.inv_width : 0.0f, mqu = s[0] * a.inv_width;
#pragma unroll
      for (int e = 0; e < E; ++e)
        d[e] += in_row<E, LANES>(e, lane, a.width) ? rstd2 * (q[e] - mq - u2[e] * mqu) : 0.0f;
    }
    if (a.dx) PX::store(d, static_cast<TX*>(a.dx) + row * a.lddx, lane, a.width);
    if constexpr (BLOCK) {
      float s[3] = {0.0f, 0.0f, 0.0f};
      float dg[FULL ? E : 1], A[E], B[E];
      if constexpr (SCALAR) {
        asm volatile("" : "+s"(gate));
        act[0] = gate_value(gate, one);
      }
      vector(0, A);
      vector(1, B);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float t = d[e] * fmaf(u1[e], A[e], B[e]);
        s[2] += t;
        if constexpr (FULL) dg[e] = t * gate_slope(act[e], a.act);
        d[e] *= gated(e);
        P1[e] = fmaf(d[e], u1[e], P1[e]);
        P2[e] += d[e];
        d[e] *= A[e];
        s[0] = fmaf(d[e], u1[e], s[0]);
        s[1] += d[e];
      }
      if constexpr (FULL)
        if (a.dg) PY::store(dg, static_cast<TY*>(a.dg) + row * a.lddg, lane, a.width);
      if (a.post || (!FULL && a.dg)) row_sum<LANES, 3>(s, lds, turn);
      if (!FULL && a.dg && lane == 0)
        static_cast<TY*>(a.dg)[row * a.lddg] = (TY)(s[2] * gate_slope(gate, a.act));
      if (a.dy) {
        if (a.post) {
          const float mp = a.post == DISCO_NORM_LAYER ? s[1] * a.inv_width : 0.0f, mpu = s[0] * a.inv_width;
#pragma unroll
          for (int e = 0; e < E; ++e) d[e] = rstd1 * (d[e] - mp - u1[e] * mpu);
        }
        PY::store(d, static_cast<TY*>(a.dy) + row * a.lddy, lane, a.width);
      }
    }
    row = next;
  }
  if (!a.partial) return;
  // column sums of the workgroup: its ROWS row groups in order, then one partial row per sum
  float* cols = reinterpret_cast<float*>(store);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!(a.partials >> k & 1)) continue;
    const float* P = k == 0 ? P1 : k == 1 ? P2 : k == 2 ? P3 : P4;
    float* to = a.partial + ((int64_t)blockIdx.x * 4 + k) * a.width;
    if constexpr (ROWS == 1) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (in_row<E, LANES>(e, lane, a.width)) to[((e >> 2) * LANES + lane) * 4 + (e & 3)] = P[e];
    } else {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) cols[(threadIdx.x / LANES) * W + ((e >> 2) * LANES + lane) * 4 + (e & 3)] = P[e];
      __syncthreads();
      for (int c = threadIdx.x; c < a.width; c += THREADS) {
        float s = 0.0f;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) s += cols[r * W + c];
        to[c] = s;
      }
    }
  }
}

template <typename TX, typename TY, bool BACK, int LANES, int E>
int residual_launch(const ResidualArgs& a, unsigned grid, hipStream_t stream) {
  const int mode = residual_mode(a.y != nullptr, a.gate);
  const dim3 threads(BACK ? residual_back_threads(LANES, E, mode) : residual_threads(LANES));
  auto launch = [&](auto which, auto odd) {
    constexpr int M = decltype(which)::value;
    constexpr bool O = decltype(odd)::value;
    if constexpr (BACK) hipLaunchKernelGGL((k_residual_backward<TX, TY, M, LANES, E, O>), dim3(grid), threads, 0, stream, a);
    else hipLaunchKernelGGL((k_residual_forward<TX, TY, M, LANES, E, O>), dim3(grid), threads, 0, stream, a);
  };
  auto by_mode = [&](auto odd) {
    if (mode == kNormOnly) launch(std::integral_constant<int, kNormOnly>(), odd);
    else if (mode == kJoin) launch(std::integral_constant<int, kJoin>(), odd);
    else launch(std::integral_constant<int, kJoinGated>(), odd);
  };
  if (a.width % 4) by_mode(std::true_type());
  else by_mode(std::false_type());
  DISCO_CHECK_LAUNCH();
  return DISCO_OK;
}

template <typename TX, typename TY, bool BACK>
int residual_dispatch(const ResidualArgs& a, unsigned grid, hipStream_t stream) {
  constexpr bool HALVES = sizeof(TY) == 2;
  constexpr int N = HALVES ? 2 : 1;      // the five narrowest variants
  const ResidualShape s = residual_shape(a.width, HALVES);
  switch (s.lanes * 100 + s.elems) {
    case 400 / N + 4 * N: return residual_launch<TX, TY, BACK, 4 / N, 4 * N>(a, grid, stream);
    case 800 / N + 4 * N: return residual_launch<TX, TY, BACK, 8 / N, 4 * N>(a, grid, stream);
    case 1600 / N + 4 * N: return residual_launch<TX, TY, BACK, 16 / N, 4 * N>(a, grid, stream);
    case 3200 / N + 4 * N: return residual_launch<TX, TY, BACK, 32 / N, 4 * N>(a, grid, stream);
    case 6400 / N + 4 * N: return residual_launch<TX, TY, BACK, 64 / N, 4 * N>(a, grid, stream);
    case 6408: return residual_launch<TX, TY, BACK, 64, 8>(a, grid, stream);
    case 6412: return residual_launch<TX, TY, BACK, 64, 12>(a, grid, stream);
    case 6416: return residual_launch<TX, TY, BACK, 64, 16>(a, grid, stream);
    case 12812: return residual_launch<TX, TY, BACK, 128, 12>(a, grid, stream);
    case 25608: return residual_launch<TX, TY, BACK, 256, 8>(a, grid, stream);
    case 25612: return residual_launch<TX, TY, BACK, 256, 12>(a, grid, stream);
    case 25616: return residual_launch<TX, TY, BACK, 256, 16>(a, grid, stream);
    case 51212: return residual_launch<TX, TY, BACK, 512, 12>(a, grid, stream);
    case 51216: return residual_launch<TX, TY, BACK, 512, 16>(a, grid, stream);
    case 102416: return residual_launch<TX, TY, BACK, 1024, 16>(a, grid, stream);
  }
  return DISCO_EUNSUPPORTED;
}

#define DISCO_RESIDUAL_PAIR(PAIR, TX, TY)                                                                  \
  namespace disco {                                                                                        \
  template <> int residual_forward<PAIR>(const ResidualArgs& a, unsigned grid, hipStream_t stream) {        \
    return residual_dispatch<TX, TY, false>(a, grid, stream);                                              \
  }                                                                                                        \
  template <> int residual_backward<PAIR>(const ResidualArgs& a, unsigned grid, hipStream_t stream) {       \
    return residual_dispatch<TX, TY, true>(a, grid, stream);                                               \
  }                                                                                                        \
  }

#endif  // DISCO_RESIDUAL_KERNELS

}  // namespace disco
#endif
