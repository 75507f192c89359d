// disco_gradnorm.hip -- one norm over all gradients of a model, and the clipping it leads to (gfx950).
//
//   norm = (sum over every element of every tensor |g|^p)^(1/p), p = 1, 2 or infinity
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// Bound by memory: the norm reads every gradient once, clipping reads it again (no element may be scaled before the last
// one has been read) and writes it once.  The tensors are named in the launch's own arguments, up to a few hundred per
// launch, so that no table is copied to the device and a launch can be captured.  Sums are float64 per lane: squares of
// float32 values neither overflow nor vanish there, and one conversion and one fused add per element cost nothing next to
// the read.  Every sum has a fixed order: the norm is the same from run to run.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "disco_internal.h"

namespace disco {

constexpr int kChunk = 4096;             // elements a workgroup takes at a time
constexpr int kNormTensors = 190;        // tensors named by one launch: its arguments stay below 4 KiB
constexpr int kClipTensors = 136;
constexpr int kMostGroups = 2048;        // workgroups of one launch: eight per compute unit

template <int MOST> struct NormTable {
  const void* src[MOST];
  int64_t numel[MOST];
  uint32_t end[MOST];                    // chunks up to and including this tensor
  int count;
};
template <int MOST> struct ClipTable {
  const void* src[MOST];
  void* dst[MOST];
  int64_t numel[MOST];
  uint32_t end[MOST];
  int count;
};

template <int P> __device__ __forceinline__ double norm_add(double s, float v) {
  if (P == 2) return fma((double)v, (double)v, s);
  const double a = fabs((double)v);
  if (P == 1) return s + a;
  return (a > s || a != a) ? a : s;      // a NaN stays: nothing compares greater than it
}
template <int P> __device__ __forceinline__ double norm_join(double s, double t) {
  if (P != 0) return s + t;
  return (t > s || t != t) ? t : s;
}

// fixed-order sum over the workgroup's 256 lanes, in every lane
template <int P> __device__ __forceinline__ double norm_block(double s, double* lds) {
  for (int o = 32; o > 0; o >>= 1) s = norm_join<P>(s, __shfl_xor(s, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  return norm_join<P>(norm_join<P>(lds[0], lds[1]), norm_join<P>(lds[2], lds[3]));
}

// the chunks [first, last) of a workgroup: contiguous, so that the table is searched once
__device__ __forceinline__ void share(uint32_t chunks, uint32_t& first, uint32_t& last) {
  first = (uint32_t)((uint64_t)chunks * blockIdx.x / gridDim.x);
  last = (uint32_t)((uint64_t)chunks * (blockIdx.x + 1) / gridDim.x);
}

template <typename T, int P>
__global__ __launch_bounds__(256) void k_norm_partial(const NormTable<kNormTensors> t, double* __restrict__ partial) {
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  constexpr int V = 16 / sizeof(T);
  __shared__ double lds[4];
  uint32_t chunk, last;
  share(t.end[t.count - 1], chunk, last);
  int k = 0;
  for (int lo = 0, hi = t.count - 1; lo <= hi;) {      // first tensor whose end lies behind the chunk
    const int mid = (lo + hi) >> 1;
    if (t.end[mid] > chunk) { k = mid; hi = mid - 1; } else lo = mid + 1;
  }
  double s = 0.0;
  for (; chunk < last; ++chunk) {
    while (t.end[k] <= chunk) ++k;
    const int64_t at = (int64_t)(chunk - (k ? t.end[k - 1] : 0)) * kChunk;
    const int64_t left = t.numel[k] - at;
    const T* p = static_cast<const T*>(t.src[k]) + at;
    if (left >= kChunk) {
      vec v[kChunk / (256 * V)];
#pragma unroll
      for (int i = 0; i < kChunk / (256 * V); ++i) v[i] = *reinterpret_cast<const vec*>(p + (i * 256 + threadIdx.x) * V);
#pragma unroll
      for (int i = 0; i < kChunk / (256 * V); ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) s = norm_add<P>(s, (float)v[i][e]);
    } else {
      for (int i = threadIdx.x; i < (int)left; i += 256) s = norm_add<P>(s, (float)p[i]);
    }
  }
  s = norm_block<P>(s, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

template <int P> __device__ __forceinline__ double norm_total(const double* __restrict__ partial, int groups, double* lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < groups; i += 256) s = norm_join<P>(s, partial[i]);
  s = norm_block<P>(s, lds);
  return P == 2 ? sqrt(s) : s;
}

template <int P> __global__ __launch_bounds__(256) void k_norm_finish(const double* __restrict__ partial, int groups, float* __restrict__ norm) {
  __shared__ double lds[4];
  const double s = norm_total<P>(partial, groups, lds);
  if (threadIdx.x == 0) *norm = (float)s;
}

template <typename T, typename U, int P>
__global__ __launch_bounds__(256) void k_clip(const ClipTable<kClipTensors> t, const double* __restrict__ partial, int groups,
                                              double max_norm, float* __restrict__ norm) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  typedef U uvec __attribute__((ext_vector_type(V), aligned(sizeof(U))));
  __shared__ double lds[4];
  // every workgroup joins the partial sums for itself, in the same order: no launch in between
  const double total = norm_total<P>(partial, groups, lds);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  const double want = max_norm / (total + 1e-6);
  // float64 like the norm: beside gradients near float32's end the factor is no normal float32.  A NaN norm stays NaN.
  const double factor = want >= 1.0 ? 1.0 : want;
  uint32_t chunk, last;
  share(t.end[t.count - 1], chunk, last);
  int k = 0;
  for (int lo = 0, hi = t.count - 1; lo <= hi;) {
    const int mid = (lo + hi) >> 1;
    if (t.end[mid] > chunk) { k = mid; hi = mid - 1; } else lo = mid + 1;
  }
  for (; chunk < last; ++chunk) {
    while (t.end[k] <= chunk) ++k;
    if (factor == 1.0 && t.src[k] == t.dst[k]) continue;      // in place and within the norm: nothing changes
    const int64_t at = (int64_t)(chunk - (k ? t.end[k - 1] : 0)) * kChunk;
    const int64_t left = t.numel[k] - at;
    const T* p = static_cast<const T*>(t.src[k]) + at;
    U* q = static_cast<U*>(t.dst[k]) + at;
    if (left >= kChunk) {
      vec v[kChunk / (256 * V)];
#pragma unroll
      for (int i = 0; i < kChunk / (256 * V); ++i) v[i] = *reinterpret_cast<const vec*>(p + (i * 256 + threadIdx.x) * V);
#pragma unroll
      for (int i = 0; i < kChunk / (256 * V); ++i) {
        uvec u;
#pragma unroll
        for (int e = 0; e < V; ++e) u[e] = (U)(float)((double)(float)v[i][e] * factor);
        *reinterpret_cast<uvec*>(q + (i * 256 + threadIdx.x) * V) = u;
      }
    } else {
      for (int i = threadIdx.x; i < (int)left; i += 256) q[i] = (U)(float)((double)(float)p[i] * factor);
    }
  }
}

struct Item { const void* src; void* dst; int64_t numel; int type, out_type; };

static int64_t size_of(int type) { return type == DISCO_F32 ? 4 : 2; }

// A destination may be its own source (in place) and overlap nothing else: two tensors that share memory would be scaled
// twice, or while they are read.
static bool overlap(const std::vector<Item>& items) {
  struct Span { uintptr_t from, to; bool written; };
  std::vector<Span> spans;
  spans.reserve(2 * items.size());
  for (const Item& i : items) {
    const uintptr_t s = reinterpret_cast<uintptr_t>(i.src), d = reinterpret_cast<uintptr_t>(i.dst);
    if (!(s == d && i.type == i.out_type)) spans.push_back({s, s + (uintptr_t)(i.numel * size_of(i.type)), false});
    spans.push_back({d, d + (uintptr_t)(i.numel * size_of(i.out_type)), true});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  uintptr_t any = 0, written = 0;
  for (const Span& s : spans) {
    if (s.from < written || (s.written && s.from < any)) return true;
    any = std::max(any, s.to);
    if (s.written) written = std::max(written, s.to);
  }
  return false;
}

static int64_t chunks_of(const Item& i) { return (i.numel + kChunk - 1) / kChunk; }

// Workgroups of the launches: what their chunks need, 2048 together at most, but at least 8 each.
static int64_t groups_of(int64_t chunks, int64_t all) {
  const int64_t part = all > kMostGroups ? std::max<int64_t>(8, chunks * kMostGroups / all) : chunks;
  return std::min(chunks, part);
}

// items of one type pair [b, e) -> launches of at most `most` tensors and 2^31 chunks
template <typename F> static int cut(const std::vector<Item>& items, size_t b, size_t e, int most, F&& launch) {
  while (b < e) {
    size_t c = b;
    int64_t chunks = 0;
    while (c < e && (int)(c - b) < most && chunks + chunks_of(items[c]) < ((int64_t)1 << 31)) chunks += chunks_of(items[c++]);
    if (c == b) return DISCO_EUNSUPPORTED;      // one tensor of 2^31 chunks: 16 TB
    const int rc = launch(b, c, chunks);
    if (rc != DISCO_OK) return rc;
    b = c;
  }
  return DISCO_OK;
}

template <typename F> static int by_type(int type, F&& f) {
  return type == DISCO_F32 ? f(float{}) : type == DISCO_F16 ? f(_Float16{}) : f(__bf16{});
}
template <typename F> static int by_norm(int norm_type, F&& f) {
  return norm_type == 2 ? f(std::integral_constant<int, 2>{}) : norm_type == 1 ? f(std::integral_constant<int, 1>{}) : f(std::integral_constant<int, 0>{});
}

static int gradient_norm(std::vector<Item>& items, int norm_type, bool clip, double max_norm, float* norm, void* ws, size_t ws_bytes,
                         hipStream_t stream) {
  double* partial = static_cast<double*>(ws);
  const int64_t room = (int64_t)(ws_bytes / sizeof(double));
  std::stable_sort(items.begin(), items.end(), [](const Item& a, const Item& b) { return a.type != b.type ? a.type < b.type : a.out_type < b.out_type; });
  int64_t all = 0, groups = 0;
  for (const Item& i : items) all += chunks_of(i);
  auto ranges = [&](bool both, auto&& f) -> int {
    for (size_t b = 0; b < items.size();) {
      size_t e = b;
      while (e < items.size() && items[e].type == items[b].type && (!both || items[e].out_type == items[b].out_type)) ++e;
      const int rc = f(b, e);
      if (rc != DISCO_OK) return rc;
      b = e;
    }
    return DISCO_OK;
  };
  int rc = ranges(false, [&](size_t b, size_t e) -> int {
    return cut(items, b, e, kNormTensors, [&](size_t from, size_t to, int64_t chunks) -> int {
      NormTable<kNormTensors> t;
      uint32_t end = 0;
      t.count = (int)(to - from);
      for (size_t i = from; i < to; ++i) {
        t.src[i - from] = items[i].src;
        t.numel[i - from] = items[i].numel;
        t.end[i - from] = end += (uint32_t)chunks_of(items[i]);
      }
      const int64_t g = groups_of(chunks, all);
      if (groups + g > room) return DISCO_EWORKSPACE;
      const int r = by_type(items[from].type, [&](auto v) -> int {
        return by_norm(norm_type, [&](auto p) -> int {
          hipLaunchKernelGGL((k_norm_partial<decltype(v), decltype(p)::value>), dim3((unsigned)g), dim3(256), 0, stream, t, partial + groups);
          DISCO_CHECK_LAUNCH();
          return DISCO_OK;
        });
      });
      groups += g;
      return r;
    });
  });
  if (rc != DISCO_OK) return rc;
  if (!clip || items.empty())
    return by_norm(norm_type, [&](auto p) -> int {
      hipLaunchKernelGGL((k_norm_finish<decltype(p)::value>), dim3(1), dim3(256), 0, stream, partial, (int)groups, norm);
      DISCO_CHECK_LAUNCH();
      return DISCO_OK;
    });
  return ranges(true, [&](size_t b, size_t e) -> int {
    return cut(items, b, e, kClipTensors, [&](size_t from, size_t to, int64_t chunks) -> int {
      ClipTable<kClipTensors> t;
      uint32_t end = 0;
      t.count = (int)(to - from);
      for (size_t i = from; i < to; ++i) {
        t.src[i - from] = items[i].src;
        t.dst[i - from] = items[i].dst;
        t.numel[i - from] = items[i].numel;
        t.end[i - from] = end += (uint32_t)chunks_of(items[i]);
      }
      const int64_t g = groups_of(chunks, all);
      float* to_norm = from == 0 ? norm : nullptr;
      return by_type(items[from].type, [&](auto v) -> int {
        return by_norm(norm_type, [&](auto p) -> int {
          auto launch = [&](auto u) -> int {
            hipLaunchKernelGGL((k_clip<decltype(v), decltype(u), decltype(p)::value>), dim3((unsigned)g), dim3(256), 0, stream, t, partial,
                               (int)groups, max_norm, to_norm);
            DISCO_CHECK_LAUNCH();
            return DISCO_OK;
          };
          return items[from].out_type == DISCO_F32 ? launch(float{}) : launch(v);
        });
      });
    });
  });
}

static int collect(const void* const* src, void* const* dst, const int64_t* numel, const int* type, const int* out_type, int64_t n,
                   std::vector<Item>* items) {
  if (n < 0 || (n > 0 && (!src || !numel || !type))) return DISCO_EINVAL;
  items->reserve((size_t)n);
  for (int64_t i = 0; i < n; ++i) {
    if (numel[i] < 0 || type[i] < DISCO_F32 || type[i] > DISCO_BF16) return DISCO_EINVAL;
    const int to = dst ? out_type[i] : type[i];
    if (to != type[i] && to != DISCO_F32) return DISCO_EINVAL;
    if (numel[i] == 0) continue;
    if (!src[i] || (dst && !dst[i])) return DISCO_EINVAL;
    items->push_back({src[i], dst ? dst[i] : nullptr, numel[i], type[i], to});
  }
  return DISCO_OK;
}

}  // namespace disco

using namespace disco;

extern "C" size_t disco_grad_norm_workspace_bytes(int64_t n_tensors) {
  if (n_tensors < 0) return 0;
  // at most 2048 groups in proportion to the chunks, 8 for each launch that is rounded up; a launch is cut at 190 tensors,
  // at a change of type (twice) and at 2^31 chunks
  return (size_t)(kMostGroups + 8 * (n_tensors / kNormTensors + 4 + 8)) * sizeof(double);
}

extern "C" int disco_grad_norm(const void* const* grads_host, const int64_t* numel_host, const int* type_host, int64_t n_tensors,
                               int norm_type, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (norm_type < 0 || norm_type > 2 || !norm || !workspace) return DISCO_EINVAL;
  try {
    std::vector<Item> items;
    const int rc = collect(grads_host, nullptr, numel_host, type_host, nullptr, n_tensors, &items);
    if (rc != DISCO_OK) return rc;
    return gradient_norm(items, norm_type, false, 0.0, norm, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
  } catch (...) {
    return DISCO_EUNSUPPORTED;      // out of host memory for the table
  }
}

extern "C" int disco_grad_clip(const void* const* grads_host, void* const* out_host, const int64_t* numel_host, const int* type_host,
                               const int* out_type_host, int64_t n_tensors, int norm_type, double max_norm, float* norm,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (norm_type < 0 || norm_type > 2 || !(max_norm >= 0.0) || !norm || !workspace || (n_tensors > 0 && (!out_host || !out_type_host)))
    return DISCO_EINVAL;
  try {
    std::vector<Item> items;
    const int rc = collect(grads_host, out_host, numel_host, type_host, out_type_host, n_tensors, &items);
    if (rc != DISCO_OK) return rc;
    if (overlap(items)) return DISCO_EINVAL;
    return gradient_norm(items, norm_type, true, max_norm, norm, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
  } catch (...) {
    return DISCO_EUNSUPPORTED;
  }
}
