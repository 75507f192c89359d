// disco_gradnorm.hip -- one norm over all gradients of a model, and the clipping it leads to (gfx950).
//
//   norm = (sum over every element of every tensor |g|^p)^(1/p), p = 1, 2 or infinity
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// Bound by memory: the norm reads every gradient once (201 M float32 values: 141 us, 5.7 TB/s), clipping reads it again, since
// no element may be scaled before the last one has been read, and writes it once.  The tensors are named in the launch's own
// arguments, 136 a launch, so that no table is copied to the device and a launch can be captured.  Sums are float64 per lane:
// squares of float32 values neither overflow nor vanish there, and one conversion and one fused add per element cost nothing
// next to the read.  Every sum has a fixed order: the norm is the same from run to run.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "disco_internal.h"

namespace disco {

// of a tensor, that a workgroup takes at a time: four loads of 16 bytes a lane (with two, bfloat16 came in at 4.4 TB/s
// instead of 5.2)
constexpr int kChunkBytes = 16384;
constexpr int kTensors = 136;            // tensors named by one launch: its arguments stay below 4 KiB
constexpr int kGroups = 8192;            // workgroups of one launch of the norm, at most
constexpr int kJoin = 2048;              // partial sums that every workgroup of the clipping joins for itself

struct Table {
  const void* src[kTensors];
  void* dst[kTensors];
  int64_t numel[kTensors];
  uint32_t end[kTensors];                // chunks up to and including this tensor
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

// fixed-order sum over the workgroup's lanes, in every lane
template <int P, int WAVES> __device__ __forceinline__ double norm_block(double s, double* lds) {
  for (int o = 32; o > 0; o >>= 1) s = norm_join<P>(s, __shfl_xor(s, o, 64));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  s = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s = norm_join<P>(s, lds[w]);
  return s;
}

// the chunks [first, last) of a workgroup: contiguous, so that the table is searched once
__device__ __forceinline__ void share(uint32_t chunks, uint32_t index, uint32_t& first, uint32_t& last) {
  first = (uint32_t)((uint64_t)chunks * index / gridDim.x);
  last = (uint32_t)((uint64_t)chunks * (index + 1) / gridDim.x);
}

template <typename T, int P>
__global__ __launch_bounds__(256) void k_norm_partial(const Table t, double* __restrict__ partial) {
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
  constexpr int V = 16 / sizeof(T), kChunk = kChunkBytes / sizeof(T);
  __shared__ double lds[4];
  uint32_t chunk, last;
  share(t.end[t.count - 1], blockIdx.x, chunk, last);
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
  s = norm_block<P, 4>(s, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

template <int P, int WAVES> __device__ __forceinline__ double norm_total(const double* __restrict__ partial, int64_t groups, double* lds) {
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < groups; i += WAVES * 64) s = norm_join<P>(s, partial[i]);
  return norm_block<P, WAVES>(s, lds);
}

template <int P>
__global__ __launch_bounds__(1024) void k_norm_finish(const double* __restrict__ partial, int64_t groups, double* __restrict__ joined,
                                                      float* __restrict__ norm) {
  __shared__ double lds[16];
  const double s = norm_total<P, 16>(partial, groups, lds);
  if (threadIdx.x == 0) {
    if (joined) *joined = s;
    if (norm) *norm = (float)(P == 2 ? sqrt(s) : s);
  }
}

template <typename T, typename U, int P>
__global__ __launch_bounds__(256) void k_clip(const Table t, const double* __restrict__ partial, int64_t groups,
                                              double max_norm, float* __restrict__ norm) {
  constexpr int V = 16 / sizeof(T), kChunk = kChunkBytes / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  typedef U uvec __attribute__((ext_vector_type(V), aligned(sizeof(U))));
  __shared__ double lds[4];
  // every workgroup joins the partial sums for itself, in the same order: no launch in between
  const double sum = norm_total<P, 4>(partial, groups, lds), total = P == 2 ? sqrt(sum) : sum;
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  const double want = max_norm / (total + 1e-6);
  // float64 like the norm: beside gradients near float32's end the factor is no normal float32.  A NaN norm stays NaN.
  const double factor = want >= 1.0 ? 1.0 : want;
  // from the end: what the norm read last still lies in the last-level cache
  uint32_t first, chunk;
  share(t.end[t.count - 1], gridDim.x - 1 - blockIdx.x, first, chunk);
  int k = t.count - 1;
  for (int lo = 0, hi = t.count - 1; lo <= hi;) {      // first tensor whose end lies at the share's end or behind it
    const int mid = (lo + hi) >> 1;
    if (t.end[mid] >= chunk) { k = mid; hi = mid - 1; } else lo = mid + 1;
  }
  while (chunk > first) {
    --chunk;
    while (k > 0 && t.end[k - 1] > chunk) --k;
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

static int64_t chunks_of(const Item& i) { return (i.numel * size_of(i.type) + kChunkBytes - 1) / kChunkBytes; }

static int64_t norm_groups(int64_t chunks) { return std::min<int64_t>(chunks, kGroups); }
// A workgroup for each chunk (up to 2^20), rather than few that walk far apart: they are dealt out in order, so memory is read
// and written in few places at a time (1.2 G values, bfloat16 to float32: 1.36 ms, with 16384 workgroups 1.49, with 2048 1.67,
// with 512 2.01).
static int64_t clip_groups(int64_t chunks) { return std::min<int64_t>(chunks, 1 << 20); }

template <typename F> static int by_type(int type, F&& f) {
  return type == DISCO_F32 ? f(float{}) : type == DISCO_F16 ? f(_Float16{}) : f(__bf16{});
}
template <typename F> static int by_norm(int norm_type, F&& f) {
  return norm_type == 2 ? f(std::integral_constant<int, 2>{}) : norm_type == 1 ? f(std::integral_constant<int, 1>{}) : f(std::integral_constant<int, 0>{});
}

struct Launch { size_t from, to; int64_t chunks; };

// runs of one type pair, cut where the table or the chunks' numbers end
static int cut(const std::vector<Item>& items, std::vector<Launch>* launches) {
  for (size_t b = 0; b < items.size();) {
    Launch l{b, b, 0};
    while (l.to < items.size() && l.to - b < (size_t)kTensors && items[l.to].type == items[b].type && items[l.to].out_type == items[b].out_type &&
           l.chunks + chunks_of(items[l.to]) < ((int64_t)1 << 31))
      l.chunks += chunks_of(items[l.to++]);
    if (l.to == b) return DISCO_EUNSUPPORTED;      // one tensor of 2^31 chunks: 32 TB
    launches->push_back(l);
    b = l.to;
  }
  return DISCO_OK;
}

static void fill(const std::vector<Item>& items, const Launch& l, Table* t) {
  uint32_t end = 0;
  t->count = (int)(l.to - l.from);
  for (size_t i = l.from; i < l.to; ++i) {
    t->src[i - l.from] = items[i].src;
    t->dst[i - l.from] = items[i].dst;
    t->numel[i - l.from] = items[i].numel;
    t->end[i - l.from] = end += (uint32_t)chunks_of(items[i]);
  }
}

static int gradient_norm(std::vector<Item>& items, int norm_type, bool clip, double max_norm, float* norm, void* ws, size_t ws_bytes,
                         hipStream_t stream) {
  double* partial = static_cast<double*>(ws);
  const int64_t room = (int64_t)(ws_bytes / sizeof(double));
  std::stable_sort(items.begin(), items.end(), [](const Item& a, const Item& b) { return a.type != b.type ? a.type < b.type : a.out_type < b.out_type; });
  std::vector<Launch> launches;
  const int rc = cut(items, &launches);
  if (rc != DISCO_OK) return rc;
  int64_t groups = 0;
  for (const Launch& l : launches) groups += norm_groups(l.chunks);
  if (groups + 1 > room) return DISCO_EWORKSPACE;
  Table t;
  int64_t at = 0;
  for (const Launch& l : launches) {
    fill(items, l, &t);
    const int64_t g = norm_groups(l.chunks);
    const int r = by_type(items[l.from].type, [&](auto v) -> int {
      return by_norm(norm_type, [&](auto p) -> int {
        hipLaunchKernelGGL((k_norm_partial<decltype(v), decltype(p)::value>), dim3((unsigned)g), dim3(256), 0, stream, t, partial + at);
        DISCO_CHECK_LAUNCH();
        return DISCO_OK;
      });
    });
    if (r != DISCO_OK) return r;
    at += g;
  }
  const bool only = !clip || items.empty();
  if (only || groups > kJoin) {
    const int r = by_norm(norm_type, [&](auto p) -> int {
      hipLaunchKernelGGL((k_norm_finish<decltype(p)::value>), dim3(1), dim3(1024), 0, stream, partial, groups, only ? nullptr : partial + groups,
                         only ? norm : nullptr);
      DISCO_CHECK_LAUNCH();
      return DISCO_OK;
    });
    if (r != DISCO_OK || only) return r;
    partial += groups;
    groups = 1;
  }
  for (size_t i = launches.size(); i-- > 0;) {
    const Launch& l = launches[i];
    if (launches.size() > 1) fill(items, l, &t);
    const int64_t g = clip_groups(l.chunks);
    float* to = i == 0 ? norm : nullptr;
    const int r = by_type(items[l.from].type, [&](auto v) -> int {
      return by_norm(norm_type, [&](auto p) -> int {
        auto launch = [&](auto u) -> int {
          hipLaunchKernelGGL((k_clip<decltype(v), decltype(u), decltype(p)::value>), dim3((unsigned)g), dim3(256), 0, stream, t, partial,
                             groups, max_norm, to);
          DISCO_CHECK_LAUNCH();
          return DISCO_OK;
        };
        return items[l.from].out_type == DISCO_F32 ? launch(float{}) : launch(v);
      });
    });
    if (r != DISCO_OK) return r;
  }
  return DISCO_OK;
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
  // launches are cut at 136 tensors, where one of the five type pairs ends, and at 2^31 chunks (32 TB); their joined sum
  return ((size_t)kGroups * (size_t)(n_tensors / kTensors + 5 + 1) + 1) * sizeof(double);
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
