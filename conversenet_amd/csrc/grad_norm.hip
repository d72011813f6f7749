// The norm over many gradients, and the gradients scaled to a largest norm.
//
//   norm = sqrt(sum_t sum_i g_ti^2)  or  max |g_ti|        out_t = g_t min(1, max_norm / (norm + 1e-6))
//
// Two passes over the elements, both bound by memory: a block per chunk of a tensor adds up squares, in 64 bits (a
// float32 square overflows above 1.8e19; the conversions and products are hidden behind the loads), then a block per
// chunk joins all blocks' sums, in the same order on every call, and scales.  (No launch of its own for the join, though
// n small tensors have n^2 sums to read that way: lists of 2000 tensors scale in 4.9 us a launch of 128 where the first pass
// takes 4.3, 10,000 in 7.8 and 50,000 in 23, 0.6 of 6.5 ms and 9 of 38 ms of the call, which its host work over the list
// bounds at any length.)  The tensors' addresses and sizes travel
// in the kernel arguments, kGnTensors at a time: no table has to be uploaded, and a recorded graph keeps its own.
#include <algorithm>
#include <vector>

#include "cvn_common.h"

namespace cvn {
namespace {

constexpr int kGnTensors = 128;  // 29 bytes each: 3.7 KB of the 4 KB a launch takes
constexpr int kGnThreads = 256;
constexpr int64_t kGnChunk = 8192;   // elements of a block at least
constexpr int64_t kGnBlocks = 2048;  // blocks of one large tensor: 8 per CU; every scaling block adds up as many sums

struct GnArgs {
  const void* src[kGnTensors];
  void* dst[kGnTensors];
  int64_t n[kGnTensors];
  uint32_t first[kGnTensors + 1];  // a tensor's first block in this launch
  uint8_t type[kGnTensors];
};

template <class T>
struct GnVec {
  typedef T v __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

template <bool INF>
__device__ __forceinline__ double gn_add(double s, double v) {
  if (!INF) return fma(v, v, s);
  v = fabs(v);
  return v > s || v != v ? v : s;  // a NaN stays
}
template <bool INF>
__device__ __forceinline__ double gn_join(double s, double v) {
  if (!INF) return s + v;
  return v > s || v != v ? v : s;
}

// The join over a block, in every thread.
template <bool INF>
__device__ __forceinline__ double gn_block(double s) {
  __shared__ double red[kGnThreads / 64];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s = gn_join<INF>(s, __shfl_xor(s, d));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = red[0];
#pragma unroll
  for (int i = 1; i < kGnThreads / 64; ++i) s = gn_join<INF>(s, red[i]);
  return s;
}

template <bool INF, class T>
__device__ __forceinline__ double gn_chunk(const T* p, int64_t n) {
  typedef typename GnVec<T>::v V;
  constexpr int W = 16 / sizeof(T);
  double s[4] = {0., 0., 0., 0.};
  const int64_t nv = n / W;
  int64_t i = threadIdx.x;
  for (; i + 3 * kGnThreads < nv; i += 4 * kGnThreads) {
    V v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = ((const V*)p)[i + j * kGnThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < W; ++e) s[j] = gn_add<INF>(s[j], (double)(float)v[j][e]);
  }
  for (; i < nv; i += kGnThreads) {
    const V v = ((const V*)p)[i];
#pragma unroll
    for (int e = 0; e < W; ++e) s[0] = gn_add<INF>(s[0], (double)(float)v[e]);
  }
  for (i = W * nv + threadIdx.x; i < n; i += kGnThreads) s[1] = gn_add<INF>(s[1], (double)(float)p[i]);
  return gn_join<INF>(gn_join<INF>(s[0], s[1]), gn_join<INF>(s[2], s[3]));
}

template <class T, bool NT>
__device__ __forceinline__ void gn_scale(const T* p, T* o, int64_t n, float f) {
  typedef typename GnVec<T>::v V;
  constexpr int W = 16 / sizeof(T);
  const int64_t nv = n / W;
  int64_t i = threadIdx.x;
  for (; i + 3 * kGnThreads < nv; i += 4 * kGnThreads) {
    V v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = ((const V*)p)[i + j * kGnThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < W; ++e) v[j][e] = (T)((float)v[j][e] * f);
      if (NT) __builtin_nontemporal_store(v[j], (V*)o + i + j * kGnThreads);
      else ((V*)o)[i + j * kGnThreads] = v[j];
    }
  }
  for (; i < nv; i += kGnThreads) {
    V v = ((const V*)p)[i];
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = (T)((float)v[e] * f);
    ((V*)o)[i] = v;
  }
  for (i = W * nv + threadIdx.x; i < n; i += kGnThreads) o[i] = (T)((float)p[i] * f);
}

template <class T>
__device__ __forceinline__ void gn_scale(const void* p, void* o, int64_t i0, int64_t n, float f, bool nt) {
  if (nt) gn_scale<T, true>((const T*)p + i0, (T*)o + i0, n, f);
  else gn_scale<T, false>((const T*)p + i0, (T*)o + i0, n, f);
}

// The tensor of a block and its chunk of it.
__device__ __forceinline__ int gn_find(const GnArgs& a, int nt, uint32_t blk) {
  int lo = 0, hi = nt;  // first[lo] <= blk < first[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (a.first[m] <= blk) lo = m;
    else hi = m;
  }
  return lo;
}

template <bool INF>
__global__ void __launch_bounds__(kGnThreads) k_gn_part(GnArgs a, int nt, int64_t chunk, double* part) {
  const int t = gn_find(a, nt, blockIdx.x);
  const int64_t i0 = (int64_t)(blockIdx.x - a.first[t]) * chunk, n = min(chunk, a.n[t] - i0);
  double s;
  if (a.type[t] == CVN_F32) s = gn_chunk<INF>((const float*)a.src[t] + i0, n);
  else if (a.type[t] == CVN_BF16) s = gn_chunk<INF>((const __bf16*)a.src[t] + i0, n);
  else s = gn_chunk<INF>((const _Float16*)a.src[t] + i0, n);
  s = gn_block<INF>(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <bool INF>
__device__ __forceinline__ double gn_norm(const double* part, int64_t np) {
  double s = 0.;
  for (int64_t i = threadIdx.x; i < np; i += kGnThreads) s = gn_join<INF>(s, part[i]);
  s = gn_block<INF>(s);
  return INF ? s : sqrt(s);
}

template <bool INF>
__global__ void __launch_bounds__(kGnThreads) k_gn_norm(const double* part, int64_t np, float* norm) {
  const double s = gn_norm<INF>(part, np);
  if (threadIdx.x == 0) *norm = (float)s;
}

// The blocks take the chunks of all tensors from the last one on (the tensors come in that order): what the first pass
// read last is still in the card's cache.
template <bool INF>
__global__ void __launch_bounds__(kGnThreads) k_gn_scale(GnArgs a, int nt, int64_t chunk, const double* part, int64_t np,
                                                         double max_norm, float* norm, bool stream) {
  const double s = gn_norm<INF>(part, np);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)s;
  const double c = max_norm / (s + 1e-6);
  const float f = c >= 1. ? 1.f : (float)c;  // a NaN norm makes every gradient NaN
  const int t = gn_find(a, nt, blockIdx.x);
  if (f == 1.f && a.src[t] == a.dst[t]) return;
  const int64_t i0 = (int64_t)(a.first[t + 1] - 1 - blockIdx.x) * chunk, n = min(chunk, a.n[t] - i0);
  if (a.type[t] == CVN_F32) gn_scale<float>(a.src[t], a.dst[t], i0, n, f, stream);
  else if (a.type[t] == CVN_BF16) gn_scale<__bf16>(a.src[t], a.dst[t], i0, n, f, stream);
  else gn_scale<_Float16>(a.src[t], a.dst[t], i0, n, f, stream);
}

int64_t gn_chunk_size(int64_t total) {
  const int64_t c = (total + kGnBlocks - 1) / kGnBlocks;
  return std::max(kGnChunk, (c + 2047) / 2048 * 2048);
}

struct GnPlan {
  int64_t chunk, blocks;
};

int gn_plan(const int64_t* numel, int64_t n, GnPlan* p) {
  if (n < 0 || (n > 0 && !numel)) return fail(CVN_ERR_ARG, "bad tensor list");
  int64_t total = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (numel[i] < 0 || numel[i] > ((int64_t)1 << 48)) return fail(CVN_ERR_ARG, "bad tensor size");
    total += numel[i];
    if (total > ((int64_t)1 << 48)) return fail(CVN_ERR_UNSUPPORTED, "more than 2^48 elements");
  }
  p->chunk = gn_chunk_size(total);
  p->blocks = 0;
  for (int64_t i = 0; i < n; ++i) p->blocks += (numel[i] + p->chunk - 1) / p->chunk;
  if (p->blocks > (int64_t)1 << 28) return fail(CVN_ERR_UNSUPPORTED, "too many tensors");
  return CVN_OK;
}

int gn_type_size(int type) { return type == CVN_F32 ? 4 : type == CVN_BF16 || type == CVN_F16 ? 2 : 0; }

// Outputs may be their own gradients; otherwise no output may share memory with a gradient or another output.
bool gn_overlap(const void* const* src, void* const* dst, const int64_t* numel, const int* types, int64_t n) {
  struct Range {
    uintptr_t lo, hi;
    bool out;
  };
  std::vector<Range> v;
  v.reserve(2 * (size_t)n);
  for (int64_t i = 0; i < n; ++i) {
    if (numel[i] == 0) continue;
    const uintptr_t bytes = (uintptr_t)numel[i] * gn_type_size(types[i]);
    v.push_back({(uintptr_t)dst[i], (uintptr_t)dst[i] + bytes, true});
    if (dst[i] != src[i]) v.push_back({(uintptr_t)src[i], (uintptr_t)src[i] + bytes, false});
  }
  std::sort(v.begin(), v.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
  uintptr_t out_end = 0, any_end = 0;
  for (const Range& r : v) {
    if (r.lo < out_end || (r.out && r.lo < any_end)) return true;
    any_end = std::max(any_end, r.hi);
    if (r.out) out_end = std::max(out_end, r.hi);
  }
  return false;
}

// From here on outputs are stored past the caches, which hold the gradients still to be read: 256 MB of float32 take
// 131 us (156 through the caches), 1.3 GB 722 us (749).  32 MB take 24-26 us either way, and fit the cache for what
// reads them next.
constexpr int64_t kGnStream = (int64_t)64 << 20;  // bytes

template <bool INF>
int gn_run(const void* const* src, void* const* dst, const int64_t* numel, const int* types, int64_t n, double max_norm,
           float* norm, double* part, const GnPlan& plan, hipStream_t st) {
  // Launches in turn, the scaling ones from the last tensor on.
  GnArgs a;
  int64_t bytes = 0;
  for (int64_t i = 0; i < n; ++i) bytes += numel[i] * gn_type_size(types[i]);
  for (int pass = 0; pass < (dst ? 2 : 1); ++pass) {
    int nt = 0;
    int64_t done = 0;
    uint32_t blocks = 0;
    for (int64_t k = 0; k <= n; ++k) {
      const int64_t i = pass ? n - 1 - k : k;
      const uint32_t nb = k < n ? (uint32_t)((numel[i] + plan.chunk - 1) / plan.chunk) : 0;
      if (nb) {
        a.src[nt] = src[i];
        a.dst[nt] = dst ? dst[i] : nullptr;
        a.n[nt] = numel[i];
        a.type[nt] = (uint8_t)types[i];
        a.first[nt] = blocks;
        blocks += nb;
        a.first[++nt] = blocks;
      }
      if (nt == 0 || (nt < kGnTensors && k < n)) continue;
      if (pass == 0)
        hipLaunchKernelGGL(k_gn_part<INF>, dim3(blocks), dim3(kGnThreads), 0, st, a, nt, plan.chunk, part + done);
      else
        hipLaunchKernelGGL(k_gn_scale<INF>, dim3(blocks), dim3(kGnThreads), 0, st, a, nt, plan.chunk, part, plan.blocks,
                           max_norm, done == 0 ? norm : nullptr, bytes >= kGnStream);
      done += blocks;
      nt = 0;
      blocks = 0;
    }
  }
  if (!dst || plan.blocks == 0)
    hipLaunchKernelGGL(k_gn_norm<INF>, dim3(1), dim3(kGnThreads), 0, st, part, plan.blocks, norm);
  return check_launch(dst ? "clip_grads" : "grad_norm");
}

int gn_entry(const void* const* src, void* const* dst, bool clip, const int64_t* numel, const int* types, int64_t n,
             int norm_kind, double max_norm, float* norm, void* ws, size_t ws_bytes, hipStream_t st) {
  GnPlan plan;
  const int rc = gn_plan(numel, n, &plan);
  if (rc != CVN_OK) return rc;
  if (norm_kind != CVN_NORM_2 && norm_kind != CVN_NORM_INF) return fail(CVN_ERR_ARG, "bad norm kind");
  if (!norm || (n > 0 && (!src || !types || (clip && !dst)))) return fail(CVN_ERR_ARG, "null pointer");
  for (int64_t i = 0; i < n; ++i) {
    if (!gn_type_size(types[i])) return fail(CVN_ERR_ARG, "bad type of tensor %lld", (long long)i);
    if (numel[i] && (!src[i] || (clip && !dst[i]))) return fail(CVN_ERR_ARG, "null pointer");
  }
  if (clip && !(max_norm >= 0.)) return fail(CVN_ERR_ARG, "max_norm must be at least 0");
  if (clip && gn_overlap(src, dst, numel, types, n)) return fail(CVN_ERR_ARG, "outputs share memory");
  if (ws_bytes < sizeof(double) * (size_t)plan.blocks || (plan.blocks && !ws) || (uintptr_t)ws % sizeof(double))
    return fail(CVN_ERR_WORKSPACE, "workspace missing, too small or not aligned to 8 bytes");
  void* const* d = clip ? dst : nullptr;
  return norm_kind == CVN_NORM_INF ? gn_run<true>(src, d, numel, types, n, max_norm, norm, (double*)ws, plan, st)
                                   : gn_run<false>(src, d, numel, types, n, max_norm, norm, (double*)ws, plan, st);
}

}  // namespace
}  // namespace cvn

using namespace cvn;

extern "C" size_t cvn_grad_norm_workspace(const int64_t* numel, int64_t n) {
  GnPlan plan;
  if (gn_plan(numel, n, &plan) != CVN_OK) return 0;
  return sizeof(double) * (size_t)std::max<int64_t>(1, plan.blocks);
}

extern "C" int cvn_grad_norm(const void* const* grads, const int64_t* numel, const int* types, int64_t n, int norm_kind,
                             float* norm, void* workspace, size_t workspace_bytes, cvn_stream_t stream) {
  return gn_entry(grads, nullptr, false, numel, types, n, norm_kind, 0., norm, workspace, workspace_bytes,
                  (hipStream_t)stream);
}

extern "C" int cvn_clip_grads(const void* const* grads, void* const* out, const int64_t* numel, const int* types, int64_t n,
                              int norm_kind, double max_norm, float* norm, void* workspace, size_t workspace_bytes,
                              cvn_stream_t stream) {
  try {
    return gn_entry(grads, out, true, numel, types, n, norm_kind, max_norm, norm, workspace, workspace_bytes,
                    (hipStream_t)stream);
  } catch (const std::bad_alloc&) {
    return fail(CVN_ERR_HIP, "out of host memory");
  }
}
