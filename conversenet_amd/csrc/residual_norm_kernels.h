// The kernels of residual_norm.h for a pair of types: T of the residual stream (x, r, y), TH of the branch (h, gate).
#pragma once
#include <algorithm>

#include "residual_norm.h"

namespace cvn {
namespace {

// A lane's pixel of a tile: `off` elements from the tile's first (base), which is uniform.
struct RnPx {
  int64_t base, q;  // element of the tile's first pixel at channel 0; the pixel's index
  int64_t b;        // its sample
  int off;
  bool ok;          // false: a pixel behind the last, loaded again from the last one and not stored
};

__device__ __forceinline__ RnPx rn_px(const RnArgs& a, int64_t tile, int lane) {
  RnPx p;
  if (a.tps) {
    const int64_t b = (uint32_t)tile / (uint32_t)a.tps;
    const int64_t p0 = (tile - b * a.tps) * 64;
    p.ok = p0 + lane < a.HW;
    const int l = (int)min((int64_t)lane, a.HW - 1 - p0);
    p.b = b;
    p.base = b * a.C * a.HW + p0;
    p.off = l;
    p.q = b * a.HW + p0 + l;
    return p;
  }
  const int64_t q0 = tile * 64;
  p.ok = q0 + lane < a.total;
  p.q = min(q0 + lane, a.total - 1);
  const uint32_t hw = (uint32_t)a.HW;
  const uint32_t b0 = (uint32_t)q0 / hw, b = (uint32_t)p.q / hw;
  const int p0 = (int)((uint32_t)q0 - b0 * hw);
  p.b = b;
  p.base = (int64_t)b0 * a.C * a.HW + p0;
  p.off = (int)((b - b0) * (uint32_t)a.C * hw) + (int)((uint32_t)p.q - b * hw) - p0;
  return p;
}

template <class T>
__device__ __forceinline__ float rn_ld(const void* p, int64_t i) {
  return (float)((const T*)p)[i];
}

// ------------------------------------------------------------------------------------------------
// Up to 256 channels: a block per tile of 64 V pixels, its channels spread over the waves, NC to a wave, so that a
// tensor's part of a tile is read once, V pixels of a channel to a lane, and stays in registers (with a thread per
// pixel and the channels read again for each step 16 x 64 x 256 x 256 takes 2.7 ms forward and backward).  Memory is the
// bound: at that size, float32 with a scale, the forward moves 1.07 GB in 198-208 us (5.2 TB/s, a copy's rate) and the
// backward 1.61 GB in 308-330 us (4.9-5.2).  With 16-bit tensors the joins and conversions show: 8 x 64 x 256 x 256 bf16,
// per-sample gate and both norms, 64 us forward (4.2 TB/s; 56 into the same outputs each time, which the card's cache
// holds) and 102 us backward (3.9); without gate and branch norm 52 and 91.  At 128 channels a block of the backward is all
// a CU holds: 4 x 128 x 128 x 128, float32 with a bf16 branch and gate, 28 us forward (4.8 TB/s) and 55 us backward (3.6).
// ------------------------------------------------------------------------------------------------

// A lane's V pixels of a tile.  The last lanes of a sample's last tile move back to its last V pixels, of which the
// first `dup` are other lanes' too; `whole`: no lane of the tile does.
template <int V>
struct RnLane {
  int64_t base, q, b;  // element of the tile's first pixel at channel 0; index of the lane's first pixel; its sample
  uint32_t off;        // the lane's first pixel behind base
  int dup;
  bool whole;

  __device__ __forceinline__ RnLane(const RnArgs& a, int64_t tile, int lane) {
    if (V == 1) {
      const RnPx p = rn_px(a, tile, lane);
      base = p.base;
      q = p.q;
      b = p.b;
      off = (uint32_t)p.off;
      dup = p.ok ? 0 : 1;
      whole = a.tps ? (tile % a.tps + 1) * 64 <= a.HW : (tile + 1) * 64 <= a.total;
      return;
    }
    b = (uint32_t)tile / (uint32_t)a.tps;
    const int hw = (int)a.HW, first = (int)(tile - b * a.tps) * (64 * V), p0 = min(first, hw - V);
    const int l = min(first + lane * V, hw - V) - p0;
    off = (uint32_t)l;
    dup = first - p0 + lane * V - l;
    whole = first + 64 * V <= hw;
    base = b * a.C * a.HW + p0;
    q = b * a.HW + p0 + l;
  }
  __device__ __forceinline__ bool any() const { return dup < V; }
};

// Addresses need only be multiples of the type's size: a lane's V pixels start anywhere in rows of odd length.
template <class T, int V>
struct RnVec {
  typedef T v __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <class T>
struct RnVec<T, 1> {
  typedef T v;
};

// p is uniform, so that the address is a scalar and a 32-bit offset.
template <class T, int V>
__device__ __forceinline__ void rn_load(float (&o)[V], const T* p, uint32_t off) {
  p += off;
  if constexpr (V == 1) {
    o[0] = (float)*p;
  } else {
    const typename RnVec<T, V>::v t = *(const typename RnVec<T, V>::v*)p;
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = (float)t[j];
  }
}

template <class T, int V>
__device__ __forceinline__ void rn_store(T* p, uint32_t off, const float (&o)[V]) {
  p += off;
  if constexpr (V == 1) {
    *p = (T)o[0];
  } else {
    typename RnVec<T, V>::v t;
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = (T)o[j];
    *(typename RnVec<T, V>::v*)p = t;
  }
}

// The pixels of a lane that are its own.
template <class T, int V>
__device__ __forceinline__ void rn_store_own(T* p, const float (&o)[V], const RnLane<V>& px) {
  if (px.dup == 0) {
    rn_store<T, V>(p, px.off, o);
  } else {
#pragma unroll
    for (int j = 1; j < V; ++j)
      if (j >= px.dup) p[px.off + j] = (T)o[j];
  }
}

// A wave's channels of a tensor, from channel c0 on; those behind the n of this wave repeat its last.
template <class T, int V, int NC>
__device__ __forceinline__ void rn_load_all(float (&o)[NC][V], const void* p, const RnLane<V>& px, int64_t HW, int c0,
                                            int n) {
  const T* t = (const T*)p + px.base + c0 * HW;
#pragma unroll
  for (int i = 0; i < NC; ++i) rn_load<T, V>(o[i], t + min(i, n - 1) * HW, px.off);
}

// The same as it was stored.
template <class T, int V, int NC>
__device__ __forceinline__ void rn_load_raw(typename RnVec<T, V>::v (&o)[NC], const void* p, const RnLane<V>& px,
                                            int64_t HW, int c0, int n) {
  const T* t = (const T*)p + px.base + c0 * HW;
#pragma unroll
  for (int i = 0; i < NC; ++i) o[i] = *(const typename RnVec<T, V>::v*)(t + min(i, n - 1) * HW + px.off);
}
template <class T, int V>
__device__ __forceinline__ float rn_at(const typename RnVec<T, V>::v& v, int j) {
  if constexpr (V == 1) return (float)v;
  else return (float)v[j];
}

template <int V>
__device__ __forceinline__ void rn_put(float* p, const float (&v)[V]) {
  if constexpr (V == 1) *p = v[0];
  else *(float2*)p = make_float2(v[0], v[1]);
}
template <int V>
__device__ __forceinline__ void rn_get(float (&v)[V], const float* p) {
  if constexpr (V == 1) {
    v[0] = *p;
  } else {
    const float2 t = *(const float2*)p;
    v[0] = t.x;
    v[1] = t.y;
  }
}

constexpr int kRnRed = 2 * 2 * 64;  // floats of red for each wave and pixel of a lane

// Two values per pixel over the waves of a block, which each wave joins in the order of the waves.  red: two buffers of
// nw 2 V 64 floats, taken in turn, so that one barrier a time is enough: a buffer is written again only after the
// barrier of the other, which a wave reaches after its reads.
template <int V>
__device__ __forceinline__ const float* rn_exchange(float* red, int& turn, int nw, int wave, int lane,
                                                    const float (&v)[2][V]) {
  float* buf = red + turn * nw * (kRnRed / 2 * V) + lane * V;
  turn ^= 1;
#pragma unroll
  for (int k = 0; k < 2; ++k) rn_put<V>(buf + (2 * wave + k) * (V * 64), v[k]);
  __syncthreads();
  return buf;
}

template <int V>
__device__ __forceinline__ void rn_block_sums(float* red, int& turn, int nw, int wave, int lane, float (&v)[2][V]) {
  if (nw == 1) return;
  const float* o = rn_exchange<V>(red, turn, nw, wave, lane, v);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) v[k][j] = 0.f;
  for (int w = 0; w < nw; ++w)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float t[V];
      rn_get<V>(t, o + (2 * w + k) * (V * 64));
#pragma unroll
      for (int j = 0; j < V; ++j) v[k][j] += t[j];
    }
}

// s / n, rounded as a division is (rn: 1 / n rounded).
__device__ __forceinline__ float rn_over(float s, float n, float rn) {
  const float u = s * rn;
  return fmaf(fmaf(-u, n, s), rn, u);
}

// mu and rho of a pixel's channels from each wave's mean and sum of squares about it (m), over count(w) channels: joined
// by the means' spread about the first wave's, so that no large mean cancels.
template <int V, class F>
__device__ __forceinline__ void rn_join(float* red, int& turn, int nw, int wave, int lane, float C, float rC, float eps,
                                        F count, float (&m)[2][V], float (&mu)[V], float (&rho)[V]) {
  if (nw > 1) {
    const float* o = rn_exchange<V>(red, turn, nw, wave, lane, m);
    float u[V], q[V], d[V] = {}, e[V] = {}, t[V];  // d, e: sums over the channels of the means' distances and squares
    rn_get<V>(u, o);
    rn_get<V>(q, o + V * 64);
    for (int w = 1; w < nw; ++w) {
      const float k = count(w);
      rn_get<V>(t, o + 2 * w * (V * 64));
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float v = t[j] - u[j], kv = k * v;
        d[j] += kv;
        e[j] = fmaf(kv, v, e[j]);
      }
      rn_get<V>(t, o + (2 * w + 1) * (V * 64));
#pragma unroll
      for (int j = 0; j < V; ++j) q[j] += t[j];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float v = rn_over(d[j], C, rC), w = fmaf(-d[j], v, e[j]);
      m[0][j] = u[j] + v;
      m[1][j] = q[j] + (w < 0.f ? 0.f : w);
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    mu[j] = m[0][j];
    rho[j] = rsqrtf(fmaf(m[1][j], rC, eps));
  }
}

// The same from the NC channels (n of them there) that each wave holds.
template <int V, int NC, bool FULL>
__device__ __forceinline__ void rn_block_moments(float* red, int& turn, int nw, int wave, int lane, int C, int n, float eps,
                                                 const float (&x)[NC][V], float (&mu)[V], float (&rho)[V]) {
  float m[2][V];
  const float fn = (float)n, rn = 1.f / fn, fC = (float)C, rC = 1.f / fC;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) s += i < n ? x[i][j] : 0.f;
    const float u = rn_over(s, fn, rn);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const float d = i < n ? x[i][j] - u : 0.f;
      q = fmaf(d, d, q);
    }
    m[0][j] = u;
    m[1][j] = q;
  }
  rn_join<V>(red, turn, nw, wave, lane, fC, rC, eps, [&](int w) { return FULL ? fn : (float)min(NC, C - w * NC); }, m, mu,
             rho);
}

// Sums over a wave's lanes of NC values at a time: each step halves the values a lane holds, sending the other half to
// the lane it is kept in, so NC sums take about NC + 6 operations; lane l ends with value l NC / 64.
__device__ __forceinline__ float rn_swap_add32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float rn_swap_add16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL>
__device__ __forceinline__ float rn_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// from lane l ^ 8, l ^ 7, l ^ 2, l ^ 1: together they reach all 16 lanes of a row
constexpr int kXor8 = 0x128, kXor7 = 0x141, kXor2 = 0x4e, kXor1 = 0xb1;
template <int CTRL>
__device__ __forceinline__ float rn_swap_add(float a, float b, bool upper) {
  return (upper ? b : a) + rn_dpp<CTRL>(upper ? a : b);
}

template <int NC>
__device__ __forceinline__ float rn_lane_sums(float (&v)[NC], int lane) {
  static_assert(NC == 8 || NC == 16, "");
#pragma unroll
  for (int i = 0; i < NC / 2; ++i) v[i] = rn_swap_add32(v[i], v[i + NC / 2]);
#pragma unroll
  for (int i = 0; i < NC / 4; ++i) v[i] = rn_swap_add16(v[i], v[i + NC / 4]);
#pragma unroll
  for (int i = 0; i < NC / 8; ++i) v[i] = rn_swap_add<kXor8>(v[i], v[i + NC / 8], lane & 8);
  if constexpr (NC == 16) v[0] = rn_swap_add<kXor7>(v[0], v[1], lane & 4);
  else v[0] += rn_dpp<kXor7>(v[0]);
  v[0] += rn_dpp<kXor2>(v[0]);
  return v[0] + rn_dpp<kXor1>(v[0]);
}

// What no kernel here writes, in the constant address space: its loads are scalar and need not wait for stores before
// them, which may be to the same memory for all the compiler knows (forward at 8 x 64 x 65536 bf16, gate and both norms:
// 64 us, 75 without).
template <class P>
__device__ __forceinline__ float rn_const(const P* p, int64_t i) {
  typedef const P __attribute__((address_space(4))) C;
  return (float)((C*)(uintptr_t)p)[i];
}

// Scale and, for a gate per sample, gate of a wave's channels (one branch for all of them, so that their loads are in
// flight together).
template <class TH, int NC, bool SAMPLE>
__device__ __forceinline__ void rn_factors(float (&k)[NC], const RnArgs& a, int64_t b, int c0, int n, bool sample = true) {
#pragma unroll
  for (int i = 0; i < NC; ++i) k[i] = 1.f;
  if (a.s) {
#pragma unroll
    for (int i = 0; i < NC; ++i) k[i] = rn_const(a.s, c0 + min(i, n - 1));
  }
  if (SAMPLE && a.gate && sample) {
#pragma unroll
    for (int i = 0; i < NC; ++i) k[i] *= rn_const((const TH*)a.gate, b * a.C + c0 + min(i, n - 1));
  }
}

// Blocks go to the 8 XCDs in turn; runs of 8 tiles to each keep the lines that two tiles share, where rows do not start
// on lines, in one L2 (64 channels of a photo of 321 x 481: forward 45 -> 40 us, backward 70 -> 65; 3 x 96 x 201 x 327 with
// gate and both norms: backward 163 -> 149).  Longer runs slow rows that do start on lines: an eighth of
// 16 x 64 x 256 x 256 to each XCD takes 219 us forward, against 202-207 us with runs of 8 or 1.
__device__ __forceinline__ int64_t rn_order(uint32_t b, uint32_t blocks) {
  if (b >= blocks / 64 * 64) return b;
  return b / 64 * 64 + b % 8 * 8 + b % 64 / 8;
}

template <class T, class TH, int V, int NC, bool FULL, bool POST, bool FG>
__global__ void __launch_bounds__(1024) k_rn_fwd(RnArgs a) {
  extern __shared__ __attribute__((aligned(16))) float red[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int C = (int)a.C, c0 = wave * NC, n = FULL ? NC : min(NC, C - c0);
  const RnLane<V> px(a, a.tile0 + rn_order(blockIdx.x, gridDim.x), lane);
  const int64_t HW = a.HW, at = px.base + c0 * HW;
  int turn = 0;
  // all loads first, as stored: a conversion would wait for its own
  typename RnVec<T, V>::v xr[NC];
  typename RnVec<TH, V>::v hr[NC], g[FG ? NC : 1];
  float k[NC];
  rn_load_raw<T, V, NC>(xr, a.x, px, HW, c0, n);
  if (a.h) rn_load_raw<TH, V, NC>(hr, a.h, px, HW, c0, n);
  if constexpr (FG) rn_load_raw<TH, V, NC>(g, a.gate, px, HW, c0, n);
  rn_factors<TH, NC, !FG>(k, a, px.b, c0, n);
  float x[NC][V];
  if (a.h) {
    float h[NC][V];
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) h[i][j] = rn_at<TH, V>(hr[i], j);
    if constexpr (POST) {
      float mu[V], rho[V];
      rn_block_moments<V, NC, FULL>(red, turn, nw, wave, lane, C, n, a.peps, h, mu, rho);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + min(i, n - 1);
        const float w = rn_const(a.pw, c), b = rn_const(a.pb, c);
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = fmaf((h[i][j] - mu[j]) * rho[j], w, b);
      }
      if (a.stats && wave == 0 && px.any()) {
        rn_store<float, V>(a.stats + 2 * a.total + px.q, 0, mu);
        rn_store<float, V>(a.stats + 3 * a.total + px.q, 0, rho);
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j)
        x[i][j] = fmaf(k[i], FG ? h[i][j] * rn_at<TH, V>(g[FG ? i : 0], j) : h[i][j], rn_at<T, V>(xr[i], j));
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = rn_at<T, V>(xr[i], j);
  }
  if (a.r && px.any())
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (i < n) rn_store<T, V>((T*)a.r + at + i * HW, px.off, x[i]);
  if (!a.nw) return;
  float mu[V], rho[V];
  rn_block_moments<V, NC, FULL>(red, turn, nw, wave, lane, C, n, a.neps, x, mu, rho);
  if (!px.any()) return;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    if (i >= n) break;
    const float w = rn_const(a.nw, c0 + i), b = rn_const(a.nb, c0 + i);
    float y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = fmaf((x[i][j] - mu[j]) * rho[j], w, b);
    rn_store<T, V>((T*)a.y + at + i * HW, px.off, y);
  }
  if (a.stats && wave == 0) {
    rn_store<float, V>(a.stats + px.q, 0, mu);
    rn_store<float, V>(a.stats + a.total + px.q, 0, rho);
  }
}

// Values that depend on v are computed in the loop they stand in: held for all channels over all tiles, parameters and
// offsets would not fit the scalar registers.
template <class P>
__device__ __forceinline__ void rn_in_loop(P& v) {
  asm volatile("" : "+s"(v));
}

__device__ __forceinline__ float rn_uniform(float v) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}

template <int V, int NC>
__device__ __forceinline__ void rn_drop(float (&v)[NC][V], int dup) {
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = j < dup ? 0.f : v[i][j];
}

template <class T, class TH, int V, int NC, bool FULL, bool POST, bool FG>
__global__ void __launch_bounds__(1024) k_rn_bwd(RnArgs a0) {
  extern __shared__ __attribute__((aligned(16))) float red[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int C = (int)a0.C, c0 = wave * NC, n = FULL ? NC : min(NC, C - c0);
  const float rC = 1.f / (float)C;
  const bool norm = a0.nw && a0.gy, branch = a0.dh || a0.dg || a0.s || POST, sample = !FG && a0.gate;
  const int mine = lane / (64 / NC);  // the channel whose sums this lane ends with
  int turn = 0;
  // The sums so far of channel c0 + mine, in 64 bits: float32 ones lose half a step a tile, and a block takes hundreds of a
  // large map.  In shared memory, where one lane alone adds to each, in the order of its tiles; in registers they spill
  // (8 x 64 x 256 x 256 bf16, gate per element: 137 us, against 121).
  const bool owns = lane % (64 / NC) == 0 && mine < n;
  double* const sums = (double*)(red + (nw == 1 ? 0 : kRnRed * V * nw)) + c0 + mine;
  auto add = [&](int q, float v) {
    if (owns) __hip_atomic_fetch_add(sums + q * C, (double)v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  if (owns)
    for (int q = 0; q < kRnSums; ++q) sums[q * C] = 0.;
  for (int64_t next = blockIdx.x; next < a0.ntiles; next += gridDim.x) {
    const int64_t tile = rn_order((uint32_t)next, (uint32_t)a0.ntiles);
    RnArgs a = a0;
    rn_in_loop(a.HW);
    rn_in_loop(a.s);
    rn_in_loop(a.nw);
    rn_in_loop(a.pw);
    rn_in_loop(a.pb);
    const int64_t HW = a.HW;
    const RnLane<V> px(a, tile, lane);
    const int64_t at = px.base + c0 * HW;
    float r[NC][V], d[NC][V], h[NC][V];
    typename RnVec<T, V>::v e[NC];  // gr and the gate as they were stored, until they are needed
    typename RnVec<TH, V>::v g[FG ? NC : 1];
    float mu[V], rho[V], mh[V], rh[V];
    if (norm) {
      rn_load_all<T, V, NC>(r, a.x, px, HW, c0, n);
      rn_load_all<T, V, NC>(d, a.gy, px, HW, c0, n);
      rn_load<float, V>(mu, a.stats + px.q, 0);
      rn_load<float, V>(rho, a.stats + a.total + px.q, 0);
    }
    if (a.gr) rn_load_raw<T, V, NC>(e, a.gr, px, HW, c0, n);
    if (a.h) rn_load_all<TH, V, NC>(h, a.h, px, HW, c0, n);
    if constexpr (FG && sizeof(T) < 4) rn_load_raw<TH, V, NC>(g, a.gate, px, HW, c0, n);
    if constexpr (POST) {
      rn_load<float, V>(mh, a.stats + 2 * a.total + px.q, 0);
      rn_load<float, V>(rh, a.stats + 3 * a.total + px.q, 0);
    }
    float k[NC];
    rn_factors<TH, NC, !FG>(k, a, px.b, c0, n);
    if (sample)
#pragma unroll
      for (int i = 0; i < NC; ++i) k[i] = rn_uniform(k[i]);
    if (!px.whole) {  // pixels of other lanes: gradients of 0, and finite values beside them
      if (norm) rn_drop<V, NC>(r, px.dup), rn_drop<V, NC>(d, px.dup);
      if (a.h) rn_drop<V, NC>(h, px.dup);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < px.dup) mu[j] = mh[j] = 0.f, rho[j] = rh[j] = 1.f;
    }
    if constexpr (POST) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][j] = (h[i][j] - mh[j]) * rh[j];  // hhat
    }
    auto gr = [&](int i, int j) { return j < px.dup ? 0.f : rn_at<T, V>(e[i], j); };
    auto gate = [&](int i, int j) { return j < px.dup ? 0.f : rn_at<TH, V>(g[FG ? i : 0], j); };
    // With float32 x and r a gate is loaded behind the norm's sums: held from the start it would not fit the registers of
    // 16 waves on a CU (4 x 128 x 16384, float32 and bfloat16: 57 us, 71 us spilt).
    auto load_gate = [&]() {
      if constexpr (FG && sizeof(T) == 4) rn_load_raw<TH, V, NC>(g, a.gate, px, HW, c0, n);
    };
    if (norm) {
      float s[2][V] = {}, t[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + min(i, n - 1);
        t[i] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (sizeof(T) < 4 && a.h) {  // x: r as the forward had it
            const float nv = POST ? fmaf(h[i][j], rn_const(a.pw, c), rn_const(a.pb, c)) : h[i][j];
            r[i][j] = fmaf(k[i], FG ? nv * gate(i, j) : nv, r[i][j]);
          }
          r[i][j] = (r[i][j] - mu[j]) * rho[j];  // rhat
          t[i] = fmaf(d[i][j], r[i][j], t[i]);
        }
      }
      add(0, rn_lane_sums<NC>(t, lane));
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const float w = i < n ? rn_const(a.nw, c0 + min(i, n - 1)) : 0.f;
        t[i] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          t[i] += d[i][j];
          d[i][j] *= w;
          s[0][j] += d[i][j];
          s[1][j] = fmaf(d[i][j], r[i][j], s[1][j]);
        }
      }
      add(1, rn_lane_sums<NC>(t, lane));
      load_gate();
      rn_block_sums<V>(red, turn, nw, wave, lane, s);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[0][j] *= rC;
        s[1][j] *= rC;
      }
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = fmaf(-r[i][j], s[1][j], d[i][j] - s[0][j]) * rho[j];
      if (a.gr) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) d[i][j] += gr(i, j);
      }
    } else {
      load_gate();
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = gr(i, j);
    }
    if (a.dx && px.any())
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (i < n) rn_store_own<T, V>((T*)a.dx + at + i * HW, d[i], px);
    if (!branch) continue;
    if (FG && a.dg && px.any()) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        if (i >= n) break;
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float nv = POST ? fmaf(h[i][j], rn_const(a.pw, c0 + i), rn_const(a.pb, c0 + i)) : h[i][j];
          o[j] = k[i] * d[i][j] * nv;
        }
        rn_store_own<TH, V>((TH*)a.dg + at + i * HW, o, px);
      }
    }
    if constexpr (FG) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] *= gate(i, j);
    }
    if (a.h) {
      const int c = c0 + min(mine, n - 1);
      const float gt = sample ? rn_ld<TH>(a.gate, px.b * C + c) : 1.f;
      float t[NC], va = 0.f;
      if constexpr (POST) {
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          t[i] = 0.f;
#pragma unroll
          for (int j = 0; j < V; ++j) t[i] += d[i][j];
        }
        va = rn_lane_sums<NC>(t, lane);
        add(2, gt * va);
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        t[i] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) t[i] = fmaf(d[i][j], h[i][j], t[i]);
      }
      const float vh = rn_lane_sums<NC>(t, lane);
      add(3, gt * vh);
      if (sample && a.dg && owns) {
        const float v = POST ? fmaf(a.pw[c], vh, a.pb[c] * va) : vh;
        a.dgpart[(px.b * C + c) * a.tps + tile % a.tps] = a.s ? a.s[c] * v : v;
      }
    }
    float s[2][V] = {};
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const float kp = i < n ? (POST ? k[i] * rn_const(a.pw, c0 + i) : k[i]) : 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[i][j] *= kp;  // dn wp
        if (POST) {
          s[0][j] += d[i][j];
          s[1][j] = fmaf(d[i][j], h[i][j], s[1][j]);
        }
      }
    }
    if constexpr (POST) {
      rn_block_sums<V>(red, turn, nw, wave, lane, s);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[0][j] *= rC;
        s[1][j] *= rC;
      }
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = fmaf(-h[i][j], s[1][j], d[i][j] - s[0][j]) * rh[j];
    }
    if (a.dh && px.any())
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (i < n) rn_store_own<TH, V>((TH*)a.dh + at + i * HW, d[i], px);
  }
  if (owns)
    for (int q = 0; q < kRnSums; ++q)
      ((float*)a0.part)[((int64_t)q * C + c0 + mine) * gridDim.x + blockIdx.x] = (float)sums[q * C];
}

// ------------------------------------------------------------------------------------------------
// More channels: a block of 16 waves per tile of 64 pixels, a pixel to a lane, each wave taking 16 channels of every 256
// in turn.  The channels are read again for each step of the formulas, from the caches (a tile of 512 float32 channels is
// 128 KB), and the sums over pixels are added to the block's row in memory, in 64 bits.
// ------------------------------------------------------------------------------------------------
constexpr int kWideWaves = 16, kWideCh = 16;

template <class T, class TH, bool POST>
struct RnWide {
  const RnArgs& a;
  const RnLane<1> px;
  const int wave, lane, C;
  float mh[1] = {0.f}, rh[1] = {1.f}, mu[1] = {0.f}, rho[1] = {1.f};  // of h and of r

  __device__ RnWide(const RnArgs& a_, int64_t tile, int wave_, int lane_)
      : a(a_), px(a_, tile, lane_), wave(wave_), lane(lane_), C((int)a_.C) {}

  // The channels of wave w below C.
  __device__ float count(int w) const {
    const int rest = C % (kWideWaves * kWideCh) - w * kWideCh;
    return (float)(C / (kWideWaves * kWideCh) * kWideCh + (rest < 0 ? 0 : min(rest, kWideCh)));
  }
  template <class F>
  __device__ void groups(F f) const {
    for (int c0 = wave * kWideCh; c0 < C; c0 += kWideWaves * kWideCh) f(c0, min(kWideCh, C - c0));
  }
  template <class P>
  __device__ void load(float (&o)[kWideCh], const void* p, int c0, int n) const {
    const P* t = (const P*)p + px.base + c0 * a.HW;
    if (a.HW == 1 && n == kWideCh) {  // a pixel's channels lie together: 256 rows of 1024, 436 -> 147 us a training pass
      constexpr int W = 16 / sizeof(P);
#pragma unroll
      for (int i = 0; i < kWideCh / W; ++i) {
        const typename RnVec<P, W>::v v = *(const typename RnVec<P, W>::v*)(t + W * i + px.off);
#pragma unroll
        for (int j = 0; j < W; ++j) o[W * i + j] = (float)v[j];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kWideCh; ++i) o[i] = (float)t[min(i, n - 1) * a.HW + px.off];
  }
  template <class P>
  __device__ void store(void* p, int c0, int n, const float (&v)[kWideCh]) const {
    if (px.dup) return;
    P* t = (P*)p + px.base + c0 * a.HW;
    if (a.HW == 1 && n == kWideCh) {
      constexpr int W = 16 / sizeof(P);
#pragma unroll
      for (int i = 0; i < kWideCh / W; ++i) {
        typename RnVec<P, W>::v o;
#pragma unroll
        for (int j = 0; j < W; ++j) o[j] = (P)v[W * i + j];
        *(typename RnVec<P, W>::v*)(t + W * i + px.off) = o;
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kWideCh; ++i)
      if (i < n) t[i * a.HW + px.off] = (P)v[i];
  }
  // h or hhat, and n of it
  __device__ void branch(float (&h)[kWideCh], int c0, int n) const {
    load<TH>(h, a.h, c0, n);
    if (POST)
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) h[i] = (h[i] - mh[0]) * rh[0];
  }
  __device__ float value(float h, int c) const { return POST ? fmaf(h, rn_const(a.pw, c), rn_const(a.pb, c)) : h; }
  // r from x; g: scratch
  __device__ void residual(float (&r)[kWideCh], int c0, int n) const {
    load<T>(r, a.x, c0, n);
    if (!a.h) return;
    float h[kWideCh], k[kWideCh], g[kWideCh];
    branch(h, c0, n);
    rn_factors<TH, kWideCh, true>(k, a, px.b, c0, n, !a.gate_full);
    if (a.gate && a.gate_full) {
      load<TH>(g, a.gate, c0, n);
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) k[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < kWideCh; ++i) r[i] = fmaf(k[i], value(h[i], c0 + min(i, n - 1)), r[i]);
  }
  // Mean and deviation over all channels of what f puts into its array.
  template <class F>
  __device__ void moments(float* red, int& turn, float eps, F f, float (&m)[1], float (&s)[1]) const {
    float cnt = 0.f, v[2][1] = {};
    groups([&](int c0, int n) {
      float x[kWideCh];
      f(x, c0, n);
      const float fn = (float)n;
      float u = 0.f, q = 0.f;
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) u += i < n ? x[i] : 0.f;
      u = rn_over(u, fn, 1.f / fn);
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) {
        const float d = i < n ? x[i] - u : 0.f;
        q = fmaf(d, d, q);
      }
      const float d = u - v[0][0], step = d * (fn / (cnt + fn));
      v[0][0] += step;
      v[1][0] += fmaf(step, d * cnt, q);  // (d * d may overflow for the first group, where d is its mean and cnt 0)
      cnt += fn;
    });
    const float fC = (float)C;
    rn_join<1>(red, turn, kWideWaves, wave, lane, fC, 1.f / fC, eps, [&](int w) { return count(w); }, v, m, s);
  }
};

template <class T, class TH, bool POST>
__global__ void __launch_bounds__(64 * kWideWaves) k_rn_fwd_wide(RnArgs a) {
  extern __shared__ __attribute__((aligned(16))) float red[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  RnWide<T, TH, POST> e(a, a.tile0 + blockIdx.x, wave, lane);
  int turn = 0;
  if constexpr (POST) {
    float mh[1], rh[1];
    e.moments(red, turn, a.peps, [&](float (&v)[kWideCh], int c0, int n) { e.template load<TH>(v, a.h, c0, n); }, mh, rh);
    e.mh[0] = mh[0];
    e.rh[0] = rh[0];
  }
  if (a.nw)
    e.moments(red, turn, a.neps, [&](float (&v)[kWideCh], int c0, int n) { e.residual(v, c0, n); }, e.mu, e.rho);
  e.groups([&](int c0, int n) {
    float r[kWideCh];
    e.residual(r, c0, n);
    if (a.r) e.template store<T>(a.r, c0, n, r);
    if (a.nw) {
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) {
        const int c = c0 + min(i, n - 1);
        r[i] = fmaf((r[i] - e.mu[0]) * e.rho[0], rn_const(a.nw, c), rn_const(a.nb, c));
      }
      e.template store<T>(a.y, c0, n, r);
    }
  });
  if (a.stats && wave == 0 && e.px.any()) {
    if (a.nw) {
      a.stats[e.px.q] = e.mu[0];
      a.stats[a.total + e.px.q] = e.rho[0];
    }
    if (POST) {
      a.stats[2 * a.total + e.px.q] = e.mh[0];
      a.stats[3 * a.total + e.px.q] = e.rh[0];
    }
  }
}

template <class T, class TH, bool POST>
__global__ void __launch_bounds__(64 * kWideWaves) k_rn_bwd_wide(RnArgs a) {
  extern __shared__ __attribute__((aligned(16))) float red[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), C = (int)a.C;
  const int mine = lane / (64 / kWideCh);
  const float rC = 1.f / (float)C;
  const bool norm = a.nw && a.gy, branch = a.dh || a.dg || a.s || POST, sample = a.gate && !a.gate_full;
  int turn = 0;
  for (int64_t tile = blockIdx.x; tile < a.ntiles; tile += gridDim.x) {
    RnWide<T, TH, POST> e(a, tile, wave, lane);
    const bool own = !e.px.dup;
    if (norm) {
      e.mu[0] = a.stats[e.px.q];
      e.rho[0] = a.stats[a.total + e.px.q];
    }
    if (POST) {
      e.mh[0] = a.stats[2 * a.total + e.px.q];
      e.rh[0] = a.stats[3 * a.total + e.px.q];
    }
    // Adds a channel's sum over the tile, which the wave's lane `mine` of it holds, to the block's row.
    auto add = [&](int k, int c0, int n, double v) {
      if (lane % (64 / kWideCh) || mine >= n) return;
      double* o = (double*)a.part + ((int64_t)k * C + c0 + mine) * gridDim.x + blockIdx.x;
      *o = tile == blockIdx.x ? v : *o + v;
    };
    // rhat and gy; a lane without a pixel of its own: zeros
    auto load = [&](float (&r)[kWideCh], float (&g)[kWideCh], int c0, int n) {
      if (sizeof(T) == 4) e.template load<T>(r, a.x, c0, n);  // r itself
      else e.residual(r, c0, n);
      e.template load<T>(g, a.gy, c0, n);
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) {
        r[i] = own ? (r[i] - e.mu[0]) * e.rho[0] : 0.f;
        g[i] = own ? g[i] : 0.f;
      }
    };
    float s[2][1] = {};
    if (norm) {
      e.groups([&](int c0, int n) {
        float r[kWideCh], g[kWideCh], t[kWideCh];
        load(r, g, c0, n);
#pragma unroll
        for (int i = 0; i < kWideCh; ++i) {
          t[i] = g[i] * r[i];
          const float w = i < n ? rn_const(a.nw, c0 + min(i, n - 1)) : 0.f;
          s[0][0] = fmaf(g[i], w, s[0][0]);
          s[1][0] = fmaf(t[i], w, s[1][0]);
        }
        add(0, c0, n, rn_lane_sums<kWideCh>(t, lane));
        add(1, c0, n, rn_lane_sums<kWideCh>(g, lane));
      });
      rn_block_sums<1>(red, turn, kWideWaves, wave, lane, s);
    }
    const float s1 = s[0][0] * rC, s2 = s[1][0] * rC;
    // dr, times a gate per element
    auto grad = [&](float (&d)[kWideCh], int c0, int n) {
      float r[kWideCh];
      if (norm) {
        load(r, d, c0, n);
#pragma unroll
        for (int i = 0; i < kWideCh; ++i)
          d[i] = fmaf(-r[i], s2, fmaf(d[i], rn_const(a.nw, c0 + min(i, n - 1)), -s1)) * e.rho[0];
      } else {
#pragma unroll
        for (int i = 0; i < kWideCh; ++i) d[i] = 0.f;
      }
      if (a.gr) {
        e.template load<T>(r, a.gr, c0, n);
#pragma unroll
        for (int i = 0; i < kWideCh; ++i) d[i] += r[i];
      }
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) d[i] = own ? d[i] : 0.f;
    };
    auto hidden = [&](float (&h)[kWideCh], int c0, int n) {
      e.branch(h, c0, n);
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) h[i] = own ? h[i] : 0.f;
    };
    auto gated = [&](float (&d)[kWideCh], int c0, int n) {
      if (!a.gate || !a.gate_full) return;
      float g[kWideCh];
      e.template load<TH>(g, a.gate, c0, n);
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) d[i] *= own ? g[i] : 0.f;
    };
    float z[2][1] = {};
    e.groups([&](int c0, int n) {
      float d[kWideCh], h[kWideCh], k[kWideCh], t[kWideCh];
      grad(d, c0, n);
      if (a.dx) e.template store<T>(a.dx, c0, n, d);
      if (!branch) return;
      if (!a.h) {  // no scale, gate and norm: dh is dr in its own type
        e.template store<TH>(a.dh, c0, n, d);
        return;
      }
      hidden(h, c0, n);
      rn_factors<TH, kWideCh, true>(k, a, e.px.b, c0, n, sample);
      if (a.dg && !sample) {
#pragma unroll
        for (int i = 0; i < kWideCh; ++i) t[i] = k[i] * d[i] * e.value(h[i], c0 + min(i, n - 1));
        e.template store<TH>(a.dg, c0, n, t);
      }
      gated(d, c0, n);
      const int c = c0 + min(mine, n - 1);
      const float gt = sample ? rn_ld<TH>(a.gate, e.px.b * C + c) : 1.f;
      float va = 0.f;
      if (POST) {
#pragma unroll
        for (int i = 0; i < kWideCh; ++i) t[i] = d[i];
        va = rn_lane_sums<kWideCh>(t, lane);
        add(2, c0, n, (double)gt * va);
      }
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) t[i] = d[i] * h[i];
      const float vh = rn_lane_sums<kWideCh>(t, lane);
      add(3, c0, n, (double)gt * vh);
      if (a.dg && sample && lane % (64 / kWideCh) == 0 && mine < n) {
        const float v = POST ? fmaf(a.pw[c], vh, a.pb[c] * va) : vh;
        a.dgpart[(e.px.b * C + c) * a.tps + tile % a.tps] = a.s ? a.s[c] * v : v;
      }
      if (POST) {
#pragma unroll
        for (int i = 0; i < kWideCh; ++i) {
          const float v = i < n ? d[i] * (k[i] * rn_const(a.pw, c0 + min(i, n - 1))) : 0.f;
          z[0][0] += v;
          z[1][0] = fmaf(v, h[i], z[1][0]);
        }
      } else if (a.dh) {
#pragma unroll
        for (int i = 0; i < kWideCh; ++i) d[i] *= k[i];
        e.template store<TH>(a.dh, c0, n, d);
      }
    });
    if (!POST) continue;
    rn_block_sums<1>(red, turn, kWideWaves, wave, lane, z);
    if (!a.dh) continue;
    const float s3 = z[0][0] * rC, s4 = z[1][0] * rC;
    e.groups([&](int c0, int n) {
      float d[kWideCh], h[kWideCh], k[kWideCh];
      grad(d, c0, n);
      gated(d, c0, n);
      hidden(h, c0, n);
      rn_factors<TH, kWideCh, true>(k, a, e.px.b, c0, n, sample);
#pragma unroll
      for (int i = 0; i < kWideCh; ++i) {
        const float v = d[i] * (k[i] * rn_const(a.pw, c0 + min(i, n - 1)));
        d[i] = fmaf(-h[i], s4, v - s3) * e.rh[0];
      }
      e.template store<TH>(a.dh, c0, n, d);
    });
  }
}

// The blocks of a backward, or a forward's tiles in as many launches as they take.
template <bool BWD>
int rn_launch(void (*k)(RnArgs), RnArgs a, int64_t blocks, int threads, size_t lds, hipStream_t st) {
  const int64_t most = rn_max_blocks(threads);
  for (a.tile0 = 0; a.tile0 < blocks; a.tile0 += most)
    hipLaunchKernelGGL(k, dim3((unsigned)std::min(most, blocks - a.tile0)), dim3(threads), lds, st, a);
  return check_launch(BWD ? "residual_norm backward" : "residual_norm");
}

template <bool BWD, class T, class TH>
int rn_launch_wide(const RnArgs& a, int64_t blocks, hipStream_t st) {
  void (*k)(RnArgs);
  if constexpr (BWD) k = a.pw ? k_rn_bwd_wide<T, TH, true> : k_rn_bwd_wide<T, TH, false>;
  else k = a.pw ? k_rn_fwd_wide<T, TH, true> : k_rn_fwd_wide<T, TH, false>;
  return rn_launch<BWD>(k, a, blocks, 64 * kWideWaves, sizeof(float) * kRnRed * kWideWaves, st);
}

template <bool BWD, class T, class TH, int V, int NC, bool FULL>
int rn_launch_tile(const RnArgs& a, int64_t blocks, hipStream_t st) {
  const int nw = (int)((a.C + NC - 1) / NC);
  const size_t lds = (nw == 1 ? 0 : sizeof(float) * kRnRed * V * nw) + (BWD ? sizeof(double) * kRnSums * a.C : 0);
  const bool fg = a.gate && a.gate_full;
  void (*k)(RnArgs);
  if constexpr (BWD)
    k = a.pw ? (fg ? k_rn_bwd<T, TH, V, NC, FULL, true, true> : k_rn_bwd<T, TH, V, NC, FULL, true, false>)
             : (fg ? k_rn_bwd<T, TH, V, NC, FULL, false, true> : k_rn_bwd<T, TH, V, NC, FULL, false, false>);
  else
    k = a.pw ? (fg ? k_rn_fwd<T, TH, V, NC, FULL, true, true> : k_rn_fwd<T, TH, V, NC, FULL, true, false>)
             : (fg ? k_rn_fwd<T, TH, V, NC, FULL, false, true> : k_rn_fwd<T, TH, V, NC, FULL, false, false>);
  if (BWD && lds > 64 * 1024)  // 121 to 128 channels
    (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  return rn_launch<BWD>(k, a, blocks, 64 * nw, lds, st);
}

template <class T, class TH>
int rn_launch_fwd(const RnArgs& a, const RnShape& s, hipStream_t st) {
  if (s.px == 0) return rn_launch_wide<false, T, TH>(a, s.ntiles, st);
  if (s.px == 2)
    return s.ch == 8 ? rn_launch_tile<false, T, TH, 2, 8, true>(a, s.ntiles, st)
                     : rn_launch_tile<false, T, TH, 2, 16, true>(a, s.ntiles, st);
  return rn_launch_tile<false, T, TH, 1, 16, false>(a, s.ntiles, st);
}

template <class T, class TH>
int rn_launch_bwd(const RnArgs& a, const RnShape& s, hipStream_t st) {
  const int64_t blocks = rn_bwd_blocks(s);
  if (s.px == 0) return rn_launch_wide<true, T, TH>(a, blocks, st);
  if (s.px == 2) return rn_launch_tile<true, T, TH, 2, 8, true>(a, blocks, st);
  if (s.ch == 8) return rn_launch_tile<true, T, TH, 1, 8, false>(a, blocks, st);
  return a.C % 16 ? rn_launch_tile<true, T, TH, 1, 16, false>(a, blocks, st)
                  : rn_launch_tile<true, T, TH, 1, 16, true>(a, blocks, st);
}

}  // namespace
}  // namespace cvn
