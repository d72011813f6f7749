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

// The sum of v over a wave's lanes, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// Any channel count: a wave per tile of 64 pixels, a pixel per lane, the channels read again for each step of the
// formulas (from the caches: a tile's channels are 64 C elements).
template <class T, class TH, bool POST>
struct RnPixel {
  const RnArgs& a;
  const RnPx p;
  float mh = 0.f, rh = 0.f;  // mu and rho of h
  __device__ RnPixel(const RnArgs& a_, const RnPx& p_) : a(a_), p(p_) {}
  __device__ int64_t at(int64_t c) const { return p.base + c * a.HW + p.off; }
  __device__ float gate(int64_t c) const {
    if (!a.gate) return 1.f;
    return rn_ld<TH>(a.gate, a.gate_full ? at(c) : p.b * a.C + c);
  }
  __device__ float hhat(int64_t c) const { return (rn_ld<TH>(a.h, at(c)) - mh) * rh; }
  __device__ float n(int64_t c) const { return POST ? fmaf(hhat(c), a.pw[c], a.pb[c]) : rn_ld<TH>(a.h, at(c)); }
  __device__ float r(int64_t c) const {
    const float x = rn_ld<T>(a.x, at(c));
    if (!a.h) return x;
    const float u = n(c) * gate(c);
    return a.s ? fmaf(a.s[c], u, x) : x + u;
  }
};

template <class F>
__device__ __forceinline__ void rn_moments(int64_t C, float eps, float& mu, float& rho, F v) {
  float s = 0.f;
  for (int64_t c = 0; c < C; ++c) s += v(c);
  mu = s / (float)C;
  float q = 0.f;
  for (int64_t c = 0; c < C; ++c) {
    const float d = v(c) - mu;
    q = fmaf(d, d, q);
  }
  rho = 1.f / sqrtf(q / (float)C + eps);
}

template <class T, class TH, bool POST>
__global__ void __launch_bounds__(64) k_rn_fwd_any(RnArgs a) {
  const RnPx px = rn_px(a, blockIdx.x, threadIdx.x);
  RnPixel<T, TH, POST> e(a, px);
  if (POST) rn_moments(a.C, a.peps, e.mh, e.rh, [&](int64_t c) { return rn_ld<TH>(a.h, e.at(c)); });
  float mu = 0.f, rho = 0.f;
  if (a.nw) rn_moments(a.C, a.neps, mu, rho, [&](int64_t c) { return e.r(c); });
  if (!px.ok) return;
  for (int64_t c = 0; c < a.C; ++c) {
    const float r = e.r(c);
    if (a.r) ((T*)a.r)[e.at(c)] = (T)r;
    if (a.nw) ((T*)a.y)[e.at(c)] = (T)fmaf((r - mu) * rho, a.nw[c], a.nb[c]);
  }
  if (a.stats) {
    if (a.nw) {
      a.stats[px.q] = mu;
      a.stats[a.total + px.q] = rho;
    }
    if (POST) {
      a.stats[2 * a.total + px.q] = e.mh;
      a.stats[3 * a.total + px.q] = e.rh;
    }
  }
}

template <class T, class TH, bool POST>
__global__ void __launch_bounds__(64) k_rn_bwd_any(RnArgs a) {
  const int lane = threadIdx.x;
  const int64_t G = gridDim.x;
  const bool branch = a.dh || a.dg || a.s || POST;
  for (int64_t tile = blockIdx.x; tile < a.ntiles; tile += G) {
    const bool first = tile == blockIdx.x;
    const RnPx px = rn_px(a, tile, lane);
    RnArgs b = a;
    if (sizeof(T) == 4) b.h = nullptr;  // x holds r
    RnPixel<T, TH, POST> e(a, px), f(b, px);
    if (POST) {
      e.mh = f.mh = a.stats[2 * a.total + px.q];
      e.rh = f.rh = a.stats[3 * a.total + px.q];
    }
    float mu = 0.f, rho = 0.f, s1 = 0.f, s2 = 0.f;
    const bool norm = a.nw && a.gy;
    if (norm) {
      mu = a.stats[px.q];
      rho = a.stats[a.total + px.q];
      for (int64_t c = 0; c < a.C; ++c) {
        const float g = rn_ld<T>(a.gy, e.at(c)) * a.nw[c];
        s1 += g;
        s2 = fmaf(g, (f.r(c) - mu) * rho, s2);
      }
      s1 /= (float)a.C;
      s2 /= (float)a.C;
    }
    auto add = [&](int k, int64_t c, float v) {  // a lane's part of a channel's sum
      v = wave_sum(px.ok ? v : 0.f);
      float* o = a.part + ((int64_t)k * a.C + c) * G + blockIdx.x;
      if (lane == 0) *o = first ? v : *o + v;
    };
    auto dr = [&](int64_t c, float gy, float rhat) {
      float d = a.gr ? rn_ld<T>(a.gr, e.at(c)) : 0.f;
      if (norm) d += rho * (gy * a.nw[c] - s1 - rhat * s2);
      return d;
    };
    float s3 = 0.f, s4 = 0.f;
    for (int64_t c = 0; c < a.C; ++c) {
      const float gy = norm ? rn_ld<T>(a.gy, e.at(c)) : 0.f, rhat = norm ? (f.r(c) - mu) * rho : 0.f;
      const float d = dr(c, gy, rhat);
      if (norm) {
        add(0, c, gy * rhat);
        add(1, c, gy);
      }
      if (a.dx && px.ok) ((T*)a.dx)[e.at(c)] = (T)d;
      if (!branch) continue;
      const float gt = e.gate(c), du = a.s ? a.s[c] * d : d, dn = du * gt;
      if (a.s || a.dg) {
        const float n = e.n(c);
        if (a.s) add(2, c, d * (n * gt));
        if (a.dg) {
          if (a.gate_full) {
            if (px.ok) ((TH*)a.dg)[e.at(c)] = (TH)(du * n);
          } else {
            const float v = wave_sum(px.ok ? du * n : 0.f);
            if (lane == 0) a.dgpart[(px.b * a.C + c) * a.tps + tile % a.tps] = v;
          }
        }
      }
      if (POST) {
        const float hh = e.hhat(c), g = dn * a.pw[c];
        add(3, c, dn * hh);
        add(4, c, dn);
        s3 += g;
        s4 = fmaf(g, hh, s4);
      } else if (a.dh && px.ok) {
        ((TH*)a.dh)[e.at(c)] = (TH)dn;
      }
    }
    if (!POST || !a.dh) continue;
    s3 /= (float)a.C;
    s4 /= (float)a.C;
    for (int64_t c = 0; c < a.C; ++c) {
      const float gy = norm ? rn_ld<T>(a.gy, e.at(c)) : 0.f, rhat = norm ? (f.r(c) - mu) * rho : 0.f;
      const float d = dr(c, gy, rhat), dn = (a.s ? a.s[c] * d : d) * e.gate(c);
      if (px.ok) ((TH*)a.dh)[e.at(c)] = (TH)(e.rh * (dn * a.pw[c] - s3 - e.hhat(c) * s4));
    }
  }
}

template <class T, class TH>
int rn_launch_fwd(const RnArgs& a, int64_t, hipStream_t st) {
  auto k = a.pw ? k_rn_fwd_any<T, TH, true> : k_rn_fwd_any<T, TH, false>;
  hipLaunchKernelGGL(k, dim3((unsigned)a.ntiles), dim3(64), 0, st, a);
  return check_launch("residual_norm");
}

template <class T, class TH>
int rn_launch_bwd(const RnArgs& a, int64_t, hipStream_t st) {
  auto k = a.pw ? k_rn_bwd_any<T, TH, true> : k_rn_bwd_any<T, TH, false>;
  hipLaunchKernelGGL(k, dim3((unsigned)rn_bwd_blocks(a.ntiles)), dim3(64), 0, st, a);
  return check_launch("residual_norm backward");
}

}  // namespace
}  // namespace cvn
