// Scaled residual and channels-first LayerNorm of a block, forward and backward: the arguments the translation units
// of residual_norm.hip and residual_norm_*.hip share, and the kernels.
//
//   n = P(h)  (LayerNorm over channels, or h itself)      u = gate n      (or n)
//   r = x + s_c u                                         y = N(r) = rhat w_c + b_c,  rhat = (r - mu) rho
//
// and from the gradients gr, gy of r and y, with <v> the mean over the channels of a pixel:
//   dr = gr + rho (gy w - <gy w> - rhat <gy w rhat>)      dx = dr
//   dgate = s dr n     dn = s gate dr                     dh = rho_h (dn wp - <dn wp> - hhat <dn wp hhat>)   (or dn)
//   ds = sum dr u      dw = sum gy rhat    db = sum gy    dwp = sum dn hhat    dbp = sum dn      (sums over pixels)
#pragma once
#include <algorithm>

#include "cvn_common.h"

namespace cvn {

// The sums over pixels a backward keeps of each channel, hh = hhat or h, g = gate or 1 (s and wp, bp factor out):
// gy rhat, gy, g dr, g dr hh.  Then dw, db are the first two, ds = wp S3 + bp S2 (or S3), dwp = s S3, dbp = s S2.
constexpr int kRnSums = 4;

struct RnArgs {
  // forward; in the backward x is the forward's r for a float32 stream, and x itself for a 16-bit one
  const void *x, *h, *gate;
  const float *s, *nw, *nb, *pw, *pb;
  float neps, peps;
  void *r, *y;
  float* stats;  // [2 or 4][total]: mu and rho of r, then of h
  // backward
  const void *gr, *gy;
  void *dx, *dh, *dg;
  void* part;     // [kRnSums][C][blocks], double for many channels, float otherwise
  float* dgpart;  // [B C][tps]
  int64_t C, HW, total;  // total = B HW
  int64_t ntiles;
  int64_t tile0;    // the first tile of a forward's launch
  int tps;          // tiles per sample, or 0: tiles of consecutive pixels of any samples
  bool gate_full;   // a gate per element; otherwise per sample and channel
};

// The launches of one pair of types (residual_norm_f32.hip, residual_norm_half.hip).
struct RnShape;
typedef int (*RnLaunch)(const RnArgs&, const RnShape&, hipStream_t);
struct RnKernels {
  RnLaunch fwd, bwd;
};
RnKernels rn_f32_f32();
RnKernels rn_f32_bf16();
RnKernels rn_f32_f16();
RnKernels rn_bf16_bf16();
RnKernels rn_f16_f16();

// A launch holds fewer than 2^32 threads: its blocks at most, in whole runs of 64 (rn_order).
inline int64_t rn_max_blocks(int threads) { return (((int64_t)1 << 32) - 1) / threads / 64 * 64; }

// How a call runs: pixels of a lane (0: the kernels for many channels), channels of a wave, and its tiles of 64 px pixels
// (64 there).
struct RnShape {
  int px, ch, waves;
  int64_t ntiles;
  int tps;  // tiles per sample, or 0: tiles of consecutive pixels of any samples
};

inline RnShape rn_shape(bool bwd, int64_t B, int64_t C, int64_t HW, bool gate_sample) {
  RnShape s = {};
  // A gate per sample and channel has its gradient summed tile by tile, so its tiles end with their sample; others do
  // where a sample's last tile is a small part of it, and only then may a lane take several pixels.
  const bool per_sample = (bwd && gate_sample) || HW >= 1024, pairs = HW >= 1024;
  // Few channels to a wave keep the backward's values in registers, more spare the forward waves to join.  Measured at
  // 4 x 128 x 128 x 128 (float32 and bfloat16, gate and both norms): forward 25-28 us with 16 channels, 35-38 us with 8;
  // backward 54-61 with 8, 147 with 16, which spill.
  if (C > 256) s.px = 0, s.ch = 16;
  else if (pairs && C <= (bwd ? 128 : 64) && C % 8 == 0) s.px = 2, s.ch = 8;
  else if (pairs && !bwd && C % 16 == 0) s.px = 2, s.ch = 16;
  else s.px = 1, s.ch = bwd && C <= 128 ? 8 : 16;
  s.waves = s.px ? (int)((C + s.ch - 1) / s.ch) : 16;
  const int64_t tile = 64 * (s.px ? s.px : 1);
  if (per_sample) {
    s.tps = (int)((HW + tile - 1) / tile);
    s.ntiles = B * s.tps;
  } else {
    s.ntiles = (B * HW + tile - 1) / tile;
  }
  return s;
}

// Blocks of the backward, which each keep a row of partial sums: what the CUs hold at once (16 waves of its kernels with
// 128 registers, 20 of those with 8 channels of one pixel).  8 x 64 x 96 x 96 takes 35 us; 39 with the tiles spread evenly
// over fewer blocks, 36 with twice as many.
inline int64_t rn_bwd_blocks(const RnShape& s) {
  const int resident = s.px == 1 && s.ch == 8 ? 20 : 16;
  return std::min<int64_t>(s.ntiles, 256 * (resident / s.waves));
}

}  // namespace cvn
