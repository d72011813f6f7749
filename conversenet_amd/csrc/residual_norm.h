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
  // where a sample's last tile is a small part of it, and only then may a lane take several pixels.  2^18 pixels of 64
  // channels, float32 with a scale, then bfloat16 with a gate per sample and both norms, two pixels a lane against one:
  // 1025 pixels a sample forward 59 against 62 us and 38 against 42, backward 91 against 98 and 65 against 99; 2304 pixels
  // 51, 50; 32, 38; 84, 91; 56, 94.  At 400 pixels 56, 53; 38, 41; 93, 93; 71, 108, and at 128 channels (float32 and
  // bfloat16, gate per element, both norms) 114, 110 and 211, 205: there half of the last tile is empty.
  const bool per_sample = (bwd && gate_sample) || HW >= 1024, pairs = HW >= 1024;
  // Few channels to a wave keep the backward's values in registers, more spare the forward waves to join.  Forward with 8
  // channels and with 16: at 128 channels 30 and 28 us (4 x 16384 pixels, float32 and bfloat16, gate per element, both
  // norms), 64 and 56 (2 x 65536), in bfloat16 21 and 15; at 96 (4 x 40000, float32) 50 and 53, in bfloat16 37 and 32; at 64
  // (8 x 65536, float32) 105 and 107, (1 x 154401) 37.5 and 37.5, in bfloat16 with both norms 59 and 55; at 32 (float32) 53
  // and 54.  Backward with 8 54-61 us at 4 x 128 x 16384, 147 with 16, which spill.
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

// Blocks of the backward, which each keep a row of partial sums: what the 256 CUs hold at once (16 waves of its kernels with
// 128 registers, 20 of those with 8 channels of one pixel).  With half of them, these and twice as many: 8 x 64 x 96 x 96
// 36.5, 35 and 36 us, 1 x 64 x 321 x 481 64, 59 and 66, 8 x 64 x 256 x 256 176, 172 and 171 (in bfloat16 with a gate per
// sample and both norms 126, 102 and 107), 4 x 128 x 128 x 128 61, 54.5 and 54, 4 x 200 x 100 x 100 74, 59 and 61;
// 2 x 512 x 64 x 64 46 each time; 8 x 16 x 256 x 256 50, 54 and 64.
inline int64_t rn_bwd_blocks(const RnShape& s) {
  const int resident = s.px == 1 && s.ch == 8 ? 20 : 16;
  return std::min<int64_t>(s.ntiles, 256 * (resident / s.waves));
}

}  // namespace cvn
