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
#include "cvn_common.h"

namespace cvn {

constexpr int kRnSums = 5;  // dw, db, ds, dwp, dbp

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
  float *part, *dgpart;  // [kRnSums][C][blocks]; [B C][tps]
  int64_t C, HW, total;  // total = B HW
  int64_t ntiles;
  int tps;          // tiles per sample, or 0: tiles of consecutive pixels of any samples
  bool gate_full;   // a gate per element; otherwise per sample and channel
};

// The launches of one pair of types (residual_norm_f32.hip, residual_norm_half.hip).
typedef int (*RnLaunch)(const RnArgs&, int64_t B, hipStream_t);
struct RnKernels {
  RnLaunch fwd, bwd;
};
RnKernels rn_f32_f32();
RnKernels rn_f32_bf16();
RnKernels rn_f32_f16();
RnKernels rn_bf16_bf16();
RnKernels rn_f16_f16();

// Blocks of the backward, which each keep a row of partial sums.
int64_t rn_bwd_blocks(int64_t ntiles);

struct RnTiles {
  int64_t n;
  int tps;
};
// Tiles of 64 pixels.  A gate per sample and channel has its gradient summed tile by tile, so its tiles end with their
// sample; others do where a sample's last tile is a small part of it.
inline RnTiles rn_tiles(int64_t B, int64_t HW, bool gate_sample) {
  if (gate_sample || HW >= 1024) {
    const int64_t tps = (HW + 63) / 64;
    return {B * tps, (int)tps};
  }
  return {(B * HW + 63) / 64, 0};
}

}  // namespace cvn
