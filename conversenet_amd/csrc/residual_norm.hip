// C entry points of residual_norm.h, and the last step of its sums over pixels.
#include <algorithm>

#include "residual_norm.h"

namespace cvn {

namespace {

// The parameters' gradients from the blocks' sums, and the per-sample gates' from their tiles': a wave per channel or
// gate, in 64 bits, in the same order on every call.
struct RnSumArgs {
  const void* part;
  const float* dgpart;
  const float *s, *pw, *pb;
  float *dw, *db, *ds, *dpw, *dpb;
  void* dg;  // (B C) of type dg_type, or null
  int dg_type;
  int C, G, tps;
  int64_t rows;  // C, and B C for the gates
};

template <class T>
__device__ __forceinline__ double rn_row_sum(const T* p, int n, int lane) {
  double s[4] = {0., 0., 0., 0.};
  int i = lane;
  for (; i + 192 < n; i += 256) {
    T v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = p[i + 64 * j];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += v[j];
  }
  for (; i < n; i += 64) s[0] += p[i];
  double t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) t += __shfl_xor(t, d);
  return t;
}

template <class T>
__global__ void __launch_bounds__(256) k_rn_sums(RnSumArgs a) {
  const int lane = threadIdx.x & 63;
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < a.rows; row += (int64_t)gridDim.x * 4) {
    if (row >= a.C) {
      const int64_t i = row - a.C;
      const float s = (float)rn_row_sum(a.dgpart + i * a.tps, a.tps, lane);
      if (lane) continue;
      if (a.dg_type == CVN_F32) ((float*)a.dg)[i] = s;
      else if (a.dg_type == CVN_BF16) ((__bf16*)a.dg)[i] = (__bf16)s;
      else ((_Float16*)a.dg)[i] = (_Float16)s;
      continue;
    }
    const int c = (int)row;
    auto sum = [&](int k) { return rn_row_sum((const T*)a.part + ((int64_t)k * a.C + c) * a.G, a.G, lane); };
    const double w = a.dw ? sum(0) : 0., b = a.db ? sum(1) : 0.;
    const double sa = a.dpb || (a.ds && a.pw) ? sum(2) : 0., sh = a.ds || a.dpw ? sum(3) : 0.;
    if (lane) continue;
    const double s = a.s ? a.s[c] : 1.;
    if (a.dw) a.dw[c] = (float)w;
    if (a.db) a.db[c] = (float)b;
    if (a.ds) a.ds[c] = (float)(a.pw ? a.pw[c] * sh + a.pb[c] * sa : sh);
    if (a.dpw) a.dpw[c] = (float)(s * sh);
    if (a.dpb) a.dpb[c] = (float)(s * sa);
  }
}

size_t rn_part_bytes(int64_t C, const RnShape& t) {
  return align_up((t.px ? sizeof(float) : sizeof(double)) * kRnSums * (size_t)C * (size_t)rn_bwd_blocks(t));
}

bool rn_kernels(int x_type, int h_type, RnKernels* k) {
  if (x_type == CVN_F32 && h_type == CVN_F32) *k = rn_f32_f32();
  else if (x_type == CVN_F32 && h_type == CVN_BF16) *k = rn_f32_bf16();
  else if (x_type == CVN_F32 && h_type == CVN_F16) *k = rn_f32_f16();
  else if (x_type == CVN_BF16 && h_type == CVN_BF16) *k = rn_bf16_bf16();
  else if (x_type == CVN_F16 && h_type == CVN_F16) *k = rn_f16_f16();
  else return false;
  return true;
}

int rn_shape_ok(int64_t B, int64_t C, int64_t HW, int x_type, int h_type, RnKernels* k) {
  if (B < 0 || C < 1 || HW < 0) return fail(CVN_ERR_ARG, "bad shape");
  if (!rn_kernels(x_type, h_type, k))
    return fail(CVN_ERR_ARG, "types %d and %d: x and h of one type, or a 16-bit h on a float32 x", x_type, h_type);
  // pixel and tile numbers are held in 32 bits, a tile's last pixel behind the last one too; offsets of elements in 64
  constexpr int64_t kPixels = INT32_MAX - 255;
  if (C > 65536 || B > kPixels || HW > kPixels || B * HW > kPixels)
    return fail(CVN_ERR_UNSUPPORTED, "more than 65536 channels or 2^31 - 256 pixels");
  return CVN_OK;
}

int rn_branch_ok(const void* h, const float* s, const void* gate, int gate_kind, const float* pw, const float* pb) {
  if (gate_kind != CVN_GATE_NONE && gate_kind != CVN_GATE_SAMPLE && gate_kind != CVN_GATE_FULL)
    return fail(CVN_ERR_ARG, "bad gate kind");
  if ((gate != nullptr) != (gate_kind != CVN_GATE_NONE)) return fail(CVN_ERR_ARG, "gate and its kind do not match");
  if ((pw != nullptr) != (pb != nullptr)) return fail(CVN_ERR_ARG, "the branch norm needs weight and bias");
  if (!h && (s || gate || pw)) return fail(CVN_ERR_ARG, "scale, gate or branch norm without a branch");
  return CVN_OK;
}

}  // namespace
}  // namespace cvn

using namespace cvn;

extern "C" int cvn_residual_norm_fwd(const void* x, int x_type, const void* h, int h_type, int64_t B, int64_t C,
                                     int64_t HW, const float* res_scale, const void* gate, int gate_kind,
                                     const float* post_w, const float* post_b, float post_eps, const float* norm_w,
                                     const float* norm_b, float norm_eps, void* r, void* y, float* stats,
                                     cvn_stream_t stream) {
  RnKernels k;
  int rc = rn_shape_ok(B, C, HW, x_type, h ? h_type : x_type, &k);
  if (rc == CVN_OK && B * HW == 0) return CVN_OK;  // empty tensors have no addresses to check
  if (rc == CVN_OK) rc = rn_branch_ok(h, res_scale, gate, gate_kind, post_w, post_b);
  if (rc != CVN_OK) return rc;
  if (!x || (h && !r) || (norm_w && (!norm_b || !y)) || (!h && !norm_w)) return fail(CVN_ERR_ARG, "null pointer");
  RnArgs a = {};
  a.x = x;
  a.h = h;
  a.gate = gate;
  a.gate_full = gate_kind == CVN_GATE_FULL;
  a.s = res_scale;
  a.nw = norm_w;
  a.nb = norm_b;
  a.pw = post_w;
  a.pb = post_b;
  a.neps = norm_eps;
  a.peps = post_eps;
  a.r = r;
  a.y = y;
  a.stats = stats;
  a.C = C;
  a.HW = HW;
  a.total = B * HW;
  const RnShape t = rn_shape(false, B, C, HW, false);
  a.ntiles = t.ntiles;
  a.tps = t.tps;
  return k.fwd(a, t, (hipStream_t)stream);
}

extern "C" size_t cvn_residual_norm_bwd_workspace(int64_t B, int64_t C, int64_t HW, int gate_kind) {
  RnKernels k;
  if (rn_shape_ok(B, C, HW, CVN_F32, CVN_F32, &k) != CVN_OK) return 0;
  const bool sample = gate_kind == CVN_GATE_SAMPLE;
  const RnShape t = rn_shape(true, B, C, HW, sample);
  const size_t part = rn_part_bytes(C, t);
  return part + (sample ? sizeof(float) * (size_t)(B * C) * (size_t)t.tps : 0) + 256;
}

extern "C" int cvn_residual_norm_bwd(const void* grad_r, const void* grad_y, const void* base, int x_type, const void* h,
                                     int h_type, int64_t B, int64_t C, int64_t HW, const float* res_scale,
                                     const void* gate, int gate_kind, const float* post_w, const float* post_b,
                                     const float* norm_w, const float* stats, void* grad_x, void* grad_h, void* grad_gate,
                                     float* grad_scale, float* grad_norm_w, float* grad_norm_b, float* grad_post_w,
                                     float* grad_post_b, void* workspace, size_t workspace_bytes, cvn_stream_t stream) {
  RnKernels k;
  int rc = rn_shape_ok(B, C, HW, x_type, h || grad_h ? h_type : x_type, &k);
  const bool empty = B == 0 || HW == 0;
  if (rc == CVN_OK && !empty) rc = rn_branch_ok(h, res_scale, gate, gate_kind, post_w, post_b);
  if (rc != CVN_OK) return rc;
  if ((grad_gate && !gate) || (grad_scale && !res_scale) || ((grad_norm_w || grad_norm_b) && !norm_w) ||
      ((grad_post_w || grad_post_b) && !post_w))
    return fail(CVN_ERR_ARG, "a gradient of an argument that was not given");
  if (!empty && ((!grad_r && !grad_y) || (grad_y && !norm_w) || (norm_w && !base) ||
                 (((norm_w && grad_y) || post_w) && !stats)))
    return fail(CVN_ERR_ARG, "null pointer");
  if (!empty && x_type != CVN_F32 && grad_y && !h && (grad_r || grad_h))
    return fail(CVN_ERR_ARG, "a 16-bit residual is summed up again from its branch");
  if (!empty && !grad_y && (grad_norm_w || grad_norm_b))
    return fail(CVN_ERR_ARG, "gradients of the norm's parameters without a gradient of y");
  const bool sample = gate_kind == CVN_GATE_SAMPLE;
  const RnShape t = rn_shape(true, B, C, HW, sample);
  if (!workspace || workspace_bytes < cvn_residual_norm_bwd_workspace(B, C, HW, gate_kind))
    return fail(CVN_ERR_WORKSPACE, "residual_norm backward workspace missing or too small");
  const int64_t G = rn_bwd_blocks(t);
  hipStream_t st = (hipStream_t)stream;
  RnArgs a = {};
  a.part = (void*)align_up((size_t)workspace);
  a.dgpart = (float*)((char*)a.part + rn_part_bytes(C, t));
  a.x = base;
  a.h = h;
  a.gate = gate;
  a.gate_full = gate_kind == CVN_GATE_FULL;
  a.s = res_scale;
  a.nw = norm_w;
  a.pw = post_w;
  a.pb = post_b;
  a.stats = const_cast<float*>(stats);
  a.gr = grad_r;
  a.gy = grad_y;
  a.dx = grad_x;
  a.dh = grad_h;
  a.dg = grad_gate;
  a.C = C;
  a.HW = HW;
  a.total = B * HW;
  a.ntiles = t.ntiles;
  a.tps = t.tps;
  if (!empty) {
    rc = k.bwd(a, t, st);
    if (rc != CVN_OK) return rc;
  }
  RnSumArgs s = {};
  s.part = a.part;
  s.dgpart = a.dgpart;
  s.C = (int)C;
  s.G = (int)G;
  s.s = res_scale;
  s.pw = post_w;
  s.pb = post_b;
  s.dw = grad_norm_w;
  s.db = grad_norm_b;
  s.ds = grad_scale;
  s.dpw = grad_post_w;
  s.dpb = grad_post_b;
  if (sample && grad_gate) {
    s.dg = grad_gate;
    s.dg_type = h_type;
    s.tps = t.tps;
  }
  s.rows = C + (s.dg ? B * C : 0);
  if (!s.dw && !s.db && !s.ds && !s.dpw && !s.dpb && !s.dg) return CVN_OK;
  // a block for every 4 rows, as far as one launch goes: 2^26 gates of one tile each are more
  hipLaunchKernelGGL(t.px ? k_rn_sums<float> : k_rn_sums<double>, dim3((unsigned)std::min((s.rows + 3) / 4, rn_max_blocks(256))), dim3(256), 0, st, s);
  return check_launch("residual_norm sums");
}
