// 1x1 convolution of MXFP4 maps with MXFP4 matrices (the format: mxfp4.h):
//   y[b,n,p] = act(sum_c w[n][c] x[b,p][c] + bias[n]) [* res_scale[n] + residual[b,n,p]]
// on the matrix units' scaled 4-bit products, which multiply 32 codes of two rows with both blocks' scales and add in float32.
#include "mxfp4.h"

namespace cvn {
namespace {

constexpr int kThreads = 256;

template <class T>
__device__ __forceinline__ void mx_store(const MxOut& o, int64_t r, int64_t n, float v) {
  if (r >= o.rows || n >= o.N) return;
  const int64_t b = r / o.HW, i = (b * o.N + n) * o.HW + (r - b * o.HW);
  if (o.bias) v += o.bias[n];
  if (o.act == CVN_ACT_GELU) v = gelu_fast(v);
  if (o.res_scale) v *= o.res_scale[n];
  if (o.residual) v += (float)((const T*)o.residual)[i];
  ((T*)o.y)[i] = (T)v;
}

// A wave makes a tile of 16 channels and 16 pixels.  Of a step of 128 channels, lane l holds the block l / 16 of its
// operands' rows l % 16, and of the result channels 4 (l / 16) .. + 3 of pixel l % 16.
template <class T>
__global__ void __launch_bounds__(kThreads) k_mx_product(const mx_i32x4* __restrict__ xc, const uint8_t* __restrict__ xs,
                                                         const mx_i32x4* __restrict__ wc, const uint8_t* __restrict__ ws,
                                                         int KB, MxOut o) {
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int64_t tn = (o.N + 15) / 16, tr = (o.rows + 15) / 16, stride = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); t < tn * tr; t += stride) {
    const int64_t n0 = t / tr * 16, r0 = (t % tr) * 16;
    const int64_t wrow = min(n0 + j, o.N - 1) * KB, xrow = min(r0 + j, o.rows - 1) * KB;
    mx_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < KB; k += 4) {
      // past the last block both scales are 2^-127: what is read there instead is lost below float32's range
      const int kb = min(k + g, KB - 1);
      const int sw = k + g < KB ? ws[wrow + kb] : 0, sx = k + g < KB ? xs[xrow + kb] : 0;
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(wc[wrow + kb]), mx_operand(xc[xrow + kb]), acc,
                                                             kMxFp4, kMxFp4, 0, sw, 0, sx);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) mx_store<T>(o, r0 + j, n0 + 4 * g + e, acc[e]);
  }
}

template <class T>
int product(const void* xc, const void* xs, const void* wc, const void* ws, int64_t KB, const MxOut& o, hipStream_t st) {
  const int64_t tiles = (o.N + 15) / 16 * ((o.rows + 15) / 16);
  hipLaunchKernelGGL(k_mx_product<T>, dim3(mx_grid((tiles + 3) / 4, kThreads)), dim3(kThreads), 0, st, (const mx_i32x4*)xc,
                     (const uint8_t*)xs, (const mx_i32x4*)wc, (const uint8_t*)ws, (int)KB, o);
  return check_launch("conv1x1_mxfp4");
}

int mx_check_product(int64_t B, int64_t C, int64_t HW, int64_t N, int type) {
  if (B < 0 || HW < 0 || C < 1 || N < 1 || !mx_type_size(type)) return fail(CVN_ERR_ARG, "bad shape or type");
  if (C > kMxMaxChannels || N > kMxMaxChannels || (HW && B > kMxMaxRows / HW))
    return fail(CVN_ERR_UNSUPPORTED, "too many channels or pixels");
  return CVN_OK;
}

bool mx_overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

}  // namespace
}  // namespace cvn

using namespace cvn;

extern "C" size_t cvn_conv1x1_mxfp4_workspace(int quantized, int64_t B, int64_t C, int64_t HW, int64_t N) {
  if (mx_check_product(B, C, HW, N, CVN_F32) != CVN_OK || quantized) return 0;
  return align_up((size_t)(B * HW * mx_blocks(C)) * 17, 16);
}

extern "C" int cvn_conv1x1_mxfp4(const void* x, void* x_codes, void* x_scales, int64_t B, int64_t C, int64_t HW,
                                 const void* w_codes, const void* w_scales, int64_t N, const float* bias, int act,
                                 const void* residual, const float* res_scale, void* y, int type, void* workspace,
                                 size_t workspace_bytes, cvn_stream_t stream) {
  const int rc = mx_check_product(B, C, HW, N, type);
  if (rc != CVN_OK) return rc;
  if (act != CVN_ACT_NONE && act != CVN_ACT_GELU) return fail(CVN_ERR_ARG, "unknown activation");
  const int64_t rows = B * HW, KB = mx_blocks(C), es = mx_type_size(type);
  if (rows == 0) return CVN_OK;
  if (!w_codes || !w_scales || !y || (!x && !x_codes) || !x_codes != !x_scales) return fail(CVN_ERR_ARG, "null pointer");
  if (((uintptr_t)w_codes | (uintptr_t)x_codes) & 15) return fail(CVN_ERR_ARG, "codes must be aligned to 16 bytes");
  const int64_t ny = rows * N * es;
  if (mx_overlap(y, ny, x, rows * C * es) || mx_overlap(y, ny, w_codes, N * KB * 16) || mx_overlap(y, ny, w_scales, N * KB) ||
      mx_overlap(y, ny, x_codes, rows * KB * 16) || mx_overlap(y, ny, x_scales, rows * KB) ||
      (y != residual && mx_overlap(y, ny, residual, ny)))
    return fail(CVN_ERR_ARG, "the output shares memory with an input");
  if (x && !x_codes) {
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < cvn_conv1x1_mxfp4_workspace(0, B, C, HW, N))
      return fail(CVN_ERR_WORKSPACE, "workspace missing, too small or not aligned to 16 bytes");
    x_codes = workspace;
    x_scales = (char*)workspace + rows * KB * 16;
  }
  const hipStream_t st = (hipStream_t)stream;
  if (x) {
    const int q = mx_quantize(x, type, B, C, HW, x_codes, x_scales, st);
    if (q != CVN_OK) return q;
  }
  const MxOut o = {bias, res_scale, residual, y, HW, N, rows, act};
  if (type == CVN_F32) return product<float>(x_codes, x_scales, w_codes, w_scales, KB, o, st);
  if (type == CVN_BF16) return product<__bf16>(x_codes, x_scales, w_codes, w_scales, KB, o, st);
  return product<_Float16>(x_codes, x_scales, w_codes, w_scales, KB, o, st);
}
