// Gradients of a 1x1 convolution of MXFP4 operands, straight through their quantisation (the format: mxfp4.h):
//   gx[b,c,p] = sum_n w[n][c] gy[b,n,p]     gw[n][c] = sum_{b,p} gy[b,n,p] x[b,p][c]     gb[n] = sum_{b,p} gy[b,n,p]
// with the 4-bit values as they are: no operand is rounded.
#include "mxfp4.h"

namespace cvn {
namespace {

constexpr int kThreads = 256;

// A thread makes eight channels of a pixel.
template <class T>
__global__ void __launch_bounds__(kThreads) k_mx_grad_x(const T* __restrict__ gy, const unsigned* __restrict__ wc,
                                                        const uint8_t* __restrict__ ws, int64_t C, int64_t N, int64_t HW,
                                                        int64_t rows, int KB, T* __restrict__ gx) {
  const int64_t stride = (int64_t)gridDim.x * kThreads, total = rows * ((C + 7) / 8);
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += stride) {
    const int64_t c8 = i / rows, r = i - c8 * rows, b = r / HW, p = r - b * HW;
    float acc[8] = {};
    for (int64_t n = 0; n < N; ++n) {
      float w[8];
      mx_unpack8(wc[n * KB * 4 + c8], mx_scale(ws[n * KB + c8 / 4]), w);
      const float g = (float)gy[(b * N + n) * HW + p];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(g, w[e], acc[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c8 * 8 + e < C) gx[(b * C + c8 * 8 + e) * HW + p] = (T)acc[e];
  }
}

// A block makes eight entries of a row of the matrix' gradient, its threads take the pixels in turn.
template <class T>
__global__ void __launch_bounds__(kThreads) k_mx_grad_w(const T* __restrict__ gy, const unsigned* __restrict__ xc,
                                                        const uint8_t* __restrict__ xs, int64_t C, int64_t N, int64_t HW,
                                                        int64_t rows, int KB, float* __restrict__ gw, float* __restrict__ gb) {
  __shared__ double red[kThreads / 64][9];
  const int64_t c8s = (C + 7) / 8;
  for (int64_t t = blockIdx.x; t < N * c8s; t += gridDim.x) {
    const int64_t n = t / c8s, c8 = t - n * c8s;
    double acc[9] = {};
    for (int64_t r = threadIdx.x; r < rows; r += kThreads) {
      const int64_t b = r / HW, p = r - b * HW;
      float v[8] = {};
      if (gw) mx_unpack8(xc[r * KB * 4 + c8], mx_scale(xs[r * KB + c8 / 4]), v);
      const double g = (double)(float)gy[(b * N + n) * HW + p];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fma(g, (double)v[e], acc[e]);
      acc[8] += g;
    }
#pragma unroll
    for (int e = 0; e < 9; ++e) {
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) acc[e] += __shfl_xor(acc[e], d);
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][e] = acc[e];
    }
    __syncthreads();
    if (threadIdx.x < 9) {
      double s = 0.;
      for (int i = 0; i < kThreads / 64; ++i) s += red[i][threadIdx.x];
      const int64_t c = c8 * 8 + threadIdx.x;
      if (threadIdx.x < 8) {
        if (gw && c < C) gw[n * C + c] = (float)s;
      } else if (gb && c8 == 0) {
        gb[n] = (float)s;
      }
    }
    __syncthreads();
  }
}

template <class T>
int grads(const void* gy, const void* xc, const void* xs, const void* wc, const void* ws, int64_t C, int64_t HW, int64_t rows,
          int64_t N, void* gx, float* gw, float* gb, hipStream_t st) {
  const int KB = (int)mx_blocks(C);
  if (gx && rows)
    hipLaunchKernelGGL(k_mx_grad_x<T>, dim3(mx_grid((rows * ((C + 7) / 8) + kThreads - 1) / kThreads, kThreads)),
                       dim3(kThreads), 0, st, (const T*)gy, (const unsigned*)wc, (const uint8_t*)ws, C, N, HW, rows, KB, (T*)gx);
  if (gw || gb)
    hipLaunchKernelGGL(k_mx_grad_w<T>, dim3(mx_grid(N * (gw ? (C + 7) / 8 : 1), kThreads)), dim3(kThreads), 0, st,
                       (const T*)gy, (const unsigned*)xc, (const uint8_t*)xs, gw ? C : 1, N, HW, rows, KB, gw, gb);
  return check_launch("conv1x1_mxfp4_backward");
}

}  // namespace
}  // namespace cvn

using namespace cvn;

extern "C" size_t cvn_conv1x1_mxfp4_bwd_workspace(int64_t B, int64_t C, int64_t HW, int64_t N) {
  (void)B, (void)C, (void)HW, (void)N;
  return 0;
}

extern "C" int cvn_conv1x1_mxfp4_bwd(const void* grad_y, int type, const void* x_codes, const void* x_scales,
                                     const void* w_codes, const void* w_scales, int64_t B, int64_t C, int64_t HW, int64_t N,
                                     void* grad_x, float* grad_w, float* grad_bias, void* workspace, size_t workspace_bytes,
                                     cvn_stream_t stream) {
  (void)workspace, (void)workspace_bytes;
  if (B < 0 || HW < 0 || C < 1 || N < 1 || !mx_type_size(type)) return fail(CVN_ERR_ARG, "bad shape or type");
  if (C > kMxMaxChannels || N > kMxMaxChannels || (HW && B > kMxMaxRows / HW))
    return fail(CVN_ERR_UNSUPPORTED, "too many channels or pixels");
  if (!grad_x && !grad_w && !grad_bias) return CVN_OK;
  const int64_t rows = B * HW;
  if ((rows && !grad_y) || (grad_x && rows && (!w_codes || !w_scales)) || (grad_w && rows && (!x_codes || !x_scales)))
    return fail(CVN_ERR_ARG, "null pointer");
  if (((uintptr_t)w_codes | (uintptr_t)x_codes) & 15) return fail(CVN_ERR_ARG, "codes must be aligned to 16 bytes");
  const hipStream_t st = (hipStream_t)stream;
  if (type == CVN_F32) return grads<float>(grad_y, x_codes, x_scales, w_codes, w_scales, C, HW, rows, N, grad_x, grad_w, grad_bias, st);
  if (type == CVN_BF16)
    return grads<__bf16>(grad_y, x_codes, x_scales, w_codes, w_scales, C, HW, rows, N, grad_x, grad_w, grad_bias, st);
  return grads<_Float16>(grad_y, x_codes, x_scales, w_codes, w_scales, C, HW, rows, N, grad_x, grad_w, grad_bias, st);
}
