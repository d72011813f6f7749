// Quantisation of maps and matrices to MXFP4, and back (the format: mxfp4.h).
#include "mxfp4.h"

namespace cvn {
namespace {

constexpr int kThreads = 256;

// A thread quantises a block of a row: neighbouring threads take neighbouring pixels of the same channels.
template <class T>
__global__ void __launch_bounds__(kThreads) k_mx_quantize(const T* __restrict__ x, int64_t C, int64_t HW, int64_t rows, int KB,
                                                          uint4* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t stride = (int64_t)gridDim.x * kThreads, total = rows * KB;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += stride) {
    const int64_t kb = i / rows, r = i - kb * rows;
    const int64_t b = r / HW, p = r - b * HW;
    const T* src = x + (b * C + kb * kMxBlock) * HW + p;
    const int n = (int)min((int64_t)kMxBlock, C - kb * kMxBlock);
    float v[kMxBlock];
    unsigned mag = 0;
#pragma unroll
    for (int c = 0; c < kMxBlock; ++c) {
      v[c] = c < n ? (float)src[c * HW] : 0.f;
      mag = max(mag, mx_mag(v[c]));
    }
    const unsigned s = mx_scale_code(mag);
    const float scale = mx_scale(s);
    uint4 q = {mx_pack8(v, scale), mx_pack8(v + 8, scale), mx_pack8(v + 16, scale), mx_pack8(v + 24, scale)};
    if (s == 255u) q = uint4{0, 0, 0, 0};
    codes[r * KB + kb] = q;
    scales[r * KB + kb] = (uint8_t)s;
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_mx_dequantize(const uint4* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            int64_t C, int64_t HW, int64_t rows, int KB, T* __restrict__ y) {
  const int64_t stride = (int64_t)gridDim.x * kThreads, total = rows * KB;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += stride) {
    const int64_t kb = i / rows, r = i - kb * rows;
    const int64_t b = r / HW, p = r - b * HW;
    T* dst = y + (b * C + kb * kMxBlock) * HW + p;
    const int n = (int)min((int64_t)kMxBlock, C - kb * kMxBlock);
    const float scale = mx_scale(scales[r * KB + kb]);
    const uint4 q = codes[r * KB + kb];
    float v[kMxBlock];
    mx_unpack8(q.x, scale, v), mx_unpack8(q.y, scale, v + 8), mx_unpack8(q.z, scale, v + 16), mx_unpack8(q.w, scale, v + 24);
#pragma unroll
    for (int c = 0; c < kMxBlock; ++c)
      if (c < n) dst[c * HW] = (T)v[c];
  }
}

int mx_check(int64_t B, int64_t C, int64_t HW, int type, const void* codes) {
  if (B < 0 || HW < 0 || C < 1 || !mx_type_size(type)) return fail(CVN_ERR_ARG, "bad shape or type");
  if (C > kMxMaxChannels || (HW && B > kMxMaxRows / HW)) return fail(CVN_ERR_UNSUPPORTED, "too many channels or pixels");
  if ((uintptr_t)codes & 15) return fail(CVN_ERR_ARG, "codes must be aligned to 16 bytes");
  return CVN_OK;
}

template <class T>
int quantize(const void* x, int64_t B, int64_t C, int64_t HW, void* codes, void* scales, hipStream_t st) {
  const int64_t rows = B * HW, KB = mx_blocks(C);
  hipLaunchKernelGGL(k_mx_quantize<T>, dim3(mx_grid((rows * KB + kThreads - 1) / kThreads, kThreads)), dim3(kThreads), 0, st,
                     (const T*)x, C, HW, rows, (int)KB, (uint4*)codes, (uint8_t*)scales);
  return check_launch("mxfp4_quantize");
}

template <class T>
int dequantize(const void* codes, const void* scales, int64_t B, int64_t C, int64_t HW, void* y, hipStream_t st) {
  const int64_t rows = B * HW, KB = mx_blocks(C);
  hipLaunchKernelGGL(k_mx_dequantize<T>, dim3(mx_grid((rows * KB + kThreads - 1) / kThreads, kThreads)), dim3(kThreads), 0, st,
                     (const uint4*)codes, (const uint8_t*)scales, C, HW, rows, (int)KB, (T*)y);
  return check_launch("mxfp4_dequantize");
}

}  // namespace

int mx_quantize(const void* x, int type, int64_t B, int64_t C, int64_t HW, void* codes, void* scales, hipStream_t st) {
  if (type == CVN_F32) return quantize<float>(x, B, C, HW, codes, scales, st);
  if (type == CVN_BF16) return quantize<__bf16>(x, B, C, HW, codes, scales, st);
  return quantize<_Float16>(x, B, C, HW, codes, scales, st);
}

}  // namespace cvn

using namespace cvn;

extern "C" int cvn_mxfp4_quantize(const void* x, int x_type, int64_t B, int64_t C, int64_t HW, void* codes, void* scales,
                                  cvn_stream_t stream) {
  const int rc = mx_check(B, C, HW, x_type, codes);
  if (rc != CVN_OK) return rc;
  if (B * HW == 0) return CVN_OK;
  if (!x || !codes || !scales) return fail(CVN_ERR_ARG, "null pointer");
  return mx_quantize(x, x_type, B, C, HW, codes, scales, (hipStream_t)stream);
}

extern "C" int cvn_mxfp4_dequantize(const void* codes, const void* scales, int64_t B, int64_t C, int64_t HW, void* y,
                                    int y_type, cvn_stream_t stream) {
  const int rc = mx_check(B, C, HW, y_type, codes);
  if (rc != CVN_OK) return rc;
  if (B * HW == 0) return CVN_OK;
  if (!y || !codes || !scales) return fail(CVN_ERR_ARG, "null pointer");
  if (y_type == CVN_F32) return dequantize<float>(codes, scales, B, C, HW, y, (hipStream_t)stream);
  if (y_type == CVN_BF16) return dequantize<__bf16>(codes, scales, B, C, HW, y, (hipStream_t)stream);
  return dequantize<_Float16>(codes, scales, B, C, HW, y, (hipStream_t)stream);
}
