// Quantisation of maps and matrices to MXFP4, and back (the format: mxfp4.h).
#include "mxfp4.h"

namespace cvn {
namespace {

constexpr int kThreads = 256;

// Maps: a lane quantises a block of V neighbouring pixels, a wave that of 64 V, and the waves of a tile of pixels its
// blocks of channels one after the other: the 16 bytes that a row gets from each meet in the cache.  (Block by block over
// the whole map, 64 channel blocks of 16384 bfloat16 pixels took 38 us.)
template <class T, int V>
__global__ void __launch_bounds__(kThreads) k_mx_quantize(const T* __restrict__ x, int64_t C, int64_t HW, int64_t rows, int KB,
                                                          mx_i32x4* __restrict__ codes, uint8_t* __restrict__ scales) {
  typedef T W __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  const int lane = threadIdx.x & 63;
  const int64_t units = (rows + 64 * V - 1) / (64 * V) * KB, stride = (int64_t)gridDim.x * (kThreads / 64);
  int64_t u = (int64_t)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (; u < units; u += stride) {
    const int64_t tile = u / KB, kb = u - tile * KB, r0 = (tile * 64 + lane) * V;
    if (r0 >= rows) continue;
    const int n = (int)min((int64_t)kMxBlock, C - kb * kMxBlock);
    int64_t b = (uint32_t)r0 / (uint32_t)HW, p = r0 - b * HW;
    W t[kMxBlock];
    if (V == 1 || (p + V <= HW && r0 + V <= rows)) {
      const T* src = x + (b * C + kb * kMxBlock) * HW + p;
#pragma unroll
      for (int c = 0; c < kMxBlock; ++c) {
        t[c] = W{};
        if (c < n) t[c] = *(const W*)src;
        src += HW;
        asm volatile("" : "+v"(src));  // (32 addresses would fill the registers)
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const T* src = x + (b * C + kb * kMxBlock) * HW + p;
        const int ne = r0 + e < rows ? n : 0;
#pragma unroll
        for (int c = 0; c < kMxBlock; ++c) {
          t[c][e] = c < ne ? *src : (T)0.f;
          src += HW;
          asm volatile("" : "+v"(src));
        }
        if (++p == HW) p = 0, ++b;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float v[kMxBlock];
      unsigned mag = 0;
#pragma unroll
      for (int c = 0; c < kMxBlock; ++c) {
        v[c] = (float)t[c][e];
        mag = max(mag, mx_mag(v[c]));
      }
      const unsigned s = mx_scale_code(mag);
      if (r0 + e < rows) {
        codes[(r0 + e) * KB + kb] = mx_pack32(v, s);
        scales[(r0 + e) * KB + kb] = (uint8_t)s;
      }
    }
  }
}

// Rows (a matrix, or one pixel a sample): four lanes to a block, eight neighbouring channels each.
template <class T>
__global__ void __launch_bounds__(kThreads) k_mx_quantize_rows(const T* __restrict__ x, int64_t C, int64_t rows, int KB,
                                                               unsigned* __restrict__ codes, uint8_t* __restrict__ scales) {
  typedef T W __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const int64_t total = rows * KB * 4, stride = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < (total + 63) / 64 * 64; i += stride) {
    const int64_t at = min(i, total - 1), blk = at >> 2, r = blk / KB, c0 = (blk - r * KB) * kMxBlock + (at & 3) * 8;
    const T* src = x + r * C + c0;
    float v[8];
    if (c0 + 8 <= C) {
      const W t = *(const W*)src;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c0 + e < C ? (float)src[e] : 0.f;
    }
    unsigned mag = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) mag = max(mag, mx_mag(v[e]));
    mag = max(mag, (unsigned)__shfl_xor((int)mag, 1));
    mag = max(mag, (unsigned)__shfl_xor((int)mag, 2));
    const unsigned s = mx_scale_code(mag);
    const unsigned q = s == 255u ? 0u : mx_pack8(v, mx_scale(s));
    if (i < total) {
      codes[i] = q;
      if ((i & 3) == 0) scales[blk] = (uint8_t)s;
    }
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

// Rows: a thread makes eight neighbouring channels.  (Blocks to threads, 8192 x 2048 float32 take 89 us.)
template <class T>
__global__ void __launch_bounds__(kThreads) k_mx_dequantize_rows(const unsigned* __restrict__ codes,
                                                                 const uint8_t* __restrict__ scales, int64_t C, int64_t rows,
                                                                 int KB, T* __restrict__ y) {
  typedef T W __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const int64_t total = rows * KB * 4, stride = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += stride) {
    const int64_t blk = i >> 2, r = blk / KB, c0 = (blk - r * KB) * kMxBlock + (i & 3) * 8;
    float v[8];
    mx_unpack8(codes[i], mx_scale(scales[blk]), v);
    T* dst = y + r * C + c0;
    if (c0 + 8 <= C) {
      W t;
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
      *(W*)dst = t;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e < C) dst[e] = (T)v[e];
    }
  }
}

int mx_check(int64_t B, int64_t C, int64_t HW, int type, const void* codes) {
  if (B < 0 || HW < 0 || C < 1 || !mx_type_size(type)) return fail(CVN_ERR_ARG, "bad shape or type");
  if (C > kMxMaxChannels || (HW && B > kMxMaxRows / HW)) return fail(CVN_ERR_UNSUPPORTED, "too many channels or pixels");
  if ((uintptr_t)codes & 15) return fail(CVN_ERR_ARG, "codes must be aligned to 16 bytes");
  return CVN_OK;
}

template <class T, int V>
void quantize_map(const T* x, int64_t C, int64_t HW, int64_t rows, int KB, void* codes, void* scales, hipStream_t st) {
  const int64_t units = (rows + 64 * V - 1) / (64 * V) * KB;
  hipLaunchKernelGGL((k_mx_quantize<T, V>), dim3(mx_grid((units + 3) / 4, kThreads)), dim3(kThreads), 0, st, x, C, HW, rows, KB,
                     (mx_i32x4*)codes, (uint8_t*)scales);
}

template <class T>
int quantize(const void* x, int64_t B, int64_t C, int64_t HW, void* codes, void* scales, hipStream_t st) {
  const int64_t rows = B * HW, KB = mx_blocks(C);
  if (HW == 1) {
    hipLaunchKernelGGL(k_mx_quantize_rows<T>, dim3(mx_grid((rows * KB * 4 + kThreads - 1) / kThreads, kThreads)), dim3(kThreads),
                       0, st, (const T*)x, C, rows, (int)KB, (unsigned*)codes, (uint8_t*)scales);
  } else {
    // 4 bytes of a channel to a lane: 16 x 64 x 256 x 256 float32 55, 54, 59 us at 1, 2, 4 pixels, bfloat16 76, 33, 39
    quantize_map<T, 4 / (int)sizeof(T)>((const T*)x, C, HW, rows, (int)KB, codes, scales, st);
  }
  return check_launch("mxfp4_quantize");
}

template <class T>
int dequantize(const void* codes, const void* scales, int64_t B, int64_t C, int64_t HW, void* y, hipStream_t st) {
  const int64_t rows = B * HW, KB = mx_blocks(C);
  if (HW == 1) {
    hipLaunchKernelGGL(k_mx_dequantize_rows<T>, dim3(mx_grid((rows * KB * 4 + kThreads - 1) / kThreads, kThreads)), dim3(kThreads),
                       0, st, (const unsigned*)codes, (const uint8_t*)scales, C, rows, (int)KB, (T*)y);
    return check_launch("mxfp4_dequantize");
  }
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
  const int64_t blocks = B * HW * mx_blocks(C);
  const MxMem mem[] = {{codes, 16 * blocks}, {scales, blocks}, {x, B * HW * C * mx_type_size(x_type)}};
  if (mx_shared(mem, 2, 3)) return fail(CVN_ERR_ARG, "an output shares memory with the input or another output");
  return mx_quantize(x, x_type, B, C, HW, codes, scales, (hipStream_t)stream);
}

extern "C" int cvn_mxfp4_dequantize(const void* codes, const void* scales, int64_t B, int64_t C, int64_t HW, void* y,
                                    int y_type, cvn_stream_t stream) {
  const int rc = mx_check(B, C, HW, y_type, codes);
  if (rc != CVN_OK) return rc;
  if (B * HW == 0) return CVN_OK;
  if (!y || !codes || !scales) return fail(CVN_ERR_ARG, "null pointer");
  const int64_t blocks = B * HW * mx_blocks(C);
  const MxMem mem[] = {{y, B * HW * C * mx_type_size(y_type)}, {codes, 16 * blocks}, {scales, blocks}};
  if (mx_shared(mem, 1, 3)) return fail(CVN_ERR_ARG, "the output shares memory with an input");
  if (y_type == CVN_F32) return dequantize<float>(codes, scales, B, C, HW, y, (hipStream_t)stream);
  if (y_type == CVN_BF16) return dequantize<__bf16>(codes, scales, B, C, HW, y, (hipStream_t)stream);
  return dequantize<_Float16>(codes, scales, B, C, HW, y, (hipStream_t)stream);
}
