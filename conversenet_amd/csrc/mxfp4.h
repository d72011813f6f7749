// Microscaled 4-bit floating point (MXFP4): what the translation units of mxfp4*.hip share.
//
// A row (a pixel's channels, or a matrix row) is cut into blocks of 32 values.  A block has a scale 2^(s - 127), s a byte,
// and a 4-bit code a value: sign, then 0, 0.5, 1, 1.5, 2, 3, 4, 6.
//   s = max(0, e - 2), e the biased exponent of the block's largest magnitude: floor(log2) of it, less 2
//   code = nearest to x / 2^(s - 127), ties to the even code, at most 6
//   a block that holds an infinity or a NaN: s = 255, and every value of it is NaN
// Stored by rows: codes [rows][KB][16] (the even value of a byte in its lower half), scales [rows][KB], KB = ceil(C / 32);
// values past C are zeros.  The matrix units read both as they are.
#pragma once
#include "cvn_common.h"

namespace cvn {

typedef int mx_i32x4 __attribute__((ext_vector_type(4)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMxBlock = 32;
inline int64_t mx_blocks(int64_t C) { return (C + kMxBlock - 1) / kMxBlock; }

// Limits of every entry point: rows are counted in 31 bits, channels in 16.
constexpr int64_t kMxMaxChannels = 65536;
constexpr int64_t kMxMaxRows = ((int64_t)1 << 31) - 256;
// Threads of a launch stay below 2^32.
inline unsigned mx_grid(int64_t blocks, int threads) {
  const int64_t most = (((int64_t)1 << 32) - 1) / threads;
  return (unsigned)(blocks < most ? blocks : most);
}

// Memory of a call, and whether the first `written` pieces of n share any with each other or with the rest.
struct MxMem {
  const void* p;  // or null
  int64_t n;      // bytes
};
inline bool mx_shared(const MxMem* m, int written, int n) {
  for (int i = 0; i < written; ++i)
    for (int k = i + 1; k < n; ++k) {
      const uintptr_t x = (uintptr_t)m[i].p, y = (uintptr_t)m[k].p;
      if (x && y && x < y + (uintptr_t)m[k].n && y < x + (uintptr_t)m[i].n) return true;
    }
  return false;
}

inline int mx_type_size(int type) { return type == CVN_F32 ? 4 : type == CVN_BF16 || type == CVN_F16 ? 2 : 0; }

// The bits of a magnitude as float32: ordered as integers, with infinities and NaNs above all numbers.
__device__ __forceinline__ unsigned mx_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// Scale code of a block whose largest magnitude has these bits.
__device__ __forceinline__ unsigned mx_scale_code(unsigned mag) {
  const unsigned e = mag >> 23;
  return e == 255u ? 255u : max(e, 2u) - 2u;
}
// 2^(s - 127) as float32 (s = 255: infinity, which the conversions take for NaN).
__device__ __forceinline__ float mx_scale(unsigned s) { return __uint_as_float(s ? s << 23 : 0x00400000u); }

// Eight values to their codes.
__device__ __forceinline__ unsigned mx_pack8(const float* v, float scale) {
  unsigned q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
  return q;
}
// A block's values to its codes, of scale code s (of a block that holds no number they are zeros).
__device__ __forceinline__ mx_i32x4 mx_pack32(const float* v, unsigned s) {
  const float scale = mx_scale(s);
  const mx_i32x4 q = {(int)mx_pack8(v, scale), (int)mx_pack8(v + 8, scale), (int)mx_pack8(v + 16, scale),
                      (int)mx_pack8(v + 24, scale)};
  return s == 255u ? mx_i32x4{0, 0, 0, 0} : q;
}
// Eight codes to their values.
__device__ __forceinline__ void mx_unpack8(unsigned q, float scale, float* v) {
  mx_f32x2 t;
  t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0), v[0] = t.x, v[1] = t.y;
  t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1), v[2] = t.x, v[3] = t.y;
  t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2), v[4] = t.x, v[5] = t.y;
  t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3), v[6] = t.x, v[7] = t.y;
}

// A 4-bit operand of the matrix units: 32 codes a lane (the upper half of the builtin's operand is for wider types).
__device__ __forceinline__ mx_i32x8 mx_operand(mx_i32x4 q) { return mx_i32x8{q.x, q.y, q.z, q.w, 0, 0, 0, 0}; }
constexpr int kMxFp4 = 4;  // the builtins' number of the type

// GELU(x) = max(x, 0) - |x| Q(|x|), Q the upper tail of the normal distribution: log2 Q is smooth, so Q = 2^p(|x|) with a polynomial p
// whose largest error a |2^p(a) - Q(a)| over 0 .. 6 is near the least for its degree (9.5e-9, at 1.69; a linear program over 3000
// points found it) and which falls beyond.  14 issue slots, four of them the exponential's, against 20 of gelu_fast, whose reciprocal takes
// four more: 8 x 64 x 256 x 256 bfloat16 to 128 channels 50 us, 53 with that.  The largest error in float32 is 1.4e-7 for |x| < 3.9 and
// 6.0e-8 |x| beyond (gelu_fast: 3.3e-7).  Infinities are the caller's.
__device__ __forceinline__ float mx_gelu(float x) {
  const float a = fabsf(x);
  float p = fmaf(-1.690395606601669e-06f, a, 2.5083225409616716e-05f);
  p = fmaf(p, a, -0.00011446223652455956f);
  p = fmaf(p, a, -0.00032334341085515916f);
  p = fmaf(p, a, 0.0073333862237632275f);
  p = fmaf(p, a, -0.05271419882774353f);
  p = fmaf(p, a, -0.4591154456138611f);
  p = fmaf(p, a, -1.151123285293579f);
  p = fmaf(p, a, -0.9999988675117493f);
  return fmaf(-a, __builtin_amdgcn_exp2f(p), __builtin_amdgcn_fmed3f(x, 0.0f, __builtin_inff()));
}

// One product y[r][n] = sum_c x[r][c] w[n][c] and what is done to it on its way out, y and the residual channels first.
struct MxOut {
  const float* bias;       // [N] or null
  const float* res_scale;  // [N] or null
  const void* residual;    // as y, or null
  void* y;
  int64_t HW, N, rows;  // rows = B HW
  int act;
  bool lines;  // rows of y start on cache lines
};

int mx_quantize(const void* x, int type, int64_t B, int64_t C, int64_t HW, void* codes, void* scales, hipStream_t st);

}  // namespace cvn
