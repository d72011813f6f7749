// Gradients of a 1x1 convolution of MXFP4 operands, straight through their quantisation (the format: mxfp4.h):
//   gx[b,c,p] = sum_n w[n][c] gy[b,n,p]     gw[n][c] = sum_{b,p} gy[b,n,p] x[b,p][c]     gb[n] = sum_{b,p} gy[b,n,p]
// The 4-bit values times their scales are bfloat16 numbers, and gy is a sum of them: one (bfloat16), two (float16: 11 bits in
// 8 + 3) or three (float32: 24 bits in 8 + 8 + 8).  So the products run on the bfloat16 matrix units, one a part, with no operand
// rounded, and are summed in float32.  (Those units take numbers below 2^-126 for zeros: parts of gy, and 4-bit values of the
// smallest scales.)
#include <algorithm>

#include "mxfp4.h"

namespace cvn {
namespace {

typedef __bf16 mx_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef short mx_i16x4 __attribute__((ext_vector_type(4)));
typedef short mx_i16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
enum { kGradX, kGradW };

template <class T>
struct MxGrad;  // values of a 16-byte vector, parts of a value, terms of a step of gx and of gw
// (gw of 8 x 64 x 256 x 256 float32 to 128: 96 us by steps of 128 bytes of a channel, 76 by 256, with gx 150 and 145; of
// bfloat16 40 and 36.5, but with gx 65 and 66.5)
template <>
struct MxGrad<float> {
  static constexpr int V = 4, P = 3, K = 32, KW = 64;
};
template <>
struct MxGrad<__bf16> {
  static constexpr int V = 8, P = 1, K = 64, KW = 64;
};
template <>
struct MxGrad<_Float16> {
  static constexpr int V = 8, P = 2, K = 64, KW = 64;
};

// A value's parts, largest first.
__device__ __forceinline__ void mx_split(__bf16 v, __bf16* p) { p[0] = v; }
__device__ __forceinline__ void mx_split(_Float16 v, __bf16* p) {
  const float f = (float)v;
  p[0] = (__bf16)f;
  const float r = f - (float)p[0];
  p[1] = (__bf16)(r == r ? r : 0.f);  // (infinities and NaNs are whole in the first part)
}
__device__ __forceinline__ __bf16 mx_top(float v) { return __builtin_bit_cast(__bf16, (short)(__float_as_uint(v) >> 16)); }
__device__ __forceinline__ void mx_split(float v, __bf16* p) {
  p[0] = mx_top(v == v ? v : __uint_as_float(0x7fc00000u));  // (a NaN cut short may look like an infinity)
  const float r = v - (float)p[0], s = r == r ? r : 0.f;
  p[1] = mx_top(s);
  p[2] = mx_top(s - (float)p[1]);
}

struct MxGradArgs {
  const void* gy;
  const mx_i32x4* codes;  // of the matrix (gx) or the map (gw)
  const uint8_t* scales;
  int64_t C, N, HW, rows;
  int KB;
  void* out;       // gx, or gw and its parts [splits][N][C]
  double* gb;      // gw: parts [splits][N], or null
  int64_t terms;   // of a split
  int ta, tb;
};

// D[i][k] = sum over terms of A's row i and B's row k, in tiles of BA x BB, a quarter to a wave.  gx: A are the matrix' columns
// (c), B the pixels, the terms n.  gw: A are the channels of gy (n), B those of x (c), the terms the pixels, shared out over
// the splits.  The codes come by terms, 32 neighbours of a tile's rows to a block, and lie in LDS as they come, in bfloat16: a
// transposing read gives a lane the terms of its column.  gy comes either way: its terms side by side (gw of maps, gx of one
// pixel a sample: ONE), or by terms.
template <class T, int KIND, bool ONE, int BA, int BB>
struct MxTile {
  typedef MxGrad<T> G;
  static constexpr int V = G::V, P = G::P, K = KIND == kGradX ? G::K : G::KW;
  static constexpr int BC = KIND == kGradX ? BA : BB, BG = KIND == kGradX ? BB : BA;  // rows of the codes' and gy's tile
  static constexpr bool kByTerms = (KIND == kGradX) != ONE;                           // gy's tile [terms][rows]
  static constexpr int GR = kByTerms ? K : BG, GC = kByTerms ? BG : K;                // its rows and columns as stored
  // Rows are padded so that what 16 lanes read at once lies in different banks: 32 bytes of four rows for the
  // transposing reads (64 of four for the two halves of a tile), 16 of neighbouring rows otherwise.
  static constexpr int CS = BC * 2 + 64, GS = GC * 2 + (kByTerms ? 64 : 16);
  static constexpr int kLds = K * CS + P * GR * GS;
};

template <class T, int KIND, bool ONE, int BA, int BB>
__device__ __forceinline__ void mx_grad(const MxGradArgs& a, int t, int split, char* lds) {
  typedef MxTile<T, KIND, ONE, BA, BB> M;
  constexpr int V = M::V, P = M::P, K = M::K, BC = M::BC, GR = M::GR, GC = M::GC, CS = M::CS, GS = M::GS;
  constexpr int BG = M::BG;
  constexpr bool kByTerms = M::kByTerms;
  constexpr int NG = GR * GC / V / kThreads, NC = (K * BC / 32 + kThreads - 1) / kThreads;
  char* const lc = lds;
  char* const lg = lds + K * CS;
  typedef T W __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, j = lane & 31, h = lane >> 5;

  const int64_t a0 = (int64_t)(t % a.ta) * BA, b0 = (int64_t)(t / a.ta) * BB;
  const int64_t c0 = KIND == kGradX ? a0 : b0, g0 = KIND == kGradX ? b0 : a0;
  const int64_t terms = KIND == kGradX ? a.N : a.rows;
  const int64_t k_first = (int64_t)split * a.terms, k_end = min(terms, k_first + a.terms);
  const T* const gy = (const T*)a.gy;

  // What is under way from memory for the next step.  (Two steps under way change nothing: 33 us either way for gx of 8192
  // bfloat16 pixels, 1024 to 1024 channels.)
  struct Step {
    W g[NG];
    mx_i32x4 q[NC];
    unsigned qs[NC];
  };
  // This thread's first vector of gy's tile and piece of the codes' (the others: a fixed number of rows on).
  constexpr int RG = kThreads / (GC / V), RC = kThreads / (BC / 32);
  const int grow = tid / (GC / V), gcol = tid % (GC / V) * V, crow = tid / (BC / 32), cpiece = tid % (BC / 32);
  // A tile whose rows are all there, with every vector in one sample, is read without a look at each vector.
  const bool inside = g0 + BG <= (KIND == kGradX ? a.rows : a.N) && c0 / 32 + BC / 32 <= a.KB && (ONE || a.HW % V == 0);
  const int64_t ghop = ONE ? a.N : a.HW;  // elements from a row of gy's tile to the next
  auto load = [&](int64_t k0, Step& s) {
    const bool fast = inside && k0 + K <= k_end;
    const mx_i32x4* codes = a.codes + (k0 + crow) * a.KB + c0 / 32 + cpiece;
    const uint8_t* scales = a.scales + (k0 + crow) * a.KB + c0 / 32 + cpiece;
    if (fast) {
      const int64_t k = k0 + (kByTerms ? grow : gcol), m = g0 + (kByTerms ? gcol : grow);
      const int64_t n = KIND == kGradX ? k : m, r = KIND == kGradX ? m : k;
      const int64_t b = ONE ? r : (uint32_t)r / (uint32_t)a.HW;
      const T* src = gy + (ONE ? r * a.N + n : (b * a.N + n) * a.HW + (r - b * a.HW));
#pragma unroll
      for (int i = 0; i < NG; ++i) s.g[i] = *(const W*)(src + i * RG * ghop);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        s.q[i] = mx_i32x4{0, 0, 0, 0};
        s.qs[i] = 127;
        if (kThreads * (i + 1) <= K * BC / 32 || crow + i * RC < K) {
          s.q[i] = codes[(int64_t)i * RC * a.KB];
          s.qs[i] = scales[(int64_t)i * RC * a.KB];
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int row = grow + i * RG;
      s.g[i] = W{};
      const int64_t k = k0 + (kByTerms ? row : gcol), m = g0 + (kByTerms ? gcol : row);
      const int64_t n = KIND == kGradX ? k : m, r = KIND == kGradX ? m : k;
      const int64_t n_end = KIND == kGradX ? k_end : a.N, r_end = KIND == kGradX ? a.rows : k_end;
      if (n >= n_end || r >= r_end) continue;
      if (ONE) {  // (rows, N): vectors along n
        const T* src = gy + r * a.N + n;
        asm volatile("" : "+v"(src));
        if (n + V <= n_end) {
          s.g[i] = *(const W*)src;
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (n + e < n_end) s.g[i][e] = src[e];
        }
      } else {  // (B, N, HW): vectors along the pixels
        int64_t b = (uint32_t)r / (uint32_t)a.HW, p = r - b * a.HW;
        const T* src = gy + (b * a.N + n) * a.HW + p;
        asm volatile("" : "+v"(src), "+v"(p));  // (addresses of single elements kept over the loop would fill the registers)
        if (p + V <= a.HW && r + V <= r_end) {
          s.g[i] = *(const W*)src;
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (r + e < r_end) s.g[i][e] = *src;
            ++src;
            if (++p == a.HW) p = 0, src += (a.N - 1) * a.HW;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      s.q[i] = mx_i32x4{0, 0, 0, 0};
      s.qs[i] = 127;
      if (crow + i * RC < K && k0 + crow + i * RC < k_end && c0 / 32 + cpiece < a.KB) {
        s.q[i] = codes[(int64_t)i * RC * a.KB];
        s.qs[i] = scales[(int64_t)i * RC * a.KB];
      }
    }
  };
  // Sums of gy over the pixels, of the rows or columns that this thread loads.
  constexpr int NB = KIND != kGradW ? 1 : kByTerms ? V : NG;
  double sum[NB] = {};
  auto store = [&](const Step& s) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int row = grow + i * RG;
      __bf16 part[P][V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        __bf16 x[P];
        mx_split(s.g[i][e], x);
#pragma unroll
        for (int p = 0; p < P; ++p) part[p][e] = x[p];
      }
      typedef __bf16 S __attribute__((ext_vector_type(V)));
#pragma unroll
      for (int p = 0; p < P; ++p) *(S*)(lg + (p * GR + row) * GS + gcol * 2) = *(const S*)part[p];
      if (KIND == kGradW && a.gb && b0 == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) sum[(kByTerms ? e : i) % NB] += (double)(float)s.g[i][e];
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int row = crow + i * RC;
      if (row >= K) continue;
      const float scale = mx_scale(s.qs[i]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const mx_bf16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)s.q[i][w], scale, 0),
                        v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)s.q[i][w], scale, 1),
                        v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)s.q[i][w], scale, 2),
                        v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)s.q[i][w], scale, 3);
        *(mx_bf16x8*)(lc + row * CS + cpiece * 64 + w * 16) = mx_bf16x8{v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
      }
    }
  };
  // Eight terms, 16 step + 8 (l / 32) on, of row `row` + l % 32 of a tile.
  typedef __attribute__((address_space(3))) mx_i16x4* lds_i16x4;
  auto by_terms = [&](const char* base, int stride, int row, int step) {
    const char* p = base + (16 * step + 8 * h + (lane & 15) / 4) * stride + (row + (lane & 16) + (lane & 3) * 4) * 2;
    const mx_i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)p),
                   hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(p + 4 * stride));
    return __builtin_bit_cast(mx_bf16x8, mx_i16x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w});
  };
  auto side_by_side = [&](const char* base, int row, int step) {
    return *(const mx_bf16x8*)(base + (row + j) * GS + (16 * step + 8 * h) * 2);
  };

  constexpr int TA = BA / 64, TB = BB / 64, TC = KIND == kGradX ? TA : TB, TG = KIND == kGradX ? TB : TA;
  const int wa = (wave & 1) * (BA / 2), wb = (wave >> 1) * (BB / 2);
  const int wc = KIND == kGradX ? wa : wb, wg = KIND == kGradX ? wb : wa;
  mx_f32x16 acc[TA][TB];
#pragma unroll
  for (int i = 0; i < TA; ++i)
#pragma unroll
    for (int k = 0; k < TB; ++k) acc[i][k] = mx_f32x16{};
  auto step = [&](int64_t k0, Step& st) {
    __syncthreads();
    store(st);
    __syncthreads();
    if (k0 + K < k_end) load(k0 + K, st);
    // Each sixteen terms' operands come from LDS while the ones before are multiplied.
    mx_bf16x8 c[2][TC], y[2][P][TG];
    auto operands = [&](int s) {
#pragma unroll
      for (int i = 0; i < TC; ++i) c[s & 1][i] = by_terms(lc, CS, wc + 32 * i, s);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < TG; ++i) {
          const char* base = lg + p * GR * GS;
          y[s & 1][p][i] = kByTerms ? by_terms(base, GS, wg + 32 * i, s) : side_by_side(base, wg + 32 * i, s);
        }
    };
    operands(0);
#pragma unroll
    for (int s = 0; s < K / 16; ++s) {
      if (s + 1 < K / 16) operands(s + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int p = P - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
          for (int k = 0; k < TB; ++k)
            acc[i][k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(KIND == kGradX ? c[s & 1][i] : y[s & 1][p][i],
                                                                KIND == kGradX ? y[s & 1][p][k] : c[s & 1][k], acc[i][k], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  Step st;
  load(k_first, st);
  for (int64_t k0 = k_first; k0 < k_end; k0 += K) step(k0, st);

  // Element e of a 32 x 32 result is its row 8 (e / 4) + 4 h + e % 4, column j.
#pragma unroll
  for (int k = 0; k < TB; ++k) {
    const int64_t col = b0 + wb + 32 * k + j;
    if (KIND == kGradX) {
      if (col >= a.rows) continue;
      const int64_t b = (uint32_t)col / (uint32_t)a.HW;
      T* out = (T*)a.out + b * a.C * a.HW + (col - b * a.HW);
#pragma unroll
      for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int64_t c = a0 + wa + 32 * i + 8 * (e / 4) + 4 * h + e % 4;
          if (c < a.C) out[c * a.HW] = (T)acc[i][k][e];
        }
    } else {
      if (col >= a.C) continue;
      float* out = (float*)a.out + (int64_t)split * a.N * a.C + col;
#pragma unroll
      for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int64_t n = a0 + wa + 32 * i + 8 * (e / 4) + 4 * h + e % 4;
          if (n < a.N) out[n * a.C] = acc[i][k][e];
        }
    }
  }
  if (KIND == kGradW && a.gb && b0 == 0) {
    double* const out = a.gb + (int64_t)split * a.N;
    if (!kByTerms) {  // the threads of a row are neighbours
      constexpr int TR = GC / V;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        double s = sum[i % NB];
#pragma unroll
        for (int d = TR / 2; d >= 1; d >>= 1) s += __shfl_xor(s, d);
        const int64_t n = a0 + (tid + i * kThreads) / TR;
        if (tid % TR == 0 && n < a.N) out[n] = s;
      }
    } else {  // those of a column are GC / V apart
      constexpr int TR = GC / V;
      double(*red)[GC] = (double(*)[GC])lds;
      static_assert(sizeof(double) * GC * (kThreads / TR) <= M::kLds, "sums fit the operands' memory");
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) red[tid / TR][tid % TR * V + e] = sum[e % NB];
      __syncthreads();
      for (int c = tid; c < GC; c += kThreads) {
        double s = 0.;
        for (int i = 0; i < kThreads / TR; ++i) s += red[i][c];
        if (a0 + c < a.N) out[a0 + c] = s;
      }
    }
  }
}

template <class T, int KIND, bool ONE, int BA, int BB>
__global__ void __launch_bounds__(kThreads, 2) k_mx_grad(MxGradArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[MxTile<T, KIND, ONE, BA, BB>::kLds];
  const int tiles = a.ta * a.tb;
  mx_grad<T, KIND, ONE, BA, BB>(a, blockIdx.x % tiles, blockIdx.x / tiles, lds);
}
// Both gradients, the blocks of gw first, whose sums a kernel behind waits for.  (Against a launch each, with the sums: float16
// maps of 3x67x45, 48 to 80 channels, 27.7 us and here 14.5; float32 of 8x96x96, 64 to 128, 41.5 and 32.6; float32 of
// 8x256x256, 64 to 128, 164 and 145; bfloat16 of 4x31x33, 2048 to 512, 103 and 88.  gw has tiles of 64 of gy's channels: tiles
// of 128 leave a CU fewer blocks of either kind, and the four take 17.3, 35.5, 171 and 96 us; they are better by 3% where
// bfloat16 of 8x32x32 goes from 1024 to 1024 channels, 76 us to 79.)
template <class T, bool ONE, int XA, int WB>
__global__ void __launch_bounds__(kThreads, 2) k_mx_grads(MxGradArgs x, MxGradArgs w, int wblocks) {
  constexpr int kX = MxTile<T, kGradX, ONE, XA, 128>::kLds, kW = MxTile<T, kGradW, ONE, 64, WB>::kLds;
  __shared__ __attribute__((aligned(16))) char lds[kX > kW ? kX : kW];
  if ((int)blockIdx.x < wblocks) {
    const int tiles = w.ta * w.tb;
    mx_grad<T, kGradW, ONE, 64, WB>(w, blockIdx.x % tiles, blockIdx.x / tiles, lds);
  } else {
    mx_grad<T, kGradX, ONE, XA, 128>(x, blockIdx.x - wblocks, 0, lds);
  }
}

// The sum over the splits, in the same order on every call: R threads an element take every R-th of them.  (One thread an
// element leaves few to wait for long chains of loads: 256 splits of 8192 elements take 70 us that way, 16 threads 6.6; 64 of 65536
// 19 and 7.6; but 16 of 262144, where one thread takes over, 7.1 and 9.6, and 4 of a million 6.4 and 28.6.)
template <int R>
__global__ void __launch_bounds__(kThreads) k_mx_grad_join(const float* __restrict__ part, int64_t n,
                                                           const double* __restrict__ gbp, int64_t nb, int splits,
                                                           float* __restrict__ gw, float* __restrict__ gb) {
  constexpr int kCols = kThreads / R;
  __shared__ double red[R][kCols];
  const int col = threadIdx.x % kCols, row = threadIdx.x / kCols;
  const int64_t blocks = (n + kCols - 1) / kCols;
  const bool bias = blockIdx.x >= blocks;
  const int64_t i = ((int64_t)blockIdx.x - (bias ? blocks : 0)) * kCols + col, end = bias ? nb : n;
  double s = 0.;
  if (i < end) {
#pragma unroll 8
    for (int k = row; k < splits; k += R) s += bias ? gbp[k * nb + i] : (double)part[k * n + i];
  }
  if (R > 1) {
    red[row][col] = s;
    __syncthreads();
  }
  if (row == 0 && i < end) {
#pragma unroll
    for (int k = 1; k < R; ++k) s += red[k][col];
    (bias ? gb : gw)[i] = (float)s;
  }
}

template <int R>
void grad_join(const float* part, int64_t n, const double* gbp, int64_t nb, int64_t splits, float* gw, float* gb, hipStream_t st) {
  constexpr int kCols = kThreads / R;
  const int64_t blocks = (n + kCols - 1) / kCols + (gb ? (nb + kCols - 1) / kCols : 0);
  hipLaunchKernelGGL(k_mx_grad_join<R>, dim3((unsigned)blocks), dim3(kThreads), 0, st, part, n, gbp, nb, (int)splits, gw, gb);
}

// The bias' gradient alone: a block for a channel.
template <class T>
__global__ void __launch_bounds__(kThreads) k_mx_grad_bias(const T* __restrict__ gy, int64_t N, int64_t HW, int64_t rows,
                                                           float* __restrict__ gb) {
  __shared__ double red[kThreads / 64];
  const int64_t n = blockIdx.x;
  double s = 0.;
  for (int64_t r = threadIdx.x; r < rows; r += kThreads) {
    const int64_t b = (uint32_t)r / (uint32_t)HW;
    s += (double)(float)gy[(b * N + n) * HW + (r - b * HW)];
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) gb[n] = (float)(red[0] + red[1] + red[2] + red[3]);
}

__global__ void __launch_bounds__(kThreads) k_mx_zero(float* p, int64_t n, float* q, int64_t m) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n || i < m; i += (int64_t)gridDim.x * kThreads) {
    if (i < n) p[i] = 0.f;
    if (i < m) q[i] = 0.f;
  }
}

// How gw's terms (the pixels) are shared out: enough splits for two blocks a CU, of at least 256 pixels, in whole steps.
struct MxSplit {
  int64_t terms, splits;
};
MxSplit mx_split_terms(int64_t rows, int64_t C, int64_t N) {
  const int64_t tiles = (N + 63) / 64 * ((C + 127) / 128);
  const int64_t want = std::max<int64_t>(1, std::min((rows + 255) / 256, 512 / tiles));
  MxSplit s;
  s.terms = std::max<int64_t>(256, ((rows + want - 1) / want + 63) / 64 * 64);
  s.splits = (rows + s.terms - 1) / s.terms;
  return s;
}
size_t mx_part_bytes(const MxSplit& s, int64_t C, int64_t N) {
  return (s.splits > 1 ? align_up((size_t)(s.splits * N * C) * sizeof(float)) : 0) + (size_t)(s.splits * N) * sizeof(double);
}

// The launches of one shape of tiles; x, w: null where that gradient is not wanted.
template <class T, bool ONE, int XA, int WB>
int grad_tiles(MxGradArgs* x, MxGradArgs* w, int64_t C, int64_t N, int64_t rows, int64_t splits, hipStream_t st) {
  int64_t xblocks = 0, wblocks = 0;
  if (x) {
    const int64_t ta = (C + XA - 1) / XA, tb = (rows + 127) / 128;
    xblocks = ta * tb;
    x->ta = (int)ta, x->tb = (int)tb;
  }
  if (w) {
    const int64_t ta = (N + 63) / 64, tb = (C + WB - 1) / WB;
    wblocks = ta * tb * splits;
    w->ta = (int)ta, w->tb = (int)tb;
  }
  if ((xblocks + wblocks) * kThreads >= (int64_t)1 << 32) return fail(CVN_ERR_UNSUPPORTED, "too many pixels and channels");
  const dim3 grid((unsigned)(xblocks + wblocks));
  if (x && w) hipLaunchKernelGGL((k_mx_grads<T, ONE, XA, WB>), grid, dim3(kThreads), 0, st, *x, *w, (int)wblocks);
  else if (x) hipLaunchKernelGGL((k_mx_grad<T, kGradX, ONE, XA, 128>), grid, dim3(kThreads), 0, st, *x);
  else hipLaunchKernelGGL((k_mx_grad<T, kGradW, ONE, 64, WB>), grid, dim3(kThreads), 0, st, *w);
  return check_launch("conv1x1_mxfp4_backward");
}

template <class T, bool ONE>
int grads(const void* gy, const void* xc, const void* xs, const void* wc, const void* ws, int64_t C, int64_t HW, int64_t rows,
          int64_t N, void* gx, float* gw, float* gb, void* work, hipStream_t st) {
  const int KB = (int)mx_blocks(C);
  const MxSplit s = mx_split_terms(rows, C, N);
  float* const part = s.splits > 1 ? (float*)work : gw;
  double* const gbp = (double*)((char*)work + (s.splits > 1 ? align_up((size_t)(s.splits * N * C) * sizeof(float)) : 0));
  MxGradArgs x = {gy, (const mx_i32x4*)wc, (const uint8_t*)ws, C, N, HW, rows, KB, gx, nullptr, N, 0, 0};
  MxGradArgs w = {gy, (const mx_i32x4*)xc, (const uint8_t*)xs, C, N, HW, rows, KB, part, gb ? gbp : nullptr, s.terms, 0, 0};
  if (gx || gw) {
    MxGradArgs *px = gx ? &x : nullptr, *pw = gw ? &w : nullptr;
    // (256 pixels, 2048 to 2048 channels: gx 36 us by 32 tiles of 128 channels, 25 by 64 of 64)
    const bool few = (C + 127) / 128 * ((rows + 127) / 128) < 256;
    const int rc = C <= 64 ? grad_tiles<T, ONE, 64, 64>(px, pw, C, N, rows, s.splits, st)
                   : few   ? grad_tiles<T, ONE, 64, 128>(px, pw, C, N, rows, s.splits, st)
                           : grad_tiles<T, ONE, 128, 128>(px, pw, C, N, rows, s.splits, st);
    if (rc != CVN_OK) return rc;
  }
  if (gw && (s.splits > 1 || gb)) {
    const int64_t n = s.splits > 1 ? N * C : 0;
    if (n >= 1 << 18) grad_join<1>(part, n, gbp, N, s.splits, gw, gb, st);
    else grad_join<16>(part, n, gbp, N, s.splits, gw, gb, st);
  } else if (gb && !gw) {
    hipLaunchKernelGGL(k_mx_grad_bias<T>, dim3((unsigned)N), dim3(kThreads), 0, st, (const T*)gy, N, HW, rows, gb);
  }
  return check_launch("conv1x1_mxfp4_backward");
}

template <class T>
int grads(const void* gy, const void* xc, const void* xs, const void* wc, const void* ws, int64_t C, int64_t HW, int64_t rows,
          int64_t N, void* gx, float* gw, float* gb, void* work, hipStream_t st) {
  return HW == 1 ? grads<T, true>(gy, xc, xs, wc, ws, C, HW, rows, N, gx, gw, gb, work, st)
                 : grads<T, false>(gy, xc, xs, wc, ws, C, HW, rows, N, gx, gw, gb, work, st);
}

int mx_check_grad(int64_t B, int64_t C, int64_t HW, int64_t N) {
  if (B < 0 || HW < 0 || C < 1 || N < 1) return fail(CVN_ERR_ARG, "bad shape");
  if (C > kMxMaxChannels || N > kMxMaxChannels || (HW && B > kMxMaxRows / HW))
    return fail(CVN_ERR_UNSUPPORTED, "too many channels or pixels");
  return CVN_OK;
}

}  // namespace
}  // namespace cvn

using namespace cvn;

extern "C" size_t cvn_conv1x1_mxfp4_bwd_workspace(int64_t B, int64_t C, int64_t HW, int64_t N) {
  if (mx_check_grad(B, C, HW, N) != CVN_OK || B * HW == 0) return 0;
  return mx_part_bytes(mx_split_terms(B * HW, C, N), C, N);
}

extern "C" int cvn_conv1x1_mxfp4_bwd(const void* grad_y, int type, const void* x_codes, const void* x_scales,
                                     const void* w_codes, const void* w_scales, int64_t B, int64_t C, int64_t HW, int64_t N,
                                     void* grad_x, float* grad_w, float* grad_bias, void* workspace, size_t workspace_bytes,
                                     cvn_stream_t stream) {
  const int rc = mx_check_grad(B, C, HW, N);
  if (rc != CVN_OK) return rc;
  if (!mx_type_size(type)) return fail(CVN_ERR_ARG, "bad type");
  if (!grad_x && !grad_w && !grad_bias) return CVN_OK;
  const int64_t rows = B * HW;
  const hipStream_t st = (hipStream_t)stream;
  if (rows == 0) {
    if (grad_w || grad_bias)
      hipLaunchKernelGGL(k_mx_zero, dim3(256), dim3(kThreads), 0, st, grad_w, grad_w ? N * C : 0, grad_bias, grad_bias ? N : 0);
    return check_launch("conv1x1_mxfp4_backward");
  }
  if (!grad_y || (grad_x && (!w_codes || !w_scales)) || (grad_w && (!x_codes || !x_scales)))
    return fail(CVN_ERR_ARG, "null pointer");
  if (((uintptr_t)w_codes | (uintptr_t)x_codes) & 15) return fail(CVN_ERR_ARG, "codes must be aligned to 16 bytes");
  const int64_t es = mx_type_size(type), KB = mx_blocks(C);
  const MxMem mem[] = {{grad_x, rows * C * es},
                       {grad_w, N * C * 4},
                       {grad_bias, N * 4},  // written up to here
                       {grad_y, rows * N * es},
                       {grad_w ? x_codes : nullptr, rows * KB * 16},
                       {grad_w ? x_scales : nullptr, rows * KB},
                       {grad_x ? w_codes : nullptr, N * KB * 16},
                       {grad_x ? w_scales : nullptr, N * KB}};
  if (mx_shared(mem, 3, 8)) return fail(CVN_ERR_ARG, "an output shares memory with an input or another output");
  if (grad_w && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < cvn_conv1x1_mxfp4_bwd_workspace(B, C, HW, N)))
    return fail(CVN_ERR_WORKSPACE, "workspace missing, too small or not aligned to 16 bytes");
  if (type == CVN_F32)
    return grads<float>(grad_y, x_codes, x_scales, w_codes, w_scales, C, HW, rows, N, grad_x, grad_w, grad_bias, workspace, st);
  if (type == CVN_BF16)
    return grads<__bf16>(grad_y, x_codes, x_scales, w_codes, w_scales, C, HW, rows, N, grad_x, grad_w, grad_bias, workspace, st);
  return grads<_Float16>(grad_y, x_codes, x_scales, w_codes, w_scales, C, HW, rows, N, grad_x, grad_w, grad_bias, workspace, st);
}
