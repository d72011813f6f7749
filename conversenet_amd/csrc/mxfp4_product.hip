// 1x1 convolution of MXFP4 maps with MXFP4 matrices (the format: mxfp4.h):
//   y[b,n,p] = act(sum_c w[n][c] x[b,p][c] + bias[n]) [* res_scale[n] + residual[b,n,p]]
// on the matrix units' scaled 4-bit products, which multiply 32 codes of two rows with both blocks' scales and add in float32.
#include <algorithm>

#include "mxfp4.h"

namespace cvn {
namespace {

// Operands of a product as the kernels read them; `x` is null where the map is given in MXFP4.
struct MxIn {
  const void* x;
  mx_i32x4* xc;  // read, or written where x is given and they are kept
  uint8_t* xs;
  const mx_i32x4* wc;
  const uint8_t* ws;
  int64_t C;
  int KB;
};

template <class T, int V>
struct MxVec {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <class T>
struct MxVec<T, 1> {
  typedef T type;
};

// Where a lane's V neighbouring pixels from row r0 on lie.
struct MxGroup {
  int64_t r0, b, p;
  bool whole;  // all in one sample
};
template <int V>
__device__ __forceinline__ MxGroup mx_group(int64_t r0, int64_t HW, int64_t rows) {
  MxGroup g;
  g.r0 = r0;
  g.b = (uint32_t)r0 / (uint32_t)HW;  // (rows are below 2^31)
  g.p = r0 - g.b * HW;
  g.whole = r0 + V <= rows && g.p + V <= HW;
  return g;
}

// What happens to R rows of V sums with their bias on the way out: act, residual scale.
template <int V, int R>
__device__ __forceinline__ void mx_finish(const MxOut& o, float (*v)[V], const float (*scale)[V]) {
  if (o.act == CVN_ACT_GELU) {
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < V; ++e) top = fmaxf(top, fabsf(v[r][e]));
    if (top == __builtin_inff()) {  // (mx_gelu makes 0 times infinity of it)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e)
          v[r][e] = fabsf(v[r][e]) == __builtin_inff() ? fmaxf(v[r][e], 0.f) : mx_gelu(v[r][e]);
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) v[r][e] = mx_gelu(v[r][e]);
    }
  }
  if (o.res_scale) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < V; ++e) v[r][e] *= scale[r][e];
  }
}

// Stores R rows, `step` elements apart, of V finished values side by side, from element `at` of the first on.  NT: past the
// caches, for rows that start on cache lines (8 x 64 x 256 x 256 float32 to 128 channels: 74 us, through the caches 98); a
// line that two waves store parts of is better put together in the cache (64 x 321 x 481 to 128: 30 us, past it 42).
template <class T, bool NT, int V, int R>
__device__ __forceinline__ void mx_store_rows(const MxOut& o, int64_t at, int64_t step, float (*v)[V]) {
  typedef typename MxVec<T, V>::type W;
  if (o.residual) {
    W res[R];
#pragma unroll
    for (int r = 0; r < R; ++r) res[r] = *(const W*)((const T*)o.residual + at + r * step);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < V; ++e) v[r][e] += (float)((const T*)&res[r])[e];
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    W out;
#pragma unroll
    for (int e = 0; e < V; ++e) ((T*)&out)[e] = (T)v[r][e];
    W* const to = (W*)((T*)o.y + at + r * step);
    if (NT) __builtin_nontemporal_store(out, to);
    else *to = out;
  }
}

// V elements of a row (channel n of a group's pixels), and which of them there are.
template <int V>
struct MxPixels {
  int64_t at[V];
  int live;
};
template <int V>
__device__ __forceinline__ MxPixels<V> mx_pixels(const MxOut& o, const MxGroup& g, int64_t n) {
  MxPixels<V> x;
  x.live = 0;
  int64_t b = g.b, p = g.p;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    x.at[e] = (b * o.N + n) * o.HW + p;
    x.live |= (g.r0 + e < o.rows) << e;
    if (++p == o.HW) p = 0, ++b;
  }
  return x;
}
// A row of them, `step` elements further on, one by one.
template <class T, int V>
__device__ __forceinline__ void mx_store_pixels(const MxOut& o, const MxPixels<V>& x, int64_t step, const float* v) {
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (x.live >> e & 1) {
      const int64_t i = x.at[e] + step;
      ((T*)o.y)[i] = (T)(o.residual ? v[e] + (float)((const T*)o.residual)[i] : v[e]);
    }
}

// ------------------------------------------------------------------------------------------------
// Many pixels of many channels: both operands in MXFP4, tiles staged through LDS.
// ------------------------------------------------------------------------------------------------
// 16384 pixels, 2048 to 4096 channels: 136 us behind the quantisation, 2.0 PFLOP/s (137 to 152 us call after call; a library's
// 8192^3 product: 3.1 PFLOP/s), bound by the wait for each step's fetch; the matrix units are busy a fifth
// of the time, LDS an eighth.  Another order of the tiles, two patches of the longer side, changes nothing.
// A step takes 256 channels: 128 bytes of codes a row, which a wave fetches 8 rows at a time straight into LDS.  A row's
// 16-byte pieces are stored in an order that depends on the row (piece ^ (row / 2 & 7)), so that 16 lanes which read the
// same piece of neighbouring rows hit all 64 banks.  Lane l of a 32 x 32 x 64 product takes the blocks 4 (l / 32) + s of rows
// l % 32 in steps s < 4: its four scales are one word.  Past the last block the codes of that block stand in, and both
// scales are 2^-127: the products are lost below float32's range.
constexpr int kStep = 8;  // blocks of a step

// The word of four scales at byte `at` of an operand's scales, as loaded from `last` at most, where the last whole word is
// (from there the four are shifted: mx_scales_tail) ..
__device__ __forceinline__ unsigned mx_scales_load(const uint8_t* s, int at, int last) {
  typedef unsigned U __attribute__((aligned(1)));
  return *(const U*)(s + (int64_t)min(at, last));
}
// .. and put right, for blocks kb .. of KB: 0 past the last.
__device__ __forceinline__ unsigned mx_scales_tail(unsigned v, int at, int last, int kb, int KB) {
  if (kb >= KB) return 0;
  v >>= 8 * (at - min(at, last));
  return KB - kb < 4 ? v & ((1u << (8 * (KB - kb))) - 1) : v;
}

typedef __attribute__((address_space(3))) void* mx_lds;
typedef const __attribute__((address_space(1))) void* mx_glob;

// Tiles of BA x BB rows of the two operands, WA x WB of them to a wave.  MAP: A is the matrix, B the pixels, and a lane
// stores TB pixels of a channel; otherwise (one pixel a sample) A is the pixels, and it stores TB channels of a pixel.
// In either case lane j of the TB 32-row tiles of a wave holds the rows TB j + 0 .. TB - 1 of B.
// A block makes tile after tile, and fetches the first step of the next before it stores.
template <class T, bool MAP, bool NT, int BA, int BB, int WA, int WB>
__global__ void __launch_bounds__((BA / WA) * (BB / WB) * 64, 1)
    k_mx_gemm(const mx_i32x4* __restrict__ ac, const uint8_t* __restrict__ as, int64_t na, const mx_i32x4* __restrict__ bc,
              const uint8_t* __restrict__ bs, int64_t nb, int KB, int ta, int tb, MxOut o) {
  constexpr int NW = (BA / WA) * (BB / WB), TA = WA / 32, TB = WB / 32;
  constexpr int D = TB;  // rows of B between neighbouring lanes
  constexpr int kBytes = (BA + BB) * 128;
  constexpr int LA = BA / 8 / NW, LB = BB / 8 / NW;
  static_assert(NW % 2 == 0, "a wave's fetches of a tile put a row's pieces in one order");
  extern __shared__ char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 31, h = lane >> 5;
  const int wa = wave % (BA / WA) * WA, wb = wave / (BA / WA) * WB;
  const int nt = ta * tb;

  // A tile's place, and what a wave reads of it: rows 8 (wave + NW i) + lane / 8 of its codes, its rows' scales.  (32-bit offsets
  // from the tile's first row: 128 rows of 65536 channels are 4 MB.)
  int64_t ra, rb;
  const char *acodes, *bcodes;
  const uint8_t *ascales, *bscales;
  int alast, blast;
  uint32_t aoff[LA], boff[LB];
  int as_at[TA], bs_at[TB];
  const int piece = (lane & 7) ^ ((4 * wave + (lane >> 4)) & 7);
  auto place = [&](int t) {
    // Blocks of one XCD take a run of tiles, in patches of eight A tiles: its L2 holds what they share.
    const int per = nt / 8, rem = nt % 8, x = t & 7, i8 = t >> 3;
    const int tile = x < rem ? x * (per + 1) + i8 : rem * (per + 1) + (x - rem) * per + i8;
    const int patch = tile / (8 * tb), a0 = patch * 8, aw = min(8, ta - a0), in = tile - patch * 8 * tb;
    ra = (int64_t)(a0 + in % aw) * BA, rb = (int64_t)(in / aw) * BB;
    acodes = (const char*)(ac + ra * KB), bcodes = (const char*)(bc + rb * KB);
    ascales = as + ra * KB, bscales = bs + rb * KB;
    const int amost = (int)min((int64_t)BA, na - ra) - 1, bmost = (int)min((int64_t)BB, nb - rb) - 1;
    alast = (int)min((na - ra) * KB, (int64_t)1 << 30) - 4, blast = (int)min((nb - rb) * KB, (int64_t)1 << 30) - 4;
#pragma unroll
    for (int i = 0; i < LA; ++i) aoff[i] = (uint32_t)(min(8 * (wave + NW * i) + (lane >> 3), amost) * KB) * 16;
#pragma unroll
    for (int i = 0; i < LB; ++i) {  // row 32 v + j of a wave's part in LDS is its row D j + v
      const int row = 8 * (wave + NW * i) + (lane >> 3), in = row % WB;
      boff[i] = (uint32_t)(min(row - in + D * (in % 32) + in / 32, bmost) * KB) * 16;
    }
#pragma unroll
    for (int i = 0; i < TA; ++i) as_at[i] = min(wa + 32 * i + j, amost) * KB + 4 * h;
#pragma unroll
    for (int i = 0; i < TB; ++i) bs_at[i] = min(wb + D * j + i, bmost) * KB + 4 * h;
  };
  unsigned sa[TA], sb[TB];
  auto fetch = [&](int kb0, char* buf) {
    const uint32_t at = (uint32_t)min(kb0 + piece, KB - 1) * 16;
#pragma unroll
    for (int i = 0; i < LA; ++i)
      __builtin_amdgcn_global_load_lds((mx_glob)(acodes + (aoff[i] + at)), (mx_lds)(buf + (wave + NW * i) * 1024), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < LB; ++i)
      __builtin_amdgcn_global_load_lds((mx_glob)(bcodes + (boff[i] + at)), (mx_lds)(buf + BA * 128 + (wave + NW * i) * 1024),
                                       16, 0, 0);
#pragma unroll
    for (int i = 0; i < TA; ++i) sa[i] = mx_scales_load(ascales, as_at[i] + kb0, alast);
#pragma unroll
    for (int i = 0; i < TB; ++i) sb[i] = mx_scales_load(bscales, bs_at[i] + kb0, blast);
  };

  place(blockIdx.x);
  fetch(0, smem);
  int cur = 0;
  // bias and residual scale of a tile's channels, behind the operands, for this tile and the next
  constexpr int NC = MAP ? BA : BB;
  float* bias = (float*)(smem + 2 * kBytes);
  for (int t = blockIdx.x;;) {
    const int64_t ra0 = ra, rb0 = rb;
    const int next = t + (int)gridDim.x;
    float* const rscale = bias + NC;
    for (int i = threadIdx.x; i < NC; i += NW * 64) {
      const int64_t n = (MAP ? ra0 : rb0) + i;
      bias[i] = o.bias && n < o.N ? o.bias[n] : 0.f;
      rscale[i] = o.res_scale && n < o.N ? o.res_scale[n] : 1.f;
    }

    mx_f32x16 acc[TA][TB];
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
      for (int k = 0; k < TB; ++k) acc[i][k] = mx_f32x16{};
    for (int kb0 = 0; kb0 < KB; kb0 += kStep) {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      unsigned ua[TA], ub[TB];
#pragma unroll
      for (int i = 0; i < TA; ++i) ua[i] = sa[i];
#pragma unroll
      for (int i = 0; i < TB; ++i) ub[i] = sb[i];
      if (kb0 + kStep < KB) {
        fetch(kb0 + kStep, smem + (cur ^ 1) * kBytes);
      } else {
#pragma unroll
        for (int i = 0; i < TA; ++i) ua[i] = mx_scales_tail(ua[i], as_at[i] + kb0, alast, kb0 + 4 * h, KB);
#pragma unroll
        for (int i = 0; i < TB; ++i) ub[i] = mx_scales_tail(ub[i], bs_at[i] + kb0, blast, kb0 + 4 * h, KB);
        if (next < nt) {
          place(next);
          fetch(0, smem + (cur ^ 1) * kBytes);
        }
      }
      const char* buf = smem + cur * kBytes;
      // Each quarter's operands come from LDS while the ones before are multiplied.
      mx_i32x4 a[2][TA], b[2][TB];
      auto operands = [&](int s) {
#pragma unroll
        for (int i = 0; i < TA; ++i) {
          const int row = wa + 32 * i + j;
          a[s & 1][i] = *(const mx_i32x4*)(buf + row * 128 + (((4 * h + s) ^ (row >> 1 & 7)) << 4));
        }
#pragma unroll
        for (int i = 0; i < TB; ++i) {
          const int row = wb + 32 * i + j;
          b[s & 1][i] = *(const mx_i32x4*)(buf + (BA + row) * 128 + (((4 * h + s) ^ (row >> 1 & 7)) << 4));
        }
      };
      operands(0);
#define MX_STEP(s)                                                                                                 \
  if (s < 3) operands(s + 1);                                                                                      \
  __builtin_amdgcn_sched_barrier(0);                                                                               \
  _Pragma("unroll") for (int i = 0; i < TA; ++i) _Pragma("unroll") for (int k = 0; k < TB; ++k) acc[i][k] =        \
      __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(a[s & 1][i]), mx_operand(b[s & 1][k]), acc[i][k], \
                                                      kMxFp4, kMxFp4, s, ua[i], s, ub[k]);                         \
  __builtin_amdgcn_sched_barrier(0);
      MX_STEP(0) MX_STEP(1) MX_STEP(2) MX_STEP(3)  // (the byte of a scale word is part of the instruction)
#undef MX_STEP
      cur ^= 1;
    }

    // Element e of a 32 x 32 result is its row 8 (e / 4) + 4 h + e % 4, column j.
    const int64_t c0 = rb0 + wb + D * j, a0 = ra0 + wa + 4 * h, step = MAP ? o.HW : o.N;  // this lane's first column and row
    MxPixels<TB> at;
    bool whole = c0 + TB <= nb;
    if (MAP) {
      const MxGroup grp = mx_group<TB>(min(c0, nb - 1), o.HW, o.rows);
      at = mx_pixels<TB>(o, grp, a0);
      whole = grp.whole;
    } else {
      at.live = 0;
#pragma unroll
      for (int k = 0; k < TB; ++k) at.at[k] = a0 * o.N + c0 + k, at.live |= (c0 + k < nb) << k;
    }
    if (c0 < nb) {
#pragma unroll
      for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int off = 32 * i + 8 * q;
          float v[4][TB], ss[4][TB];
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int k = 0; k < TB; ++k) {
              const int n = MAP ? wa + off + 4 * h + r : wb + D * j + k;
              v[r][k] = acc[i][k][4 * q + r] + bias[n], ss[r][k] = rscale[n];
            }
          mx_finish<TB, 4>(o, v, ss);
          const int64_t left = na - a0 - off;
          if (whole && left >= 4) {
            mx_store_rows<T, NT, TB, 4>(o, at.at[0] + off * step, step, v);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r < left) mx_store_pixels<T, TB>(o, at, (off + r) * step, v[r]);
          }
        }
    }
    if (next >= nt) return;
    t = next;
    bias = bias == (float*)(smem + 2 * kBytes) ? bias + 2 * NC : bias - 2 * NC;
  }
}

template <class T, bool MAP, bool NT, int BA, int BB, int WA, int WB>
int gemm_tile(const MxIn& in, const MxOut& o, hipStream_t st) {
  constexpr int kThreads = (BA / WA) * (BB / WB) * 64, kLds = 2 * (BA + BB) * 128 + 16 * (MAP ? BA : BB);
  const int64_t na = MAP ? o.N : o.rows, nb = MAP ? o.rows : o.N;
  const int64_t ta = (na + BA - 1) / BA, tb = (nb + BB - 1) / BB;
  if (ta * tb >= (int64_t)1 << 30) return fail(CVN_ERR_UNSUPPORTED, "too many pixels and channels");
  auto k = k_mx_gemm<T, MAP, NT, BA, BB, WA, WB>;
  static std::atomic<uint64_t> done;
  once_per_device(done, [&] { (void)hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, kLds); });
  // as many blocks as the CUs hold at once; each takes tiles in turn
  static std::atomic<int> most[64];
  std::atomic<int>& m = most[current_device() & 63];
  if (!m.load(std::memory_order_relaxed)) {
    int per = 0, cus = 0;
    (void)hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, (const void*)k, kThreads, kLds);
    (void)hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, current_device());
    m.store(std::max(8, std::max(1, per) * cus / 8 * 8), std::memory_order_relaxed);
  }
  const int64_t blocks = std::min<int64_t>(ta * tb, m.load(std::memory_order_relaxed));
  hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(kThreads), kLds, st, MAP ? in.wc : in.xc, MAP ? in.ws : in.xs, na,
                     MAP ? in.xc : in.wc, MAP ? in.xs : in.ws, nb, in.KB, (int)ta, (int)tb, o);
  return check_launch("conv1x1_mxfp4");
}

template <class T, bool MAP>
int gemm(const MxIn& in, const MxOut& o, hipStream_t st) {
  // Tiles of 128 from one for every CU on, 64 below.  (16384 pixels, 2048 to 4096 channels: 136 us, 64: 230; 8192 pixels, 1024 to
  // 1024: 14.3, 64: 22.8; 4092 pixels, 1024 to 1024, where the rule begins: 14.3, 64: 12.1; 256 pixels, 2048 to 2048: 12.6, 64:
  // 9.3; 17 vectors, 4096 to 4096: 17.4, 64: 10.8.)
  if ((o.N + 127) / 128 * ((o.rows + 127) / 128) >= 256)
    return o.lines ? gemm_tile<T, MAP, true, 128, 128, 64, 64>(in, o, st) : gemm_tile<T, MAP, false, 128, 128, 64, 64>(in, o, st);
  return gemm_tile<T, MAP, false, 64, 64, 32, 32>(in, o, st);
}

// ------------------------------------------------------------------------------------------------
// A few pixels: a block makes 16 NT channels of 16 of them at a time, its waves take the channels of the sum in turn.
// ------------------------------------------------------------------------------------------------
// The matrix is read once; the pixels' codes are made on the way by every block.  4096 to 4096 channels: 7.3 us, four rounds
// of loads, quantisation and products a wave, not the 9 MB (1.7 us); four rounds' loads at once took as long, and twice as long
// for 16 pixels, whose loads past the end cost as much as the others.
template <class T>
__device__ __forceinline__ unsigned mx_quantize_row(const T* x, int64_t step, int n, mx_i32x4* q) {
  float v[kMxBlock];
  unsigned mag = 0;
  if (step == 1 && n == kMxBlock) {
    typedef typename MxVec<T, 16 / sizeof(T)>::type V;
#pragma unroll
    for (int i = 0; i < kMxBlock / (16 / (int)sizeof(T)); ++i) {
      const V t = ((const V*)x)[i];
#pragma unroll
      for (int e = 0; e < 16 / (int)sizeof(T); ++e) v[i * (16 / sizeof(T)) + e] = (float)t[e];
    }
  } else {
#pragma unroll
    for (int c = 0; c < kMxBlock; ++c) v[c] = c < n ? (float)x[c * step] : 0.f;
  }
#pragma unroll
  for (int c = 0; c < kMxBlock; ++c) mag = max(mag, mx_mag(v[c]));
  const unsigned s = mx_scale_code(mag);
  *q = mx_pack32(v, s);
  return s;
}

constexpr int kFewWaves = 8, kFewRows = 16;
template <class T, int NT>
__global__ void __launch_bounds__(kFewWaves * 64) k_mx_few(MxIn in, MxOut o) {
  __shared__ float part[kFewWaves][16 * NT][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16 * NT;
  for (int64_t r0 = (int64_t)blockIdx.y * 16; r0 < o.rows; r0 += (int64_t)gridDim.y * 16) {
    const int64_t r = r0 + j;
    const bool live = r < o.rows;
    const int64_t b = live ? (uint32_t)r / (uint32_t)o.HW : 0, p = r - b * o.HW;
    const T* x = (const T*)in.x + b * in.C * o.HW + p;
    mx_f32x4 acc[NT] = {};
    for (int k = 4 * wave; k < in.KB; k += 4 * kFewWaves) {
      // lane l holds block k + l / 16 of its operands' rows l % 16; past the last both scales are 2^-127
      const bool in_row = k + g < in.KB;
      const int kb = min(k + g, in.KB - 1);
      mx_i32x4 w[NT];
      unsigned sw[NT], sx = 0;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int64_t at = min(n0 + 16 * i + j, o.N - 1) * in.KB + kb;
        w[i] = in.wc[at];
        sw[i] = in.ws[at];
      }
      mx_i32x4 q = {0, 0, 0, 0};
      if (live && in_row) {
        if (in.x) {
          sx = mx_quantize_row(x + (int64_t)kb * kMxBlock * o.HW, o.HW, (int)min((int64_t)kMxBlock, in.C - kb * kMxBlock), &q);
          if (blockIdx.x == 0) {
            in.xc[r * in.KB + kb] = q;
            in.xs[r * in.KB + kb] = (uint8_t)sx;
          }
        } else {
          q = in.xc[r * in.KB + kb];
          sx = in.xs[r * in.KB + kb];
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(w[i]), mx_operand(q), acc[i], kMxFp4, kMxFp4, 0,
                                                                  in_row ? (int)sw[i] : 0, 0, (int)sx);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[wave][16 * i + 4 * g + e][j] = acc[i][e];
    __syncthreads();
    if (threadIdx.x < 256 * NT) {
      // neighbouring threads store neighbours: channels of one pixel a sample, pixels otherwise
      const int a = threadIdx.x & 15, c = threadIdx.x >> 4 & 15, i = threadIdx.x >> 8;
      const int n = 16 * i + (o.HW == 1 ? a : c), k = o.HW == 1 ? c : a;
      const int64_t rk = r0 + k;
      if (rk < o.rows && n0 + n < o.N) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) v += part[w][n][k];
        const int64_t rb = (uint32_t)rk / (uint32_t)o.HW;
        float out[1][1] = {{o.bias ? v + o.bias[n0 + n] : v}};
        const float scale[1][1] = {{o.res_scale ? o.res_scale[n0 + n] : 1.f}};
        mx_finish<1, 1>(o, out, scale);
        mx_store_rows<T, false, 1, 1>(o, (rb * o.N + n0 + n) * o.HW + (rk - rb * o.HW), 0, out);
      }
    }
    __syncthreads();
  }
}

// A parameter's values at the 16 rows of a lane's part of a result: element e of it is row 8 (e / 4) + 4 h + e % 4.
__device__ __forceinline__ mx_f32x16 mx_channels(const float* p, int64_t n0, int h, int64_t N, float none) {
  mx_f32x16 v;
  if (!p) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = none;
  } else if (n0 + 32 <= N) {
    typedef MxVec<float, 4>::type W;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const W w = *(const W*)(p + n0 + 8 * i + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * i + e] = w[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = p[min((uint32_t)n0 + 8 * (e / 4) + 4 * h + e % 4, (uint32_t)N - 1)];
  }
  return v;
}

// ------------------------------------------------------------------------------------------------
// Maps of up to 256 channels: quantised in registers, every product and the store in one pass.
// ------------------------------------------------------------------------------------------------
// Bound by memory.  Lane l of a wave loads the blocks 2 s + l / 32 of two neighbouring pixels (8 bytes of a float32 channel,
// 256 in a row over 32 lanes), makes their codes, and keeps them as operands for every 32 channels of the result: the
// products of pixels 2 j and 2 j + 1 give it two neighbouring pixels of a channel again.  (Four pixels a lane: 128 x 256 x 256
// x 8 float32 to 64 90 us, two 77, half the registers.)  blockIdx.y takes a share of the channels where there are too few
// pixels for the CUs.
template <class T, bool NT, int S>
__global__ void __launch_bounds__(256, 2) k_mx_conv(MxIn in, MxOut o, int share) {
  constexpr int V = 2;
  typedef typename MxVec<T, V>::type W;
  const int lane = threadIdx.x & 63, j = lane & 31, h = lane >> 5;
  const int64_t w0 = ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * (32 * V), r0 = w0 + V * j;
  if (w0 >= o.rows) return;  // (no wave waits for another)
  const MxGroup grp = mx_group<V>(min(r0, o.rows - 1), o.HW, o.rows);
  // Channels are read from the wave's first pixel on, by 32-bit offsets (64-bit ones of 32 channels would fill the
  // registers); lanes whose sample is too far off read one by one, as those whose pixels lie in two samples.
  const int64_t b0 = (uint32_t)w0 / (uint32_t)o.HW, p0 = w0 - b0 * o.HW;
  const int64_t off = ((grp.b - b0) * in.C + (int64_t)h * kMxBlock) * o.HW + grp.p - p0;
  const bool near = grp.whole && off * (int64_t)sizeof(T) < (int64_t)1 << 31;
  const uint32_t lane_off = (uint32_t)(near ? off : 0) * (uint32_t)sizeof(T);
  mx_i32x4 q[S][V];
  unsigned sx[S];  // the scales of the V pixels, a byte each
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int kb = 2 * s + h;
    sx[s] = 0;
    if (kb >= in.KB) {
#pragma unroll
      for (int e = 0; e < V; ++e) q[s][e] = mx_i32x4{0, 0, 0, 0};
      continue;
    }
    const int n = (int)min((int64_t)kMxBlock, in.C - kb * kMxBlock);
    W t[kMxBlock];
    if (near && n == kMxBlock) {
      const char* x = (const char*)((const T*)in.x + (b0 * in.C + 2 * s * kMxBlock) * o.HW + p0);
#pragma unroll
      for (int c = 0; c < kMxBlock; ++c) {
        t[c] = *(const W*)(x + lane_off);
        x += o.HW * (int64_t)sizeof(T);
      }
    } else {
      int64_t b = grp.b, p = grp.p;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const T* x = (const T*)in.x + (b * in.C + kb * kMxBlock) * o.HW + p;
        const int ne = grp.r0 + e < o.rows ? n : 0;
#pragma unroll
        for (int c = 0; c < kMxBlock; ++c) {
          t[c][e] = c < ne ? *x : (T)0.f;
          x += o.HW;
          asm volatile("" : "+v"(x));  // (one address at a time)
        }
        if (++p == o.HW) p = 0, ++b;
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
      const unsigned code = mx_scale_code(mag);
      q[s][e] = mx_pack32(v, code);
      sx[s] |= code << (8 * e);
      if (in.xc && blockIdx.y == 0 && r0 + e < o.rows) {
        in.xc[(r0 + e) * in.KB + kb] = q[s][e];
        in.xs[(r0 + e) * in.KB + kb] = (uint8_t)code;
      }
    }
  }
  const MxPixels<V> pix = mx_pixels<V>(o, grp, 4 * h);
  const int64_t n1 = min(o.N, (int64_t)(blockIdx.y + 1) * share);
  for (int64_t n0 = (int64_t)blockIdx.y * share; n0 < n1; n0 += 32) {
    const int64_t wrow = min(n0 + j, o.N - 1) * in.KB;
    mx_f32x16 acc[V];
    acc[0] = mx_channels(o.bias, n0, h, o.N, 0.f);  // the sums begin with the bias of their rows
#pragma unroll
    for (int e = 1; e < V; ++e) acc[e] = acc[0];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int kb = 2 * s + h, at = min(kb, in.KB - 1);
      const mx_i32x8 w = mx_operand(in.wc[wrow + at]);
      const int sw = kb < in.KB ? in.ws[wrow + at] : 0;
      // (the byte of the scales is part of the instruction)
      acc[0] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, mx_operand(q[s][0]), acc[0], kMxFp4, kMxFp4, 0, sw, 0,
                                                               (int)sx[s]);
      acc[1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, mx_operand(q[s][1]), acc[1], kMxFp4, kMxFp4, 0, sw, 1,
                                                               (int)sx[s]);
    }
    if (r0 >= o.rows) continue;
    const mx_f32x16 ss = mx_channels(o.res_scale, n0, h, o.N, 1.f);
    MxPixels<V> px = pix;
#pragma unroll
    for (int e = 0; e < V; ++e) asm volatile("" : "+v"(px.at[e]));  // (each row's address is made where it is used: kept
                                                                    // over the loop, 64 of them would fill the registers)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = n0 + 8 * i + 4 * h;
      float v[4][V], sc[4][V];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) v[r][e] = acc[e][4 * i + r], sc[r][e] = ss[4 * i + r];
      mx_finish<V, 4>(o, v, sc);
      const int64_t step = (n0 + 8 * i) * o.HW;
      if (grp.whole && n + 4 <= o.N) {
        mx_store_rows<T, NT, V, 4>(o, px.at[0] + step, o.HW, v);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < o.N) mx_store_pixels<T, V>(o, px, step + r * o.HW, v[r]);
      }
    }
  }
}

template <class T, bool NT>
int conv_to(const MxIn& a, const MxOut& o, hipStream_t st) {
  const int64_t tiles = (o.rows + 255) / 256, n32 = (o.N + 31) / 32;
  // as many shares of the channels as give every CU four blocks (160 x 177 x 131 x 4 float32 to 352: 55 us, eight 67)
  const int64_t shares = std::min(n32, std::max<int64_t>(1, 1024 / tiles)), share = (n32 + shares - 1) / shares * 32;
  const dim3 grid((unsigned)tiles, (unsigned)((o.N + share - 1) / share));
  switch ((a.KB + 1) / 2) {
    case 1: hipLaunchKernelGGL((k_mx_conv<T, NT, 1>), grid, dim3(256), 0, st, a, o, (int)share); break;
    case 2: hipLaunchKernelGGL((k_mx_conv<T, NT, 2>), grid, dim3(256), 0, st, a, o, (int)share); break;
    case 3: hipLaunchKernelGGL((k_mx_conv<T, NT, 3>), grid, dim3(256), 0, st, a, o, (int)share); break;
    default: hipLaunchKernelGGL((k_mx_conv<T, NT, 4>), grid, dim3(256), 0, st, a, o, (int)share); break;
  }
  return check_launch("conv1x1_mxfp4");
}

template <class T>
int conv(const MxIn& in, const MxOut& o, bool keep, hipStream_t st) {
  MxIn a = in;
  if (!keep) a.xc = nullptr;
  return o.lines ? conv_to<T, true>(a, o, st) : conv_to<T, false>(a, o, st);
}

int mx_check_product(int64_t B, int64_t C, int64_t HW, int64_t N, int type) {
  if (B < 0 || HW < 0 || C < 1 || N < 1 || !mx_type_size(type)) return fail(CVN_ERR_ARG, "bad shape or type");
  if (C > kMxMaxChannels || N > kMxMaxChannels || (HW && B > kMxMaxRows / HW))
    return fail(CVN_ERR_UNSUPPORTED, "too many channels or pixels");
  return CVN_OK;
}

template <class T>
int product(const MxIn& in, const MxOut& o, int type, bool keep, hipStream_t st) {
  // (the tiled kernel reads scales by words of four)
  if (o.rows <= kFewRows || o.N * in.KB < 4) {
    // Every block reads all of x: two tiles to a block from two blocks a CU on (16 float16 pixels, 2048 to 8192 channels: 7.3 us,
    // one tile 9.0).
    const unsigned y = (unsigned)std::min<int64_t>((o.rows + 15) / 16, 4096);
    if (o.N >= 16 * 512) {
      hipLaunchKernelGGL((k_mx_few<T, 2>), dim3((unsigned)((o.N + 31) / 32), y), dim3(kFewWaves * 64), 0, st, in, o);
    } else {
      hipLaunchKernelGGL((k_mx_few<T, 1>), dim3((unsigned)((o.N + 15) / 16), y), dim3(kFewWaves * 64), 0, st, in, o);
    }
    return check_launch("conv1x1_mxfp4");
  }
  if (in.x && in.KB <= 8 && o.HW > 1) return conv<T>(in, o, keep, st);
  if (in.x) {
    const int q = mx_quantize(in.x, type, o.rows / o.HW, in.C, o.HW, in.xc, in.xs, st);
    if (q != CVN_OK) return q;
  }
  return o.HW == 1 ? gemm<T, false>(in, o, st) : gemm<T, true>(in, o, st);
}

}  // namespace
}  // namespace cvn

using namespace cvn;

extern "C" size_t cvn_conv1x1_mxfp4_workspace(int x_given, int w_given, int64_t B, int64_t C, int64_t HW, int64_t N) {
  if (mx_check_product(B, C, HW, N, CVN_F32) != CVN_OK) return 0;
  return (x_given ? 0 : align_up((size_t)(B * HW * mx_blocks(C)) * 17)) + (w_given ? 0 : align_up((size_t)(N * mx_blocks(C)) * 17));
}

extern "C" int cvn_conv1x1_mxfp4(const void* x, void* x_codes, void* x_scales, int64_t B, int64_t C, int64_t HW, const void* w,
                                 int w_type, void* w_codes, void* w_scales, int64_t N, const float* bias, int act,
                                 const void* residual, const float* res_scale, void* y, int type, void* workspace,
                                 size_t workspace_bytes, cvn_stream_t stream) {
  const int rc = mx_check_product(B, C, HW, N, type);
  if (rc != CVN_OK) return rc;
  if (act != CVN_ACT_NONE && act != CVN_ACT_GELU) return fail(CVN_ERR_ARG, "unknown activation");
  if (w && !mx_type_size(w_type)) return fail(CVN_ERR_ARG, "bad type of the matrix");
  const int64_t rows = B * HW, KB = mx_blocks(C), es = mx_type_size(type);
  if (!x_codes != !x_scales || !w_codes != !w_scales || (!w && !w_codes) || (rows && (!y || (!x && !x_codes))))
    return fail(CVN_ERR_ARG, "null pointer");
  if (((uintptr_t)w_codes | (uintptr_t)x_codes) & 15) return fail(CVN_ERR_ARG, "codes must be aligned to 16 bytes");
  // What is written is apart from all else, but y may be the residual.
  const MxMem mem[] = {{y, rows * N * es},
                       {x ? x_codes : nullptr, rows * KB * 16},
                       {x ? x_scales : nullptr, rows * KB},
                       {w ? w_codes : nullptr, N * KB * 16},
                       {w ? w_scales : nullptr, N * KB},  // written up to here
                       {x, rows * C * es},
                       {w, w ? N * C * mx_type_size(w_type) : 0},
                       {x ? nullptr : x_codes, rows * KB * 16},
                       {x ? nullptr : x_scales, rows * KB},
                       {w ? nullptr : w_codes, N * KB * 16},
                       {w ? nullptr : w_scales, N * KB},
                       {residual == y ? nullptr : residual, rows * N * es},
                       {bias, N * 4},
                       {res_scale, N * 4}};
  if (mx_shared(mem, 5, 14)) return fail(CVN_ERR_ARG, "an output shares memory with an input or another output");
  const bool keep = x_codes != nullptr;
  const size_t need = cvn_conv1x1_mxfp4_workspace(keep, w_codes != nullptr, B, C, HW, N);
  if (need && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))
    return fail(CVN_ERR_WORKSPACE, "workspace missing, too small or not aligned to 16 bytes");
  char* work = (char*)workspace;
  const hipStream_t st = (hipStream_t)stream;
  if (!w_codes) {
    w_codes = work;
    w_scales = work + N * KB * 16;
    work += align_up((size_t)(N * KB) * 17);
  }
  if (w) {
    const int q = mx_quantize(w, w_type, N, C, 1, w_codes, w_scales, st);
    if (q != CVN_OK) return q;
  }
  if (rows == 0) return CVN_OK;
  if (!keep) {
    x_codes = work;
    x_scales = work + rows * KB * 16;
  }
  const MxIn in = {x, (mx_i32x4*)x_codes, (uint8_t*)x_scales, (const mx_i32x4*)w_codes, (const uint8_t*)w_scales, C, (int)KB};
  const bool lines = (((HW > 1 ? HW : N) * es) | (int64_t)(uintptr_t)y) % 128 == 0;
  const MxOut o = {bias, res_scale, residual, y, HW, N, rows, act, lines};
  if (type == CVN_F32) return product<float>(in, o, type, keep, st);
  if (type == CVN_BF16) return product<__bf16>(in, o, type, keep, st);
  return product<_Float16>(in, o, type, keep, st);
}
