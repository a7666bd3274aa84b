// pclseg_i8.h — the 8-bit linear layer: rows of activations quantised symmetrically with one scale per row, an int8 x int8
// product on the matrix cores with exact int32 sums, one scale per output channel, and the epilogue of op_conv2d.
//
//   s[i] = max_k |x[i,k]| / 127,  q[i,k] = round(x[i,k] / s[i]) (ties to even, within +-127; 0 where s[i] is 0)
//   y[i,j] = act( s[i] t[j] sum_k q[i,k] w[j,k] + bias[j] ) + residual[i,j]
//
// Codes lie in rows of `ld` bytes, a multiple of 64 (of 128 for k > 64) and zero behind k: every tile is read whole, without
// a test for the end of a row.  |q w| <= 128 * 128 and k <= 131071 keep the int32 sums exact; they are rounded to float32
// once, and once more by each product of the epilogue.
#ifndef PCLSEG_I8_H_
#define PCLSEG_I8_H_

#include "pclseg_rows.h"

namespace pclseg {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------------------------------------- quantisation
struct QuantArgs {
  const void* x;
  int64_t rows, stride;
  int cols;
  int8_t* q;
  int64_t ld;
  float* scale;
};

// The largest magnitude of a row is taken on the bits: without the sign they order like unsigned integers, infinities and
// NaN above everything finite, and 16-bit elements go two to an instruction.
template <typename T> struct RowMax {
  typedef uint16_t U2 __attribute__((ext_vector_type(2)));
  U2 m{0, 0};
  static constexpr uint32_t kInf = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
  __device__ __forceinline__ void add(const u32x4& v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(U2, v[e] & 0x7fff7fffu));
  }
  __device__ __forceinline__ uint32_t bits() const { return m[0] > m[1] ? m[0] : m[1]; }
  static __device__ __forceinline__ float value(uint32_t b) {
    return Elem<T>::get(u32x4{b, 0u, 0u, 0u}, 0);
  }
};
template <> struct RowMax<float> {
  uint32_t m = 0;
  static constexpr uint32_t kInf = 0x7f800000u;
  __device__ __forceinline__ void add(const u32x4& v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) m = max(m, v[e] & 0x7fffffffu);
  }
  __device__ __forceinline__ uint32_t bits() const { return m; }
  static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b); }
};

// Rows below 2^-60 are scaled by 2^64 (pre), so that s and 1 / s stay normal numbers.
struct RowScale { float pre, s, inv, half; };
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.pre = amax < 0x1p-60f ? 0x1p64f : 1.f;
  // amax / 127, rounded once: the quotient by the rounded reciprocal, corrected by its exact remainder (equal to the IEEE
  // division for every mantissa)
  constexpr float c = 1.f / 127.f;
  const float a = amax * r.pre, q = a * c;
  r.s = fmaf(fmaf(-127.f, q, a), c, q);
  if (r.pre != 1.f && r.s < 0x1p-62f) {
    // the scale that is stored is s 2^-64, a subnormal number: the codes belong to what it is rounded to.  That takes two
    // roundings, of which the exact remainder against 63.5 units says whether the second went the wrong way (a is a whole
    // number of units, so there are no ties)
    constexpr float unit = 0x1p-85f;
    r.s = (r.s * 0x1p-64f) * 0x1p64f;
    const float rest = fmaf(-127.f, r.s, a);
    r.s += rest > 63.5f * unit ? unit : rest < -63.5f * unit ? -unit : 0.f;
  }
  r.inv = r.s > 0.f ? __builtin_amdgcn_rcpf(r.s) : 0.f;      // one unit off: 2^-16 of a step in a code's quotient
  r.half = 0.5f * r.s;
  return r;
}
constexpr float kRound = 12582912.f;      // 1.5 * 2^23: x + kRound rounds x to an integer, whose code is the sum's low byte
// The code of x has to be the integer nearest to the exact quotient x / s.  u = x * (1/s) + kRound, one fma, holds the nearest
// integer or, within 2^-16 of a half step, its neighbour; the remainder t = x - q s, exact in one fma, says which: below half
// a step the code stands, otherwise (rare: one of 2^16 elements) `nearest` decides.
__device__ __forceinline__ float quant(float x, const RowScale& r, float& worst) {
  const float u = fmaf(x, r.inv, kRound), t = fmaf(-(u - kRound), r.s, x);
  worst = fmaxf(worst, fabsf(t));
  return u;
}
__device__ __forceinline__ float nearest(float x, const RowScale& r) {
  const float u = fmaf(x, r.inv, kRound), q = u - kRound, t = fmaf(-q, r.s, x), m = fabsf(t);
  const bool odd = __float_as_uint(u) & 1;
  return m > r.half || (m == r.half && odd) ? u + (t > 0.f ? 1.f : -1.f) : u;
}
__device__ __forceinline__ uint32_t pack4(const float* u) {
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(u[1]), __float_as_uint(u[0]), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(u[3]), __float_as_uint(u[2]), 0x04000c0cu);
  return lo | hi;
}

// eight elements of a row: 16 bytes, or 32 of floats
template <typename T> struct Eight {
  static constexpr int N = 8 / Elem<T>::VEC;
  u32x4 v[N];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int h = 0; h < N; ++h) v[h] = load16(p + h * Elem<T>::VEC);
  }
  // elements [c, c + 8) of a row in two steps, so that all of a lane's loads are in flight before the first is waited for:
  // request() reads 16 or 32 bytes inside the row whatever c is, settle() puts 0 behind the row's end
  __device__ __forceinline__ void request(const T* row, int c, int cols) {
    if (cols >= 8) load(row + (c + 8 <= cols ? c : 0));
  }
  __device__ __forceinline__ void settle(const T* row, int c, int cols) {
    if (c + 8 > cols) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
      if (c < cols) {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (c + e < cols) f[e] = Elem<T>::load(row + c + e);
      }
#pragma unroll
      for (int h = 0; h < N; ++h) v[h] = pack16<T>(f + h * Elem<T>::VEC);
    }
  }
  __device__ __forceinline__ void load(const T* row, int c, int cols) {
    request(row, c, cols);
    settle(row, c, cols);
  }
  __device__ __forceinline__ void add_to(RowMax<T>& m) const {
#pragma unroll
    for (int h = 0; h < N; ++h) m.add(v[h]);
  }
  __device__ __forceinline__ u32x2 codes(const RowScale& r) const {
    float x[8], u[8], worst = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elem<T>::get(v[e / Elem<T>::VEC], e % Elem<T>::VEC);
    if (r.pre != 1.f) {
      const float most = 127.f * r.s;      // a rounded subnormal scale may be short of the row: 127 is the last code
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fminf(fmaxf(x[e] * r.pre, -most), most);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = quant(x[e], r, worst);
    if (worst >= r.half) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = nearest(x[e], r);
    }
    return u32x2{pack4(u), pack4(u + 4)};
  }
};

// Bound by memory: 8192 x 4096 bf16 in 16.4 us, 131072 x 512 float32 in 56 us (one call after the other; 6.1 and 6.0 TB/s of
// what is read and written).
// G lanes own a row, each 8 elements of every stretch of 8 G; four stretches are kept in registers, so a row of up to 32 G
// elements is read once.  Longer rows (REREAD) are read twice, the second time from the L2.  A row with an infinity or a
// NaN gets the scale NaN and codes 0: its outputs are NaN, like those of a float32 product.
template <typename T, int G, bool REREAD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
  constexpr int NV = 4;
  __shared__ uint32_t red[4];
  const int g = threadIdx.x % G;
  const int64_t row0 = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = row0 < a.rows;
  const int64_t row = live ? row0 : a.rows - 1;
  const T* src = static_cast<const T*>(a.x) + row * a.stride;
  const int nv = (a.cols + 8 * G - 1) / (8 * G);
  Eight<T> x[NV];
  RowMax<T> mx;
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (v < nv) x[v].request(src, (v * G + g) * 8, a.cols);
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (v < nv) x[v].settle(src, (v * G + g) * 8, a.cols);
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (v < nv) x[v].add_to(mx);
  if constexpr (REREAD) {
    for (int v = NV; v < nv; ++v) {
      Eight<T> t;
      t.load(src, (v * G + g) * 8, a.cols);
      t.add_to(mx);
    }
  }
  uint32_t top = mx.bits();
  top = group_reduce<(G < 64 ? G : 64)>(top, [](uint32_t a, uint32_t b) { return max(a, b); });
  if constexpr (G == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(red[0], red[1]), max(red[2], red[3]));
  }
  const bool finite = top < RowMax<T>::kInf;
  const RowScale r = row_scale(finite ? RowMax<T>::value(top) : 0.f);
  if (!live) return;
  if (g == 0) a.scale[row] = finite ? r.s / r.pre : __builtin_nanf("");
  const bool zero = r.inv == 0.f;      // nothing but zeros, or no scale
  int8_t* dst = a.q + row * a.ld;
  const int nq = (int)((a.ld + 8 * G - 1) / (8 * G));      // the zeros behind the row too
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * G + g) * 8;
    if (v < nv && c < a.ld) *reinterpret_cast<u32x2*>(dst + c) = zero ? u32x2{0u, 0u} : x[v].codes(r);
  }
  for (int v = nv < NV ? nv : NV; v < nq; ++v) {
    const int c = (v * G + g) * 8;
    if (c >= a.ld) break;
    u32x2 w{0u, 0u};
    if (REREAD && c < a.cols && !zero) {
      Eight<T> t;
      t.load(src, c, a.cols);
      w = t.codes(r);
    }
    *reinterpret_cast<u32x2*>(dst + c) = w;
  }
}

// ---------------------------------------------------------------------------------------------- product
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_LEAKY = 2, ACT_SIGMOID = 3 };

struct I8Args {
  const int8_t *a, *b;        // codes of the rows [m, lda] and of the channels [n, ldb]
  const float *sa, *sb;       // scales
  int64_t lda, ldb;
  int64_t m;
  int n, kp;                  // kp: k rounded up to whole steps (<= lda, ldb)
  const float* bias;          // NULL: none
  int act;
  const void* residual;       // NULL: none
  int64_t ldr;
  void* y;
  int64_t ldy;
};

__device__ __forceinline__ float relu(float v) { return v > 0.f ? v : (v != v ? v : 0.f); }
__device__ __forceinline__ float leaky(float v) { return v > 0.f ? v : 0.1f * v; }
// v_exp_f32 and v_rcp_f32, one unit in the last place each: within 4 * 2^-24 of the sigmoid, whose slope is 1/4.  Far below 0 the
// error is |v| 2^-24 of the value, by the rounding of the exponent
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}
__device__ __forceinline__ float activate(float v, int act) {
  return act == ACT_RELU ? relu(v) : act == ACT_LEAKY ? leaky(v) : act == ACT_SIGMOID ? sigmoid(v) : v;
}

// acc sa sb + bias.  Below 2^64 a row's scale takes the sum nowhere near the end of float32 (2^31 2^64); from there on the
// channel's scale goes first, and what overflows then does so in the product of all three.  Whole multiples of a subnormal scale
// are exact, so neither order loses bits below.
constexpr float kFarScale = 0x1p64f;
__device__ __forceinline__ float scaled(float acc, float sa, float sb, float bias) {
  const bool far = sa >= kFarScale;
  return fmaf(acc * (far ? sb : sa), far ? sa : sb, bias);
}

template <typename T>
__device__ __forceinline__ void i8_store(const I8Args& p, int64_t i, int j, int acc, float sa, float sb, float bias) {
  float v = activate(scaled((float)acc, sa, sb, bias), p.act);
  if (p.residual) v += Elem<T>::load(static_cast<const T*>(p.residual) + i * p.ldr + j);
  static_cast<T*>(p.y)[i * p.ldy + j] = Elem<T>::from(v);
}

// ---- few rows: the weights are read once, straight into the matrix operands
// A block owns 16 channels and all of k; its NW waves take stretches of k (64 bytes of 16 weight rows an instruction, four
// instructions in flight) and add their partial sums through LDS.  MT tiles of 16 rows share every weight fragment.  The
// same kernel, with more rows in the grid's second axis, serves outputs of few tiles: k is split over the waves of a block
// instead of one block walking all of it (80 x 146 x 3606: 14 us in six 64x64 tiles, 4 in 50 blocks).
template <typename T, int MT, int NW>
__global__ __launch_bounds__(NW * 64) void i8_few_rows(I8Args p) {
  __shared__ int part[NW][MT][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, ko = (lane >> 4) * 16;
  const int n0 = blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const int jn = n0 + r < p.n ? n0 + r : p.n - 1;
  const int8_t* wb = p.b + (int64_t)jn * p.ldb + ko;
  const int8_t* xa[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t i = m0 + t * 16 + r;
    xa[t] = p.a + (i < p.m ? i : p.m - 1) * p.lda + ko;
  }
  i32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = i32x4{0, 0, 0, 0};
  const int steps = p.kp / 64;
  int s = wave * 4;
  for (; s + 4 <= steps; s += NW * 4) {
    i32x4 w[4], x[MT][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = *reinterpret_cast<const i32x4*>(wb + (int64_t)(s + u) * 64);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < 4; ++u) x[t][u] = *reinterpret_cast<const i32x4*>(xa[t] + (int64_t)(s + u) * 64);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[t][u], w[u], acc[t], 0, 0, 0);
  }
  for (int e = s; e < steps && e < s + 4; ++e) {
    const i32x4 w = *reinterpret_cast<const i32x4*>(wb + (int64_t)e * 64);
#pragma unroll
    for (int t = 0; t < MT; ++t)
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4*>(xa[t] + (int64_t)e * 64), w, acc[t], 0, 0, 0);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][t][((lane >> 4) * 4 + i) * 16 + r] = acc[t][i];
  __syncthreads();
  for (int o = threadIdx.x; o < MT * 256; o += NW * 64) {
    const int64_t i = m0 + o / 16;
    const int j = n0 + (o & 15);
    if (i >= p.m || j >= p.n) continue;
    int v = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += part[w][o >> 8][o & 255];
    i8_store<T>(p, i, j, v, p.sa[i], p.sb[j], p.bias ? p.bias[j] : 0.f);
  }
}

// ---- up to 32 short rows: quantisation and product in one launch
// Every block quantises all rows again (from the L2), where a launch and a workspace of their own cost 3.5 us of a pass.
// Its first weights are requested before the rows; loads come back in order, so the maximum waits for both and the weights are
// there when the codes are.  The rows are cut into items of 512 elements, eight a lane; a wave takes
// up to eight items and holds them in registers between the maximum and the codes.  Codes and scales stay in LDS.  MT tiles
// of 16 rows share a weight fragment.
constexpr int kFusedRows = 32, kFusedItems = 64;
template <typename T, typename Y, int MT>
__global__ __launch_bounds__(512) void i8_fused_rows(I8Args p, const T* x, int64_t x_stride, int k) {
  constexpr int NW = 8, D = 8;
  extern __shared__ __attribute__((aligned(16))) int8_t codes[];      // [m][kp]
  __shared__ int part[NW][MT][256];
  __shared__ uint32_t tops[16 * MT];
  __shared__ float scales[16 * MT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, ko = (lane >> 4) * 16;
  const int n0 = blockIdx.x * 16, m = (int)p.m;
  const int jn = n0 + r < p.n ? n0 + r : p.n - 1;
  const int steps = p.kp / 64, s0 = steps * wave / NW, s1 = steps * (wave + 1) / NW;      // a wave's stretch of k
  const int8_t* wb = p.b + (int64_t)jn * p.ldb + ko;
  i32x4 w[D];
#pragma unroll
  for (int u = 0; u < D; ++u) w[u] = *reinterpret_cast<const i32x4*>(wb + (int64_t)(s0 + u < s1 ? s0 + u : steps - 1) * 64);
  constexpr int IW = kFusedItems / NW;
  const int cuts = (p.kp + 511) / 512, items = m * cuts;
  Eight<T> e[IW];
#pragma unroll
  for (int h = 0; h < IW; ++h) {
    const int it = h * NW + wave, row = it / cuts;
    if (it < items) e[h].request(x + row * x_stride, (it - row * cuts) * 512 + lane * 8, k);
  }
  if ((int)threadIdx.x < m) tops[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int h = 0; h < IW; ++h) {
    const int it = h * NW + wave, row = it / cuts;
    if (it < items) {
      e[h].settle(x + row * x_stride, (it - row * cuts) * 512 + lane * 8, k);
      RowMax<T> mx;
      e[h].add_to(mx);
      const uint32_t top = group_reduce<64>(mx.bits(), [](uint32_t a, uint32_t b) { return max(a, b); });
      if (lane == 0) atomicMax(&tops[row], top);
    }
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < IW; ++h) {
    const int it = h * NW + wave, row = it / cuts, c = (it - row * cuts) * 512 + lane * 8;
    if (it < items) {
      const uint32_t top = tops[row];
      const bool finite = top < RowMax<T>::kInf;
      const RowScale q = row_scale(finite ? RowMax<T>::value(top) : 0.f);
      if (c == 0) scales[row] = finite ? q.s / q.pre : __builtin_nanf("");
      if (c < p.kp) *reinterpret_cast<u32x2*>(codes + row * p.kp + c) = q.inv != 0.f ? e[h].codes(q) : u32x2{0u, 0u};
    }
  }
  __syncthreads();
  i32x4 acc[MT];
  const int8_t* xa[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    acc[t] = i32x4{0, 0, 0, 0};
    xa[t] = codes + (t * 16 + r < m ? t * 16 + r : 0) * p.kp + ko;      // rows behind m are not stored
  }
  for (int s = s0; s < s1; s += D) {
#pragma unroll
    for (int u = 0; u < D; ++u) {
      if (s + u < s1) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
          acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const i32x4*>(xa[t] + (s + u) * 64), w[u], acc[t], 0, 0, 0);
        if (s + u + D < s1) w[u] = *reinterpret_cast<const i32x4*>(wb + (int64_t)(s + u + D) * 64);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][t][((lane >> 4) * 4 + i) * 16 + r] = acc[t][i];
  __syncthreads();
  for (int o = threadIdx.x; o < m * 16; o += NW * 64) {
    const int i = o / 16, j = n0 + (o & 15);
    if (j >= p.n) continue;
    int v = 0;
#pragma unroll
    for (int u = 0; u < NW; ++u) v += part[u][o >> 8][o & 255];
    i8_store<Y>(p, i, j, v, scales[i], p.sb[j], p.bias ? p.bias[j] : 0.f);
  }
}

// ---- tiles
// BM x BN outputs a block, BK bytes of k a step, WM x WN waves.  Both operands go straight from memory into LDS (16 bytes a
// lane, no registers between), two buffers: the next step's tile is in flight while this one is multiplied.  A row of a tile
// is BK bytes; its 16-byte chunks are permuted by the row number, so that the 16 lanes an LDS read serves at once, the same
// chunk of 16 rows, lie in 16 different places of the 64 banks (256 bytes hold 256 / BK rows, hence the shift; with rows
// permuted by row % 8, counters showed every second cycle of the LDS lost to conflicts).  The permutation is made on the
// global side: LDS is written linearly.
template <int BK>
__device__ __forceinline__ int swizzle(int row) { return (row * BK / 256) & (BK / 16 - 1); }
template <int BK>
__device__ __forceinline__ int lds_chunk(int row, int chunk) { return row * BK + (chunk ^ swizzle<BK>(row)) * 16; }

// Where a thread's 16-byte pieces of a tile of ROWS rows come from: offsets from the tile's first byte, fixed for all steps.
template <int ROWS, int BK, int THREADS>
struct TileSource {
  static constexpr int C = BK / 16, N = ROWS * C / THREADS;
  static_assert(ROWS * C % THREADS == 0, "whole waves");
  const int8_t* base;      // uniform
  uint32_t off[N];
  __device__ __forceinline__ TileSource(const int8_t* src, int64_t ld, int64_t row0, int64_t rows) : base(src + row0 * ld) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int pos = i * THREADS + threadIdx.x;
      const int r = pos / C, ch = (pos % C) ^ swizzle<BK>(r);
      const int rr = row0 + r < rows ? r : (int)(rows - 1 - row0);       // rows behind the last repeat it
      off[i] = (uint32_t)rr * (uint32_t)ld + ch * 16;
    }
  }
  __device__ __forceinline__ void stage(int64_t k0, int8_t* lds, int wave) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(base + k0 + off[i]),
                                       (__attribute__((address_space(3))) void*)(lds + (i * THREADS + wave * 64) * 16), 16, 0, 0);
  }
};

// four neighbouring outputs of a row
template <typename T> struct Quad;
template <> struct Quad<float> {
  static __device__ __forceinline__ void load(const float* p, float* f) {
    const u32x4 v = load16(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(v[e]);
  }
  static __device__ __forceinline__ void store(float* p, const float* f) { stream16(p, pack16<float>(f)); }
};
template <typename T> struct Quad16 {
  static __device__ __forceinline__ void load(const T* p, float* f) {
    const u32x2 v = *reinterpret_cast<const u32x2a2*>(p);
    const u32x4 w{v[0], v[1], 0u, 0u};
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = Elem<T>::get(w, e);
  }
  static __device__ __forceinline__ void store(T* p, const float* f) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    typedef float F2 __attribute__((ext_vector_type(2)));
    u32x2 v;
#pragma unroll
    for (int e = 0; e < 2; ++e) v[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(F2{f[2 * e], f[2 * e + 1]}, T2));
    __builtin_nontemporal_store((u32x2a2)v, reinterpret_cast<u32x2a2*>(p));
  }
};
template <> struct Quad<__bf16> : Quad16<__bf16> {};
template <> struct Quad<_Float16> : Quad16<_Float16> {};

// act is uniform: one scalar branch for all values
template <int N> __device__ __forceinline__ void activate_all(float* v, int act) {
  if (act == ACT_RELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = relu(v[e]);
  } else if (act == ACT_LEAKY) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = leaky(v[e]);
  } else if (act == ACT_SIGMOID) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = sigmoid(v[e]);
  }
}

// Measured (the product alone, one call after the other): 8192x4096 -> 8192 bf16 235 us (2.3 PFLOP/s; 271 under a profiler, where the
// matrix pipes were busy 59 % of the time at the 1.8 GHz that the power limit leaves), 131072x512 -> 1024 float32 138 us (4.4 TB/s),
// 8192x1024 -> 512 float32 with residual 10.2 us.
// The loop: a step's fragments are read from LDS one 32-byte slice of k ahead of the matrix instructions that use them, and
// the barrier that hands a buffer over lies before the step's last slice, whose fragments are already in registers: the first
// reads of the next tile run under those matrix instructions.
// The epilogue goes through LDS, 32 rows of a wave at a time in a slab of its own: the weights are the matrix instruction's
// first operand, so a lane's accumulators are four neighbouring channels of one row, and memory wants whole 128-byte lines
// of a row.  Tiles inside the output take a path without a test; loads (scales, residual) are in flight before the slab is
// written.  (With one tested, branching store after the other the epilogue alone took 155 us of 134 M outputs.)
template <typename T, int BM, int BN, int BK, int WM, int WN, int OCC>
__global__ __launch_bounds__(WM * WN * 64, OCC) void i8_tiles(I8Args p, unsigned tiles_m, unsigned tiles_n) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;      // 32x32 tiles of a wave
  constexpr int KK = BK / 32, TILE = (BM + BN) * BK;
  static_assert(KK % 2 == 0, "slices alternate between two sets of registers");
  constexpr int SW = TN * 32, SLD = SW + 4;                // slab: 32 rows of SW floats; + 4: 16 rows' quads fill 64 banks
  constexpr int SLABS = WM * WN * 32 * SLD * 4;
  __shared__ __attribute__((aligned(128))) int8_t lds[2 * TILE > SLABS ? 2 * TILE : SLABS];
  // an XCD works on neighbouring tiles, taken from groups of 4 tile rows column by column: 32 blocks of an XCD share 4 tiles
  // of a and 8 of b
  const unsigned id = xcd_contiguous(blockIdx.x, gridDim.x);
  const unsigned group = id / (4 * tiles_n), in_group = id - group * 4 * tiles_n;
  const unsigned gm = tiles_m - group * 4 < 4 ? tiles_m - group * 4 : 4;
  const int64_t m0 = (int64_t)(group * 4 + in_group % gm) * BM;
  const int n0 = (int)(in_group / gm) * BN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  i32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  const int steps = p.kp / BK;
  const TileSource<BM, BK, THREADS> sa(p.a, p.lda, m0, p.m);
  const TileSource<BN, BK, THREADS> sb(p.b, p.ldb, n0, p.n);
  i32x4 fa[2][TM], fb[2][TN];
  auto fragments = [&](int buf, int kk, int slot) {
    const int8_t* la = lds + buf * TILE;
    const int8_t* lb = la + BM * BK;
    const int ch = kk * 2 + (lane >> 5), r = lane & 31;
#pragma unroll
    for (int i = 0; i < TM; ++i) fa[slot][i] = *reinterpret_cast<const i32x4*>(la + lds_chunk<BK>(wm + i * 32 + r, ch));
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[slot][j] = *reinterpret_cast<const i32x4*>(lb + lds_chunk<BK>(wn + j * 32 + r, ch));
  };
  auto multiply = [&](int slot) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[slot][j], fa[slot][i], acc[i][j], 0, 0, 0);
  };
  auto interleave = [&]() {      // the slice's LDS reads spread over its matrix instructions, and nothing moved out of the slice
#pragma unroll
    for (int i = 0; i < TM * TN; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      constexpr int each = (TM + TN + TM * TN - 1) / (TM * TN);
      if (i * each < TM + TN) __builtin_amdgcn_sched_group_barrier(0x100, each, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  sa.stage(0, lds, wave);
  sb.stage(0, lds + BM * BK, wave);
  __syncthreads();
  if (steps > 1) {
    sa.stage(BK, lds + TILE, wave);
    sb.stage(BK, lds + TILE + BM * BK, wave);
  }
  fragments(0, 0, 0);
  for (int s = 0; s + 1 < steps; ++s) {
#pragma unroll
    for (int kk = 0; kk + 1 < KK; ++kk) {
      fragments(s & 1, kk + 1, (kk + 1) & 1);
      multiply(kk & 1);
      interleave();
    }
    __syncthreads();      // the next tile has landed, this one is read no more
    if (s + 2 < steps) {
      sa.stage((int64_t)(s + 2) * BK, lds + (s & 1) * TILE, wave);
      sb.stage((int64_t)(s + 2) * BK, lds + (s & 1) * TILE + BM * BK, wave);
    }
    fragments((s + 1) & 1, 0, 0);
    multiply((KK - 1) & 1);
    interleave();
  }
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    if (kk + 1 < KK) fragments((steps - 1) & 1, kk + 1, (kk + 1) & 1);
    multiply(kk & 1);
  }
  __syncthreads();      // the tiles are read no more: the waves' slabs take their place
  float* slab = reinterpret_cast<float*>(lds) + wave * 32 * SLD;
  constexpr int QR = SW / 4, RP = 64 / QR, NR = 32 / RP;       // lanes a row, rows a pass, passes
  const int qc = (lane % QR) * 4, qr = lane / QR;
  const int col = n0 + wn + qc;
  float scale[4], bias[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    scale[e] = col + e < p.n ? p.sb[col + e] : 0.f;
    bias[e] = p.bias && col + e < p.n ? p.bias[col + e] : 0.f;
  }
  auto to_slab = [&](int i) {
    wave_lds_fence();
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = __float_as_uint((float)acc[i][j][q * 4 + e]);
        *reinterpret_cast<u32x4*>(slab + (lane & 31) * SLD + j * 32 + q * 8 + (lane >> 5) * 4) = w;
      }
    wave_lds_fence();
  };
  if (m0 + BM <= p.m && n0 + BN <= p.n && p.ldy < (1 << 26) && p.ldr < (1 << 26)) {
    // uniform row addresses plus a lane's 32-bit offset; four passes at a time bound the registers
    const uint32_t yo = (uint32_t)(qr * (int)p.ldy + qc) * sizeof(T), ro = (uint32_t)(qr * (int)p.ldr + qc) * sizeof(T);
    constexpr int HR = NR < 4 ? NR : 4;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      to_slab(i);
#pragma unroll
      for (int h = 0; h < NR; h += HR) {
        const int64_t row0 = m0 + wm + i * 32 + h * RP;
        const char* rb = static_cast<const char*>(p.residual) + (row0 * p.ldr + n0 + wn) * (int64_t)sizeof(T);
        char* yb = static_cast<char*>(p.y) + (row0 * p.ldy + n0 + wn) * (int64_t)sizeof(T);
        float s[HR], res[HR][4], v[HR][4];
        if (p.residual) {
#pragma unroll
          for (int r = 0; r < HR; ++r)
            Quad<T>::load(reinterpret_cast<const T*>(rb + r * RP * p.ldr * (int64_t)sizeof(T) + ro), res[r]);
        }
#pragma unroll
        for (int r = 0; r < HR; ++r) s[r] = (p.sa + row0 + r * RP)[qr];
        float most = s[0];
#pragma unroll
        for (int r = 1; r < HR; ++r) most = fmaxf(most, s[r]);
        const bool far = __ballot(most >= kFarScale) != 0;      // uniform: the selects cost nothing where no row needs them
#pragma unroll
        for (int r = 0; r < HR; ++r) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(slab + ((h + r) * RP + qr) * SLD + qc);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[r][e] = __uint_as_float(w[e]);
        }
        if (__builtin_expect(far, 0)) {
#pragma unroll
          for (int r = 0; r < HR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[r][e] = scaled(v[r][e], s[r], scale[e], bias[e]);
        } else {
#pragma unroll
          for (int r = 0; r < HR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[r][e] = fmaf(v[r][e] * s[r], scale[e], bias[e]);
        }
        activate_all<HR * 4>(&v[0][0], p.act);
        if (p.residual) {
#pragma unroll
          for (int r = 0; r < HR; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[r][e] += res[r][e];
        }
#pragma unroll
        for (int r = 0; r < HR; ++r) Quad<T>::store(reinterpret_cast<T*>(yb + r * RP * p.ldy * (int64_t)sizeof(T) + yo), v[r]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return;
  }
  // a tile at an edge: the same with a test a quad; a quad cut by the last channel goes element by element
  const bool quad = col + 4 <= p.n, cut = col < p.n && !quad;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    to_slab(i);
#pragma unroll 4
    for (int r = qr; r < 32; r += RP) {
      const int64_t row = m0 + wm + i * 32 + r;
      const bool live = row < p.m;
      const float s = p.sa[live ? row : p.m - 1];
      const u32x4 w = *reinterpret_cast<const u32x4*>(slab + r * SLD + qc);
      float v[4], res[4] = {0.f, 0.f, 0.f, 0.f};
      if (p.residual && quad && live) Quad<T>::load(static_cast<const T*>(p.residual) + row * p.ldr + col, res);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = scaled(__uint_as_float(w[e]), s, scale[e], bias[e]);
      activate_all<4>(v, p.act);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += res[e];
      if (quad && live) Quad<T>::store(static_cast<T*>(p.y) + row * p.ldy + col, v);
      if (cut && live) {
#pragma unroll
        for (int e = 0; e < 3; ++e) {
          if (col + e < p.n) {
            if (p.residual) v[e] += Elem<T>::load(static_cast<const T*>(p.residual) + row * p.ldr + col + e);
            static_cast<T*>(p.y)[row * p.ldy + col + e] = Elem<T>::from(v[e]);
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

}  // namespace pclseg

#endif  // PCLSEG_I8_H_
