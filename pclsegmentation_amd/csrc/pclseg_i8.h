// pclseg_i8.h — the 8-bit linear layer: rows of activations quantised symmetrically with one scale per row, an int8 x int8
// product on the matrix cores with exact int32 sums, one scale per output channel, and the epilogue of op_conv2d.
//
//   s[i] = max_k |x[i,k]| / 127,  q[i,k] = round(x[i,k] / s[i]) (ties to even)
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

// A row's code needs round(x / s) to be the nearest integer of the exact quotient: x * (1/s) is within two roundings of it,
// so rint() of that is the nearest integer or its neighbour, and the remainder x - q s — exact in one fma, |q| <= 128 —
// says which.  Rows below 2^-60 are scaled by 2^64 first, so that s and 1/s stay normal numbers.
struct RowScale { float pre, s, inv, half; };
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.pre = amax < 0x1p-60f ? 0x1p64f : 1.f;
  r.s = amax * r.pre / 127.f;
  r.inv = r.s > 0.f ? 1.f / r.s : 0.f;
  r.half = 0.5f * r.s;
  return r;
}
__device__ __forceinline__ int quant(float x, const RowScale& r) {
  const float v = x * r.pre;
  float q = rintf(v * r.inv);
  const float t = fmaf(-q, r.s, v), m = fabsf(t);
  const bool odd = ((int)q & 1) != 0;
  if (m > r.half || (m == r.half && odd)) q += t > 0.f ? 1.f : -1.f;
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return (uint32_t)(a & 0xff) | ((uint32_t)(b & 0xff) << 8) | ((uint32_t)(c & 0xff) << 16) | ((uint32_t)(d & 0xff) << 24);
}

// elements [c, c + 8) of a row, 0 behind its end
template <typename T> __device__ __forceinline__ void load8_zero(const T* row, int c, int cols, float* f) {
  constexpr int VEC = Elem<T>::VEC;
  if (c + 8 <= cols) {
#pragma unroll
    for (int h = 0; h < 8 / VEC; ++h) {
      const u32x4 v = load16(row + c + h * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[h * VEC + e] = Elem<T>::get(v, e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c + e < cols ? Elem<T>::load(row + c + e) : 0.f;
  }
}
__device__ __forceinline__ float amax8(const float* f, float a) {
  // NaN has to survive the maximum: a row with a NaN or an infinity has no scale
#pragma unroll
  for (int e = 0; e < 8; ++e) a = (fabsf(f[e]) > a || f[e] != f[e]) ? fabsf(f[e]) : a;
  return a;
}
__device__ __forceinline__ u32x2 quant8(const float* f, const RowScale& r, bool finite) {
  int q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = finite ? quant(f[e], r) : 0;
  return u32x2{pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7])};
}

// G lanes own a row, each 8 elements of every stretch of 8 G; NV stretches are kept in registers, so a row of up to
// 8 G NV elements is read once.  Longer rows (REREAD) are read twice, the second time from the L2.  A row with an
// infinity or a NaN gets the scale NaN and codes 0: its outputs are NaN, like those of a float32 product.
template <typename T, int G, bool REREAD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
  constexpr int NV = 4;
  __shared__ float red[4];
  const int g = threadIdx.x % G;
  const int64_t row0 = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = row0 < a.rows;
  const int64_t row = live ? row0 : a.rows - 1;
  const T* src = static_cast<const T*>(a.x) + row * a.stride;
  const int nv = (a.cols + 8 * G - 1) / (8 * G);
  float f[NV][8], amax = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (v < nv) load8_zero(src, (v * G + g) * 8, a.cols, f[v]);
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (v < nv) amax = amax8(f[v], amax);
  if constexpr (REREAD) {
    for (int v = NV; v < nv; ++v) {
      float t[8];
      load8_zero(src, (v * G + g) * 8, a.cols, t);
      amax = amax8(t, amax);
    }
  }
#pragma unroll
  for (int d = 1; d < (G < 64 ? G : 64); d <<= 1) {
    const float o = __shfl_xor(amax, d);
    amax = (o > amax || o != o) ? o : amax;
  }
  if constexpr (G == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) amax = (red[w] > amax || red[w] != red[w]) ? red[w] : amax;
  }
  const bool finite = amax < __builtin_inff();      // false for NaN too
  const RowScale r = row_scale(finite ? amax : 0.f);
  if (!live) return;
  if (g == 0) a.scale[row] = finite ? r.s / r.pre : __builtin_nanf("");
  int8_t* dst = a.q + row * a.ld;
  const int nq = (int)((a.ld + 8 * G - 1) / (8 * G));      // the zeros behind the row too
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * G + g) * 8;
    if (v < nv) {
      if (c < a.ld) *reinterpret_cast<u32x2*>(dst + c) = quant8(f[v], r, finite);
    }
  }
  for (int v = nv < NV ? nv : NV; v < nq; ++v) {
    const int c = (v * G + g) * 8;
    if (c >= a.ld) break;
    float t[8];
    if (REREAD && c < a.cols) {
      load8_zero(src, c, a.cols, t);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = 0.f;
    }
    *reinterpret_cast<u32x2*>(dst + c) = quant8(t, r, finite);
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
// v_exp_f32 and v_rcp_f32, one unit in the last place each: within 4 * 2^-24 of the sigmoid, whose slope is 1/4
__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}
__device__ __forceinline__ float activate(float v, int act) {
  return act == ACT_RELU ? relu(v) : act == ACT_LEAKY ? leaky(v) : act == ACT_SIGMOID ? sigmoid(v) : v;
}

template <typename T>
__device__ __forceinline__ void i8_store(const I8Args& p, int64_t i, int j, int acc, float sa, float sb, float bias) {
  float v = activate((float)acc * sa * sb + bias, p.act);
  if (p.residual) v += Elem<T>::load(static_cast<const T*>(p.residual) + i * p.ldr + j);
  static_cast<T*>(p.y)[i * p.ldy + j] = Elem<T>::from(v);
}

// ---- few rows: the weights are read once, straight into the matrix operands
// A block owns 16 channels and all of k; its NW waves take stretches of k (64 bytes of 16 weight rows an instruction, four
// instructions in flight) and add their partial sums through LDS.  MT tiles of 16 rows share every weight fragment.
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

// ---- tiles
// BM x BN outputs a block, BK bytes of k a step, WM x WN waves.  Both operands go straight from memory into LDS (16 bytes a
// lane, no registers between), two buffers: the next step's tile is in flight while this one is multiplied.  A row of a tile
// is BK bytes; its 16-byte chunks are permuted by the row number, so that the 8 lanes an LDS read serves at once, one chunk
// of 8 neighbouring rows, lie in different banks.  The permutation is made on the global side: LDS is written linearly.
template <int BK>
__device__ __forceinline__ int lds_chunk(int row, int chunk) {
  constexpr int C = BK / 16;
  return row * BK + ((chunk ^ (row * C / 8)) & (C - 1)) * 16;
}

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
      const int r = pos / C, ch = (pos ^ (r * C / 8)) & (C - 1);
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
  static __device__ __forceinline__ void store(float* p, const float* f) { store16(p, pack16<float>(f)); }
};
struct __attribute__((packed, aligned(2))) Pack8a2 { u32x2 v; };
template <typename T> struct Quad16 {
  static __device__ __forceinline__ void load(const T* p, float* f) {
    const u32x2 v = reinterpret_cast<const Pack8a2*>(p)->v;
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
    reinterpret_cast<Pack8a2*>(p)->v = v;
  }
};
template <> struct Quad<__bf16> : Quad16<__bf16> {};
template <> struct Quad<_Float16> : Quad16<_Float16> {};

// act is uniform: one scalar branch for four values
__device__ __forceinline__ void activate4(float* v, int act) {
  if (act == ACT_RELU) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = relu(v[e]);
  } else if (act == ACT_LEAKY) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = leaky(v[e]);
  } else if (act == ACT_SIGMOID) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = sigmoid(v[e]);
  }
}

// The loop: a step's fragments are read from LDS one 32-byte slice of k ahead of the matrix instructions that use them, and
// the barrier that hands a buffer over lies before the step's last slice, whose fragments are already in registers: the first
// reads of the next tile run under those matrix instructions.
// The epilogue goes through LDS, 32 rows of a wave at a time in a slab of its own: the accumulators hold one column a lane,
// memory wants whole 128-byte lines of a row.
template <typename T, int BM, int BN, int BK, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void i8_tiles(I8Args p, unsigned tiles_m, unsigned tiles_n) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int TM = BM / WM / 32, TN = BN / WN / 32;      // 32x32 tiles of a wave
  constexpr int KK = BK / 32, TILE = (BM + BN) * BK;
  static_assert(KK % 2 == 0, "slices alternate between two sets of registers");
  constexpr int SW = TN * 32, SLD = SW + 8;                // slab: 32 rows of SW floats; + 8: a lane's two row groups differ by 32 banks
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
      for (int i = 0; i < TM; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[slot][i], fb[slot][j], acc[i][j], 0, 0, 0);
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
  constexpr int QR = SW / 4, RP = 64 / QR;       // lanes a row, rows a pass
  const int qc = (lane % QR) * 4, qr = lane / QR;
  const int col = n0 + wn + qc;
  float scale[4], bias[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    scale[e] = col + e < p.n ? p.sb[col + e] : 0.f;
    bias[e] = p.bias && col + e < p.n ? p.bias[col + e] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    wave_lds_fence();
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        slab[((e >> 2) * 8 + (lane >> 5) * 4 + (e & 3)) * SLD + j * 32 + (lane & 31)] = (float)acc[i][j][e];
    wave_lds_fence();
#pragma unroll 4
    for (int r = qr; r < 32; r += RP) {
      const int64_t row = m0 + wm + i * 32 + r;
      if (row >= p.m || col >= p.n) continue;
      const u32x4 w = *reinterpret_cast<const u32x4*>(slab + r * SLD + qc);
      const float s = p.sa[row];
      float v[4], res[4];
      const bool whole = col + 4 <= p.n;
      const T* rp = static_cast<const T*>(p.residual) + row * p.ldr + col;
      T* yp = static_cast<T*>(p.y) + row * p.ldy + col;
      if (p.residual) {
        if (whole) {
          Quad<T>::load(rp, res);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) res[e] = col + e < p.n ? Elem<T>::load(rp + e) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(__uint_as_float(w[e]) * s, scale[e], bias[e]);
      activate4(v, p.act);
      if (p.residual) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += res[e];
      }
      if (whole) {
        Quad<T>::store(yp, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < p.n) yp[e] = Elem<T>::from(v[e]);
      }
    }
  }
}

}  // namespace pclseg

#endif  // PCLSEG_I8_H_
