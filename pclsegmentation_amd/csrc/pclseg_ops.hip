// pclseg_ops.hip — C entry points of the row operators (include/pclseg.h): argument checks, choice of a kernel, launch.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdio.h>

#include <algorithm>
#include <string>

#include "../../include/pclseg.h"
#include "pclseg_i8.h"
#include "pclseg_score.h"
#include "pclseg_status.h"

using namespace pclseg;

namespace {

#define OP_CATCH catch (...) { return pclseg::op_exception(); }

int bad(const char* op, const char* what) { return op_fail(PCLSEG_ERR_BAD_ARG, std::string(op) + ": " + what); }
int bad_shape(const char* op, const char* what) { return op_fail(PCLSEG_ERR_BAD_SHAPE, std::string(op) + ": " + what); }
int launched(const char* op) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return PCLSEG_OK;
  return op_fail(e == hipErrorOutOfMemory ? PCLSEG_ERR_OOM : PCLSEG_ERR_HIP, std::string(op) + ": " + hipGetErrorString(e));
}
bool dtype_ok(int d) { return d == PCLSEG_F32 || d == PCLSEG_BF16 || d == PCLSEG_F16; }
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
size_t dtype_size(int d) { return d == PCLSEG_F32 ? 4 : 2; }

// Rows of `cols` elements of `size` bytes, `stride` elements apart.
struct Rows { const void* p; int64_t stride, cols, size; };
// Do two arrays of m >= 1 rows share a byte?  With equal strides in bytes the rows may lie side by side in one buffer; with
// different ones address ranges that meet count as shared.
bool overlap(const Rows& a, const Rows& b, int64_t m) {
  typedef unsigned __int128 U;
  const U a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p, as = (U)a.stride * (U)a.size, bs = (U)b.stride * (U)b.size;
  const U aw = (U)(a.cols * a.size), bw = (U)(b.cols * b.size), above = (U)(m - 1);
  if (a0 + above * as + aw <= b0 || b0 + above * bs + bw <= a0) return false;
  if (m == 1 || as != bs) return true;
  const U d = b0 >= a0 ? (b0 - a0) % as : (as - (a0 - b0) % as) % as;      // b's rows begin d bytes into a's
  return d < aw || d + bw > as;
}
constexpr int64_t kMaxBlocks = 0x7fffffff, kMaxThreads = 0xffffffff;      // of a launch: blocks, and threads along an axis
// columns are counted in 32 bits, with room for a block's share behind the last; products of rows and columns stay below 2^63
constexpr int64_t kMaxRows = (int64_t)1 << 40, kMaxColumns = 1 << 30;

// Launches on a stream one after the other; after one that fails or does not fit a launch, none.  dry: looks the sizes over only.
struct Launch {
  const char* op;
  hipStream_t s;
  bool dry = false;
  int rc = PCLSEG_OK;
  template <typename... P, typename... A> void run(void (*kernel)(P...), int64_t blocks, unsigned blocks_y, int threads, size_t lds, A... args) {
    if (rc) return;
    if (blocks > std::min<int64_t>(kMaxBlocks, kMaxThreads / threads)) {
      rc = bad_shape(op, "more rows or output tiles than a launch has blocks for");
      return;
    }
    if (dry) return;
    kernel<<<dim3((unsigned)blocks, blocks_y), dim3(threads), lds, s>>>(args...);
    rc = launched(op);
  }
  template <typename... P, typename... A> void operator()(void (*kernel)(P...), int64_t blocks, int threads, A... args) {
    run(kernel, blocks, 1, threads, 0, args...);
  }
};

// calls f with a value of the element type
template <typename F> void with_type(int dtype, F f) {
  if (dtype == PCLSEG_F32) f(float{});
  else if (dtype == PCLSEG_BF16) f(__bf16{});
  else f(_Float16{});
}

// ---------------------------------------------------------------------------------------------- quantisation, product
int64_t row_bytes(int64_t k) {
  if (k < 1 || k > PCLSEG_I8_K_MAX) return 0;
  return k <= 64 ? 64 : (k + 127) / 128 * 128;
}

template <typename T, int G> void launch_quant(const QuantArgs& a, Launch& go) {
  const int64_t blocks = (a.rows + 256 / G - 1) / (256 / G);
  if (a.cols > 32 * G) go(quantize_rows_kernel<T, G, true>, blocks, 256, a);
  else go(quantize_rows_kernel<T, G, false>, blocks, 256, a);
}

int quantize(Launch go, const void* x, int dtype, int64_t rows, int64_t cols, int64_t stride, int8_t* q, float* scale) {
  QuantArgs a{x, rows, stride, (int)cols, q, row_bytes(cols), scale};
  with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (cols <= 256) launch_quant<T, 8>(a, go);
    else if (cols <= 2048) launch_quant<T, 64>(a, go);
    else launch_quant<T, 256>(a, go);
  });
  return go.rc;
}

template <typename T, int BM, int BN, int BK, int WM, int WN, int OCC>
void launch_tiles(const I8Args& p, Launch& go) {
  const int64_t tm = (p.m + BM - 1) / BM, tn = (p.n + BN - 1) / BN;
  go(i8_tiles<T, BM, BN, BK, WM, WN, OCC>, tm * tn, WM * WN * 64, p, (unsigned)tm, (unsigned)tn);
}

int matmul(Launch go, const I8Args& p, int dtype) {
  auto tiles = [&](int bm, int bn) { return ((p.m + bm - 1) / bm) * ((p.n + (int64_t)bn - 1) / bn); };
  with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (p.m <= 64 || tiles(64, 64) < 192) {
      // row tiles a block shares its weights among: as many as there are, while 256 blocks remain
      const int64_t cols = (p.n + 15) / 16;
      const int mt = p.m > 32 && cols * ((p.m + 63) / 64) >= 256 ? 4 : p.m > 16 && cols * ((p.m + 31) / 32) >= 256 ? 2 : 1;
      const unsigned rows = (unsigned)((p.m + 16 * mt - 1) / (16 * mt));
      if (mt == 1) go.run(i8_few_rows<T, 1, 8>, cols, rows, 512, 0, p);
      else if (mt == 2) go.run(i8_few_rows<T, 2, 8>, cols, rows, 512, 0, p);
      else go.run(i8_few_rows<T, 4, 8>, cols, rows, 512, 0, p);
      return;
    }
    // The largest tile that fills the 256 CUs.  m x n x k, the product alone, one call after the other: 8192x8192x4096 bf16
    // 290 us with 256x256 tiles, 303 with 128x128, 426 with 64x64; 8192x512x1024 float32 17.5 / 9.5 / 10.5 us; 512x4096x4096
    // 44 / 20.6 / 18.0 us.  Between the first two the rounds decide, in units of a CU's time for a 128x128 tile: one 256x256 tile
    // a CU costs 4, two 128x128 tiles 2 and 5 % more (15642x1260x2235 float32 with its quantisation, ten calls in a graph:
    // 116 us in two rounds of 256x256, 1.2 of them needed, 97 in three of 128x128).
    // Up to 256 columns of many rows a tile is mostly stores: 128x128 with steps of 64 bytes, three of them on a CU, one
    // storing while the others multiply, from 16 tiles a CU on (with the quantisation, ten in a graph: 131072x512x128 float32
    // 68 us against 78 with 256x256, 131072x512x256 89 against 97; the product 8192x2048x256 bf16, four tiles a CU: 24.5
    // against 21.7; 131072x1024x512 float32: 206 against 205, and 286 against 276 with the caches flushed before each call).
    // Up to 64 channels nothing wider than they are (the product 131072x64x128: 8.4 us against 14.1 with 128x128; with the
    // quantisation and flushed caches 131072x64x50 bf16: 23 against 33).
    const int64_t big = (tiles(256, 256) + 255) / 256 * 4 * 20, mid = (tiles(128, 128) + 511) / 512 * 2 * 21;
    if (p.n <= 64 && p.kp == 64) launch_tiles<T, 128, 64, 64, 2, 2, 4>(p, go);
    else if (p.n <= 64) launch_tiles<T, 64, 64, 128, 2, 2, 4>(p, go);
    else if (p.kp == 64 || (p.kp <= 256 && tiles(128, 128) >= 4096)) launch_tiles<T, 128, 128, 64, 2, 2, 3>(p, go);
    else if (tiles(256, 256) >= 192 && big <= mid) launch_tiles<T, 256, 256, 128, 2, 4, 2>(p, go);
    else if (tiles(128, 128) >= 192) launch_tiles<T, 128, 128, 128, 4, 2, 4>(p, go);
    else launch_tiles<T, 64, 64, 128, 2, 2, 4>(p, go);
  });
  return go.rc;
}

// Up to 32 rows of together 64 items of 512 elements in one launch, no workspace (see i8_fused_rows): every block of 16 channels
// quantises all rows, which saves a launch and a workspace (3.5 us of a pass, 13 us with two) and costs with the blocks.  A
// pass of bf16 rows, one launch / two: up to 512 blocks, two a CU, and 2^14 items quantised in all
//   1x1024 -> 8192   9.5 / 13.0   16x1024 -> 8192  10.9 / 13.2   32x1024 -> 4096  11.7 / 13.1     (one launch)
//   1x1024 -> 32768 19.5 / 12.6    8x4096 -> 8192  15.5 / 12.8   32x1024 -> 8192  16.5 / 13.2   32x1024 -> 131072 180 / 53
// and one or two rows of 4096 columns and more for any n: a block's 64 KB of weights take longer than its items
//   1x4096 -> 131072  92 / 111     2x4096 -> 131072 102 / 113     4x4096 -> 32768  34.8 / 31.6 (two launches).
bool fused_rows(int64_t m, int64_t n, int64_t k) {
  const int64_t items = m * ((row_bytes(k) + 511) / 512), blocks = (n + 15) / 16;
  if (m > kFusedRows || items > kFusedItems) return false;
  return (m <= 2 && k >= 4096) || (blocks <= 512 && items * blocks <= 1 << 14);
}
size_t linear_workspace(int64_t m, int64_t n, int64_t k) {
  return fused_rows(m, n, k) ? 0 : (size_t)m * ((size_t)row_bytes(k) + sizeof(float));
}

int check_product(const char* op, int64_t m, int64_t n, int64_t k, const int8_t* b, const float* b_scale, int act,
                  const void* residual, int64_t residual_stride, const void* y, int64_t y_stride, int dtype) {
  if (!dtype_ok(dtype)) return bad(op, "unknown dtype");
  if (act < 0 || act > 3) return bad(op, "unknown activation");
  if (m < 0 || m > kMaxRows || n < 1 || n > kMaxColumns) return bad_shape(op, "m must be in [0, 2^40], n must be in [1, 2^30]");
  if (!row_bytes(k)) return bad_shape(op, "k must be in [1, 131071]");
  if (!b || !b_scale || (m && !y)) return bad(op, "NULL buffer");
  if (!aligned(b, 16)) return bad(op, "codes must be 16-byte aligned");
  if (y_stride < n || (residual && residual_stride < n)) return bad_shape(op, "row stride smaller than n");
  if (!aligned(y, dtype_size(dtype)) || !aligned(residual, dtype_size(dtype))) return bad(op, "misaligned y or residual");
  // an element's residual is read by the lane that stores it: y itself is fine, any other overlap is a race
  const int64_t sz = (int64_t)dtype_size(dtype);
  if (m && residual && !(residual == y && residual_stride == y_stride) &&
      overlap({residual, residual_stride, n, sz}, {y, y_stride, n, sz}, m))
    return bad(op, "y overlaps the residual without being it");
  return PCLSEG_OK;
}

// ---------------------------------------------------------------------------------------------- log probabilities
constexpr int kThreadRow = 32, kGroupRow = 2048, kPiece = 2048, kRounds = 4, kManyRows = 2048, kFewRows = 256;
constexpr int kSortRows = 8192, kOneLaunch = 16, kFewWaves = 4;       // pieces one block of 16 waves takes, pieces that 4 waves are enough for

// blocks a row is cut into: one up to 32768 classes (a piece for each of 16 waves) and from 32 rows on; else as many as keep
// few rows from waiting on few CUs (one row of 131072 with 20 alternatives: 22 us in one block, 12 in 16 and a second
// launch that joins them)
int score_segs(int64_t rows, int64_t classes) {
  const int64_t pieces = (classes + kPiece - 1) / kPiece;
  if (pieces <= kOneLaunch || rows >= 32) return 1;
  return (int)std::min<int64_t>(std::min<int64_t>(pieces / 4, 64), 256 / rows);
}
size_t score_workspace(int64_t rows, int64_t classes, int top_k) {
  const int segs = rows > 0 ? score_segs(rows, classes) : 1;
  return segs == 1 ? 0 : (size_t)rows * segs * (sizeof(ScorePart) + (top_k ? 64 * sizeof(Key) : 0));
}

template <typename T, bool MASK, int CAP> void launch_thread_rows(const ScoreArgs& a, Launch& go) {
  if constexpr (CAP > Elem<T>::VEC) {
    if (a.classes <= CAP - Elem<T>::VEC) return launch_thread_rows<T, MASK, CAP - Elem<T>::VEC>(a, go);
  }
  go(logprob_thread_rows<T, CAP, MASK>, (a.rows + 255) / 256, 256, a);
}

template <typename T, bool MASK> void launch_score(const ScoreArgs& a, Launch& go) {
  const int v = a.classes;
  if (v <= kThreadRow) {
    launch_thread_rows<T, MASK, kThreadRow>(a, go);
  } else if (v <= kGroupRow && (a.top_k <= kRounds || (v <= 256 && a.rows > kSortRows))) {
    // (longer lists go to the waves below, which sort, unless many short rows make a wave for each the larger cost:
    // 673x56 with 20 alternatives 23 us here, 8 there)
    auto blocks = [&](int g) { return (a.rows + 256 / g - 1) / (256 / g); };
    if (v <= 8 * 32) go(logprob_group_rows<T, 8, MASK>, blocks(8), 256, a);
    else if (v <= 16 * 32) go(logprob_group_rows<T, 16, MASK>, blocks(16), 256, a);
    else if (v <= 32 * 32) go(logprob_group_rows<T, 32, MASK>, blocks(32), 256, a);
    else go(logprob_group_rows<T, 64, MASK>, blocks(64), 256, a);
  } else {
    const int64_t blocks = a.rows * a.segs;
    // one wave a row where that fills the chip: a list is kept and merged once a row instead of four times
    if (v > kPiece && a.rows < kManyRows) {
      if (v > kFewWaves * kPiece && a.rows <= kFewRows && a.segs == 1) {
        if (a.top_k) go(logprob_wave_rows<T, 16, true, MASK>, blocks, 1024, a);
        else go(logprob_wave_rows<T, 16, false, MASK>, blocks, 1024, a);
      } else {
        if (a.top_k) go(logprob_wave_rows<T, 4, true, MASK>, blocks, 256, a);
        else go(logprob_wave_rows<T, 4, false, MASK>, blocks, 256, a);
      }
    } else {
      if (a.top_k) go(logprob_wave_rows<T, 1, true, MASK>, blocks, 64, a);
      else go(logprob_wave_rows<T, 1, false, MASK>, blocks, 64, a);
    }
    if (a.segs > 1) {
      if (a.top_k) go(logprob_join<T, true>, a.rows, 256, a);
      else go(logprob_join<T, false>, a.rows, 256, a);
    }
  }
}

int check_rows(const char* op, const void* logits, int dtype, int64_t rows, int64_t classes, int64_t stride,
               const void* labels, int label_bytes, const uint8_t* allowed, int64_t allowed_stride, int top_k) {
  if (!dtype_ok(dtype)) return bad(op, "unknown dtype");
  if (rows < 0 || rows > kMaxRows || classes < 1 || classes > kMaxColumns)
    return bad_shape(op, "rows must be in [0, 2^40], classes must be in [1, 2^30]");
  if (stride < classes) return bad_shape(op, "row stride smaller than classes");
  if (top_k < 0 || top_k > PCLSEG_TOP_MAX) return bad(op, "top_k must be in [0, 64]");
  if (rows && !logits) return bad(op, "logits is NULL");
  if (!aligned(logits, dtype_size(dtype))) return bad(op, "misaligned logits");
  if (labels && label_bytes != 4 && label_bytes != 8) return bad(op, "labels are int32 or int64");
  if (labels && !aligned(labels, (size_t)label_bytes)) return bad(op, "misaligned labels");
  if (allowed && allowed_stride != 0 && allowed_stride < classes) return bad_shape(op, "mask stride smaller than classes");
  return PCLSEG_OK;
}

int score_grad(const char* op, const void* logits, int dtype, int64_t rows, int64_t classes, int64_t stride, const void* labels,
               int label_bytes, const uint8_t* allowed, int64_t allowed_stride, const float* lse, const float* entropy,
               const float* logprob, const int32_t* top_ids, const float* top_logprobs, const float* d_logprob,
               const float* d_entropy, const float* d_top, int top_k, void* grad, int64_t grad_stride, void* hip_stream) {
  const int rc = check_rows(op, logits, dtype, rows, classes, stride, labels, label_bytes, allowed, allowed_stride, top_k);
  if (rc) return rc;
  if (!d_logprob && !d_entropy && !d_top) return bad(op, "no gradient arrives");
  if (d_logprob && !labels) return bad(op, "d_logprob needs labels");
  if (d_entropy && !entropy) return bad(op, "d_entropy needs entropy");
  if (d_top && (!top_ids || top_k < 1)) return bad(op, "d_top needs top_ids and top_k");
  if (logprob && !labels) return bad(op, "logprob needs labels");
  if (top_logprobs && (!top_ids || top_k < 1)) return bad(op, "top_logprobs needs top_ids and top_k");
  if (grad_stride < classes) return bad_shape(op, "gradient stride smaller than classes");
  if (rows == 0) return PCLSEG_OK;
  if (!lse || !grad) return bad(op, "NULL buffer");
  if (!aligned(grad, dtype_size(dtype))) return bad(op, "misaligned grad");
  const int64_t sz = (int64_t)dtype_size(dtype);
  if (overlap({logits, stride, classes, sz}, {grad, grad_stride, classes, sz}, rows)) return bad(op, "grad overlaps the logits");
  GradArgs a{logits, rows, stride, (int)classes, d_logprob || logprob ? labels : nullptr, label_bytes == 8, allowed, allowed_stride,
             lse, entropy, d_logprob, d_entropy, top_ids, d_top, d_top || top_logprobs ? top_k : 0, logprob, top_logprobs, grad,
             grad_stride, 1, 1, 1, 0};
  // a block takes 256 NI 16-byte pieces: that many of a long row, or whole short rows.  NI grows while the blocks are more
  // than the 2048 that run at once
  const int64_t vec = 16 / sz, nvec = (classes + vec - 1) / vec;
  const int64_t all = std::min<int64_t>(rows, kMaxBlocks) * nvec;
  const int ni = all <= 2048 * 256 ? 1 : all <= 2 * 2048 * 256 ? 2 : 4;
  if (nvec > 256 * ni) {
    a.vecs = 256 * ni;
    a.cuts = (int)((nvec + 1 + a.vecs - 1) / a.vecs);      // one piece more: a row may begin inside its first
  } else {
    a.vecs = (int)nvec;
    a.rows_per_block = (int)std::min<int64_t>(std::min<int64_t>(256, 256 * ni / nvec), kGradNames / (a.top_k + 1));
  }
  a.magic = (uint32_t)(((1u << 20) + a.vecs - 1) / a.vecs);
  const int64_t blocks = a.cuts > 1 ? rows * a.cuts : (rows + a.rows_per_block - 1) / a.rows_per_block;
  Launch go{op, (hipStream_t)hip_stream};
  with_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    if (allowed) {
      if (ni == 1) go(logprob_grad<T, true, 1>, blocks, 256, a);
      else if (ni == 2) go(logprob_grad<T, true, 2>, blocks, 256, a);
      else go(logprob_grad<T, true, 4>, blocks, 256, a);
    } else {
      if (ni == 1) go(logprob_grad<T, false, 1>, blocks, 256, a);
      else if (ni == 2) go(logprob_grad<T, false, 2>, blocks, 256, a);
      else go(logprob_grad<T, false, 4>, blocks, 256, a);
    }
  });
  return go.rc;
}

}  // namespace

extern "C" {

int64_t pclseg_i8_row_bytes(int64_t k) { return row_bytes(k); }

int pclseg_op_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_stride, int8_t* q,
                            float* scale, void* hip_stream) try {
  const char* op = "op_quantize_rows";
  if (!dtype_ok(dtype)) return bad(op, "unknown dtype");
  if (rows < 0 || rows > kMaxBlocks || !row_bytes(cols)) return bad_shape(op, "rows must be in [0, 2^31), cols in [1, 131071]");
  if (x_stride < cols) return bad_shape(op, "row stride smaller than cols");
  if (rows == 0) return PCLSEG_OK;
  if (!x || !q || !scale) return bad(op, "NULL buffer");
  if (!aligned(x, dtype_size(dtype)) || !aligned(q, 8)) return bad(op, "misaligned x or codes");
  const int rc = quantize({op, nullptr, true}, x, dtype, rows, cols, x_stride, q, scale);
  if (rc) return rc;
  const int64_t ld = row_bytes(cols);
  if (overlap({x, x_stride, cols, (int64_t)dtype_size(dtype)}, {q, ld, ld, 1}, rows)) return bad(op, "codes overlap x");
  return quantize({op, (hipStream_t)hip_stream}, x, dtype, rows, cols, x_stride, q, scale);
} OP_CATCH

int pclseg_op_matmul_i8(const int8_t* a, const float* a_scale, const int8_t* b, const float* b_scale, int64_t m,
                        int64_t n, int64_t k, const float* bias, int act, const void* residual, int64_t residual_stride,
                        void* y, int64_t y_stride, int dtype, void* hip_stream) try {
  const char* op = "op_matmul_i8";
  const int rc = check_product(op, m, n, k, b, b_scale, act, residual, residual_stride, y, y_stride, dtype);
  if (rc) return rc;
  if (m == 0) return PCLSEG_OK;
  if (!a || !a_scale) return bad(op, "NULL buffer");
  if (!aligned(a, 16)) return bad(op, "codes must be 16-byte aligned");
  I8Args p{a, b, a_scale, b_scale, row_bytes(k), row_bytes(k), m, (int)n, (int)row_bytes(k), bias, act, residual,
           residual_stride, y, y_stride};
  return matmul({op, (hipStream_t)hip_stream}, p, dtype);
} OP_CATCH

int pclseg_op_linear_i8_workspace(int64_t m, int64_t n, int64_t k, size_t* bytes) try {
  const char* op = "op_linear_i8_workspace";
  if (!bytes) return bad(op, "bytes is NULL");
  if (m < 0 || m > kMaxBlocks || n < 1 || !row_bytes(k)) return bad_shape(op, "m must be in [0, 2^31), n positive, k in [1, 131071]");
  *bytes = linear_workspace(m, n, k);
  return PCLSEG_OK;
} OP_CATCH

int pclseg_op_linear_i8(const void* x, int dtype, int64_t x_stride, const int8_t* weight, const float* weight_scale,
                        int64_t m, int64_t n, int64_t k, const float* bias, int act, const void* residual,
                        int64_t residual_stride, void* y, int64_t y_stride, int y_dtype, void* workspace,
                        size_t workspace_bytes, void* hip_stream) try {
  const char* op = "op_linear_i8";
  const int rc = check_product(op, m, n, k, weight, weight_scale, act, residual, residual_stride, y, y_stride, y_dtype);
  if (rc) return rc;
  if (!dtype_ok(dtype)) return bad(op, "unknown dtype");
  if (m > kMaxBlocks || x_stride < k) return bad_shape(op, "m must be below 2^31, the row stride at least k");
  if (m == 0) return PCLSEG_OK;
  if (!x) return bad(op, "NULL buffer");
  if (!aligned(x, dtype_size(dtype))) return bad(op, "misaligned x");
  const int64_t ld = row_bytes(k);
  Launch go{op, (hipStream_t)hip_stream};
  // few rows in one launch: every block reads all of x while others store y.  Refused for any number of rows alike, after the
  // checks of sizes
  const bool shared = overlap({x, x_stride, k, (int64_t)dtype_size(dtype)}, {y, y_stride, n, (int64_t)dtype_size(y_dtype)}, m);
  if (fused_rows(m, n, k)) {
    I8Args p{nullptr, weight, nullptr, weight_scale, ld, ld, m, (int)n, (int)ld, bias, act, residual, residual_stride, y, y_stride};
    go.dry = shared;
    with_type(dtype, [&](auto t) {
      with_type(y_dtype, [&](auto u) {
        typedef decltype(t) T;
        typedef decltype(u) Y;
        const int64_t blocks = (n + 15) / 16;
        const size_t lds = (size_t)(m * ld);
        if (m <= 16) go.run(i8_fused_rows<T, Y, 1>, blocks, 1, 512, lds, p, static_cast<const T*>(x), x_stride, (int)k);
        else go.run(i8_fused_rows<T, Y, 2>, blocks, 1, 512, lds, p, static_cast<const T*>(x), x_stride, (int)k);
      });
    });
    return go.rc ? go.rc : shared ? bad(op, "y overlaps x") : PCLSEG_OK;
  }
  if (!workspace || workspace_bytes < linear_workspace(m, n, k)) return bad(op, "workspace too small");
  if (!aligned(workspace, 16)) return bad(op, "misaligned workspace");
  int8_t* q = static_cast<int8_t*>(workspace);
  float* scale = reinterpret_cast<float*>(q + m * ld);
  I8Args p{q, weight, scale, weight_scale, ld, ld, m, (int)n, (int)ld, bias, act, residual, residual_stride, y, y_stride};
  const int rm = matmul({op, go.s, true}, p, y_dtype);      // a product that does not fit a launch is refused before the first
  if (rm) return rm;
  go.dry = shared;
  const int rq = quantize(go, x, dtype, m, k, x_stride, q, scale);
  if (rq) return rq;
  return shared ? bad(op, "y overlaps x") : matmul(go, p, y_dtype);
} OP_CATCH

int pclseg_op_label_logprobs_workspace(int64_t rows, int64_t classes, int top_k, size_t* bytes) try {
  const char* op = "op_label_logprobs_workspace";
  if (!bytes) return bad(op, "bytes is NULL");
  const int rc = check_rows(op, bytes, PCLSEG_BF16, rows, classes, classes, nullptr, 0, nullptr, 0, top_k);
  if (rc) return rc;
  *bytes = score_workspace(rows, classes, top_k);
  return PCLSEG_OK;
} OP_CATCH

int pclseg_op_label_logprobs(const void* logits, int dtype, int64_t rows, int64_t classes, int64_t stride,
                             const void* labels, int label_bytes, const uint8_t* allowed, int64_t allowed_stride, int top_k,
                             float* logprob, float* entropy, float* lse, int32_t* top_ids, float* top_logprobs,
                             void* workspace, size_t workspace_bytes, void* hip_stream) try {
  const char* op = "op_label_logprobs";
  const int rc = check_rows(op, logits, dtype, rows, classes, stride, labels, label_bytes, allowed, allowed_stride, top_k);
  if (rc) return rc;
  if (logprob && !labels) return bad(op, "logprob needs labels");
  if (rows == 0) return PCLSEG_OK;
  if (top_k && (!top_ids || !top_logprobs)) return bad(op, "top_k without top_ids and top_logprobs");
  const size_t need = score_workspace(rows, classes, top_k);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return bad(op, "workspace too small or misaligned");
  ScoreArgs a{logits, rows, stride, (int)classes, labels, label_bytes == 8, allowed, allowed_stride, top_k,
              logprob, entropy, lse, top_ids, top_logprobs, workspace, score_segs(rows, classes)};
  Launch go{op, (hipStream_t)hip_stream};
  with_type(dtype, [&](auto t) {
    if (allowed) launch_score<decltype(t), true>(a, go);
    else launch_score<decltype(t), false>(a, go);
  });
  return go.rc;
} OP_CATCH

int pclseg_op_label_logprobs_grad(const void* logits, int dtype, int64_t rows, int64_t classes, int64_t stride,
                                  const void* labels, int label_bytes, const uint8_t* allowed, int64_t allowed_stride,
                                  const float* lse, const float* entropy, const float* d_logprob, const float* d_entropy,
                                  const int32_t* top_ids, const float* d_top, int top_k, void* grad, int64_t grad_stride,
                                  void* hip_stream) try {
  return score_grad("op_label_logprobs_grad", logits, dtype, rows, classes, stride, labels, label_bytes, allowed, allowed_stride, lse,
                    entropy, nullptr, top_ids, nullptr, d_logprob, d_entropy, d_top, top_k, grad, grad_stride, hip_stream);
} OP_CATCH

}  // extern "C"

#ifndef PCLSEG_OPS_SHA
#define PCLSEG_OPS_SHA "unknown"
#endif

extern "C" {

const char* pclseg_ops_build_sha(void) { return PCLSEG_OPS_SHA; }

// the gradient with what the forward pass knew of the names

int pclseg_op_label_logprobs_grad_ex(const void* logits, int dtype, int64_t rows, int64_t classes, int64_t stride,
                                     const void* labels, int label_bytes, const uint8_t* allowed, int64_t allowed_stride,
                                     const float* lse, const float* entropy, const float* logprob, const int32_t* top_ids,
                                     const float* top_logprobs, const float* d_logprob, const float* d_entropy,
                                     const float* d_top, int top_k, void* grad, int64_t grad_stride, void* hip_stream) try {
  return score_grad("op_label_logprobs_grad_ex", logits, dtype, rows, classes, stride, labels, label_bytes, allowed, allowed_stride,
                    lse, entropy, logprob, top_ids, top_logprobs, d_logprob, d_entropy, d_top, top_k, grad, grad_stride, hip_stream);
} OP_CATCH

}  // extern "C"
