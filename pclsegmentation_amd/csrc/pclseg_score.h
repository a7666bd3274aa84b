// pclseg_score.h — log probabilities of given labels, entropy and top alternatives of rows of logits, and their gradient.
//
// For a row x[0..V) with the classes A = {j : allowed[j], x[j] > -inf}:
//   M = max x,  S = sum e^(x-M),  T = sum e^(x-M) (x-M)          (sums over A)
//   lse = M + ln S,   logprob = (x[label] - M) - ln S,   entropy = ln S - T / S
// (M, S, T) of two disjoint parts join with M = max(M1, M2), d = Mi - M <= 0:  S += Si e^d, T += e^d (Ti + d Si), so a row
// is read once and can be cut anywhere.  Rows are often decided: S = 1 + rest with a rest of 2^-10 would leave ln S 14 bits.
// The maximum's term is kept apart from the others (one, s below), and ln S = ln(1 + rest) keeps the bits of the rest.
// All of it is float32: the terms of S and T have one sign, and the differences x - M are taken before the exponential, so large
// logits lose nothing.  A lane adds up to 32 elements one after the other; such sums of a long row's pieces are added with the
// rounding of each addition carried into the next, so that a sum is a few tens of roundings from the exact one, 2^-24 each,
// whatever the row's length (131072 terms one after the other, most of them alike: 450 roundings off).
// The exponential is v_exp_f32 on (x-M) log2 e: the rounding of that product makes an error of |x-M| 2^-24 of the term, which
// weighs e^(x-M) (4096 x 50001 bf16: 5.3e-8 from the exact values all in all).
// Terms with x - M < -200 are 0 in float32; the clamp of the second factor at -200 keeps 0 * inf out of T.
//
// Three kernels, by the length of a row (what a row costs besides its elements is what differs):
//   logprob_thread_rows   V <= 32    a thread owns a row: no exchange between lanes at all
//   logprob_group_rows    V <= 2048  8, 16, 32 or 64 lanes own a row, held in registers; a short top list by rounds of argmax
//   logprob_wave_rows     longer     a wave, the waves of a block, or several blocks stream a row in pieces of 2048 elements;
//                                    a long top list as one sorted key per lane
// What they reach, one call after the other: 4194304 x 20 float32 with 3 alternatives 112 us (503 MB, 4.5 TB/s), 4096 x 50001 bf16
// with 8 alternatives 87 us and without 81 us (410 MB, 5.1 TB/s), 333 x 1031 f16 with 32 alternatives 8.2 us.
#ifndef PCLSEG_SCORE_H_
#define PCLSEG_SCORE_H_

#include "pclseg_rows.h"

namespace pclseg {

struct ScoreArgs {
  const void* x;             // logits, rows of `classes` elements, `stride` elements apart
  int64_t rows, stride;
  int classes;
  const void* labels;        // int32 or int64 (label64), NULL: none
  int label64;
  const uint8_t* allowed;    // NULL: all classes
  int64_t allowed_stride;    // 0: one mask for all rows
  int top_k;
  float *logprob, *entropy, *lse;   // each may be NULL
  int32_t* top_ids;
  float* top_logprobs;
  void* part;                // workspace of a split row
  int segs;                  // blocks a row is cut into
};

constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.44269504088896340736f;

// S = one + s: one is 1 where the term of a maximum is left out of s, else 0; t holds all of T
struct Stat { float m, one, s, t; };

__device__ __forceinline__ float fast_exp(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }

// What elements are worth that were summed relative to the maximum m: s the terms, below the terms less than 1 (a term of 1
// has the fraction 0), t.  The two sums differ by the count of maxima; a single one is kept apart.
__device__ __forceinline__ Stat stat_of(float m, float s, float below, float t) {
  const bool one = rintf(s - below) == 1.f;
  return Stat{m, one ? 1.f : 0.f, one ? below : s, t};
}
// sum += v with the rounding of the last addition: sum - lost is the sum
__device__ __forceinline__ void add_carried(float& sum, float& lost, float v) {
  const float y = v - lost, u = sum + y;
  lost = (u - sum) - y;
  sum = u;
}

// a row's results.  S == 0: nothing is allowed (or every allowed logit is -inf); S NaN: an allowed logit is NaN or +inf, the
// row has no distribution and every float result is NaN.
struct RowOut { float m, logs, lse, entropy; bool empty, bad; };
__device__ __forceinline__ RowOut row_out(const Stat& a) {
  RowOut o;
  const float sum = a.one + a.s;
  o.empty = sum == 0.f;
  o.bad = !(sum < __builtin_inff());
  o.m = a.m;
  // ln(one + s) of the rounded sum, and what the rounding left, to first order: the bits of a small s stay
  o.logs = logf(sum) + (a.s - (sum - a.one)) * __builtin_amdgcn_rcpf(sum);
  o.lse = o.empty ? neg_inf() : (o.bad ? __builtin_nanf("") : a.m + o.logs);
  o.entropy = o.empty ? 0.f : (o.bad ? __builtin_nanf("") : o.logs - a.t / sum);
  return o;
}
__device__ __forceinline__ float row_logprob(const RowOut& o, float x) {
  if (o.bad) return __builtin_nanf("");
  return x == neg_inf() ? neg_inf() : (x - o.m) - o.logs;
}

__device__ __forceinline__ int64_t label_of(const ScoreArgs& a, int64_t row) {
  if (!a.labels) return -1;
  return a.label64 ? static_cast<const int64_t*>(a.labels)[row] : static_cast<const int32_t*>(a.labels)[row];
}

// logprob, entropy and lse of a row: called by one lane
template <typename T> __device__ __forceinline__ void write_row(const ScoreArgs& a, int64_t row, const RowOut& o) {
  if (a.entropy) a.entropy[row] = o.entropy;
  if (a.lse) a.lse[row] = o.lse;
  if (a.logprob) {
    const int64_t lab = label_of(a, row);
    float lp = 0.f;
    if (lab >= 0 && lab < a.classes) {
      float x = Elem<T>::load(static_cast<const T*>(a.x) + row * a.stride + lab);
      if (a.allowed && !a.allowed[row * a.allowed_stride + lab]) x = neg_inf();
      lp = row_logprob(o, x);
    }
    a.logprob[row] = lp;
  }
}

// 16 bytes of a row and the bytes of its mask (MASK): requested first, looked at later, so that a lane's loads are all in
// flight
template <typename T, bool MASK> struct Piece {
  static constexpr int VEC = Elem<T>::VEC;
  u32x4 v;
  uint32_t mk[MASK ? VEC / 4 : 1];
  // elements [c, c + VEC) of a row, all inside it
  __device__ __forceinline__ void load(const T* row, const uint8_t* mask, int64_t c) {
    v = load16(row + c);
    if constexpr (MASK) {
#pragma unroll
      for (int h = 0; h < VEC / 4; ++h) mk[h] = reinterpret_cast<const Pack4a1*>(mask + c + h * 4)->v;
    }
  }
  __device__ __forceinline__ void expand(float* f) const {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = Elem<T>::get(v, e);
    if constexpr (MASK) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = (mk[e / 4] >> (8 * (e % 4))) & 0xff ? f[e] : neg_inf();
    }
  }
};
// the same where the row may begin (c < 0) or end inside: -inf outside of it
template <typename T, bool MASK>
__device__ __forceinline__ void load_tail(const T* row, const uint8_t* mask, int c, int classes, float* f) {
  constexpr int VEC = Elem<T>::VEC;
  if (c >= 0 && c + VEC <= classes) {
    Piece<T, MASK> m;
    m.load(row, mask, c);
    m.expand(f);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      f[e] = neg_inf();
      if (c + e >= 0 && c + e < classes && (!MASK || mask[c + e])) f[e] = Elem<T>::load(row + c + e);
    }
  }
}

// ---- V <= 32: a thread owns a row
// CAP = classes rounded up to whole 16 bytes: only the last of the row's pieces can be cut.  A row of 20 floats is 80 bytes:
// the 16-byte loads of a wave touch 40 lines, five times over, all of them in the L1 after the first.  Four blocks a CU: with
// six, 20 classes take the same (2097152 rows, float32: 39.7 us) and 24 or 32 spill (45 -> 59, 69 -> 143 us).
template <typename T, int CAP, bool MASK>
__global__ __launch_bounds__(256, 4) void logprob_thread_rows(ScoreArgs a) {
  constexpr int VEC = Elem<T>::VEC, NV = CAP / VEC;
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows) return;
  const T* src = static_cast<const T*>(a.x) + row * a.stride;
  const uint8_t* mask = MASK ? a.allowed + row * a.allowed_stride : nullptr;
  float x[CAP];
  Piece<T, MASK> raw[NV];
#pragma unroll
  for (int v = 0; v + 1 < NV; ++v) raw[v].load(src, mask, v * VEC);
  load_tail<T, MASK>(src, mask, CAP - VEC, a.classes, x + CAP - VEC);
#pragma unroll
  for (int v = 0; v + 1 < NV; ++v) raw[v].expand(x + v * VEC);
  float top = kLowest, sum = 0.f, below = 0.f, t = 0.f;
#pragma unroll
  for (int j = 0; j < CAP; ++j) top = fmaxf(top, x[j]);
#pragma unroll
  for (int j = 0; j < CAP; ++j) {
    const float z = x[j] - top, e = fast_exp(z);
    sum += e;
    below += __builtin_amdgcn_fractf(e);
    t = fmaf(e, fmaxf(z, -200.f), t);
  }
  const RowOut o = row_out(stat_of(top, sum, below, t));
  write_row<T>(a, row, o);
  if (a.top_k == 0) return;
  int32_t* ids = a.top_ids + row * a.top_k;
  float* tops = a.top_logprobs + row * a.top_k;
  if (a.top_k <= 4 && !o.bad) {
    // up to four alternatives: the four largest values by insertion (a maximum and three medians an element), their indices
    // by comparison, downwards so that the lowest stays; equal values among them take the rounds below
    float b[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()};
#pragma unroll
    for (int j = 0; j < CAP; ++j) {
      b[3] = __builtin_amdgcn_fmed3f(b[2], b[3], x[j]);
      b[2] = __builtin_amdgcn_fmed3f(b[1], b[2], x[j]);
      b[1] = __builtin_amdgcn_fmed3f(b[0], b[1], x[j]);
      b[0] = fmaxf(b[0], x[j]);
    }
    if (b[0] != b[1] && b[1] != b[2] && b[2] != b[3]) {      // (-inf, -inf: fewer than four classes, the rounds too)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (k >= a.top_k) break;
        int id = -1;
#pragma unroll
        for (int j = CAP - 1; j >= 0; --j) id = x[j] == b[k] ? j : id;
        ids[k] = b[k] == neg_inf() ? -1 : id;
        tops[k] = row_logprob(o, b[k]);
      }
      return;
    }
  }
  for (int k = 0; k < a.top_k; ++k) {
    float best = neg_inf();
    int id = -1;
#pragma unroll
    for (int j = 0; j < CAP; ++j) {     // ascending and strict: the lowest index among equals
      const bool g = x[j] > best;
      best = g ? x[j] : best;
      id = g ? j : id;
    }
#pragma unroll
    for (int j = 0; j < CAP; ++j) x[j] = j == id ? neg_inf() : x[j];
    ids[k] = o.bad ? -1 : id;
    tops[k] = row_logprob(o, best);
  }
}

// A class as one 64-bit key: the float mapped to an unsigned of the same order above the complement of the index, so one
// comparison decides value first and lowest index among equals; 0 is no entry.
typedef unsigned long long Key;
__device__ __forceinline__ Key make_key(float x, int idx) {
  const uint32_t u = __float_as_uint(x + 0.0f);       // -0 and +0 are equal: one key
  const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((Key)o << 32) | (uint32_t)~(uint32_t)idx;
}
__device__ __forceinline__ float key_value(Key k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ int key_index(Key k) { return (int)~(uint32_t)k; }

// ---- V <= 2048: G lanes own a row
template <int G> __device__ __forceinline__ float group_max(float v) {
  return group_reduce<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int G> __device__ __forceinline__ float group_sum(float v) {
  return group_reduce<G>(v, [](float a, float b) { return a + b; });
}

template <typename T, int G, bool MASK>
__global__ __launch_bounds__(256) void logprob_group_rows(ScoreArgs a) {
  constexpr int VEC = Elem<T>::VEC, NV = 32 / VEC;
  const int g = threadIdx.x & (G - 1);
  const int64_t row0 = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const bool live = row0 < a.rows;
  const int64_t row = live ? row0 : a.rows - 1;      // lanes behind the last row repeat it and write nothing
  const T* src = static_cast<const T*>(a.x) + row * a.stride;
  const uint8_t* mask = MASK ? a.allowed + row * a.allowed_stride : nullptr;
  const int nv = (a.classes + G * VEC - 1) / (G * VEC);   // uniform
  float x[NV][VEC];
  float bv = neg_inf();      // this lane's largest element that is left, and its index
  int bi = 0x7fffffff;
  Piece<T, MASK> raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v)      // stretches that lie inside the row for all lanes: a uniform test, all loads in flight
    if ((v + 1) * G * VEC <= a.classes) raw[v].load(src, mask, (v * G + g) * VEC);
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if ((v + 1) * G * VEC <= a.classes) raw[v].expand(x[v]);
    else if (v < nv) load_tail<T, MASK>(src, mask, (v * G + g) * VEC, a.classes, x[v]);
  }
  if (a.top_k) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (v < nv) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const bool b = x[v][e] > bv;
          bv = b ? x[v][e] : bv;
          bi = b ? (v * G + g) * VEC + e : bi;
        }
      }
    }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (v < nv) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) bv = fmaxf(bv, x[v][e]);
      }
    }
  }
  const float top = group_max<G>(fmaxf(bv, kLowest));
  float sum = 0.f, below = 0.f, t = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (v < nv) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float z = x[v][e] - top, f = fast_exp(z);
        sum += f;
        below += __builtin_amdgcn_fractf(f);
        t = fmaf(f, fmaxf(z, -200.f), t);
      }
    }
  }
  const RowOut o = row_out(stat_of(top, group_sum<G>(sum), group_sum<G>(below), group_sum<G>(t)));
  if (g == 0 && live) write_row<T>(a, row, o);
  for (int k = 0; k < a.top_k; ++k) {
    // value first, then the lowest index: one key (-0 counts as 0)
    const Key win = group_reduce<G>(bi == 0x7fffffff ? (Key)0 : make_key(bv, bi), [](Key a, Key b) { return a > b ? a : b; });
    const float best = win ? key_value(win) : neg_inf();
    const int id = win ? key_index(win) : 0x7fffffff;
    const bool none = best == neg_inf();
    if (g == 0 && live) {
      a.top_ids[row * a.top_k + k] = none || o.bad ? -1 : id;
      a.top_logprobs[row * a.top_k + k] = row_logprob(o, best);
    }
    if (bi == id) {      // the winner's lane looks for its next one: after (best, id) in the order value down, index up
      bv = neg_inf();
      bi = 0x7fffffff;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (v < nv) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int i = (v * G + g) * VEC + e;
            const bool b = (x[v][e] < best || (x[v][e] == best && i > id)) && x[v][e] > bv;
            bv = b ? x[v][e] : bv;
            bi = b ? i : bi;
          }
        }
      }
    }
  }
}

// ---- longer rows: waves stream pieces of 2048 elements.  A wave's top list is one key per lane, sorted downwards.
// lane `src` (uniform)
__device__ __forceinline__ float read_lane(float v, int src) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), src));
}
__device__ __forceinline__ Key read_lane(Key k, int src) {
  return ((Key)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), src) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, src);
}
// the next float above a finite one (NaN and infinities do not get here)
__device__ __forceinline__ float next_above(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  return __uint_as_float((u & 0x80000000u) ? u - 1 : u + 1);
}

// one step of a bitonic network: lane and lane ^ D keep the larger and the smaller; `up` lanes keep the smaller of a pair's
// lower lane
template <int D, typename V> __device__ __forceinline__ V bitonic_step(V v, int lane, bool up) {
  const V o = lane_xor<D>(v);
  const bool want_max = !(lane & D) != up;
  return ((o > v) == want_max) ? o : v;
}
template <int D, typename V> __device__ __forceinline__ V bitonic_tail(V v, int lane, bool up) {      // steps D, D / 2, ... 1
  v = bitonic_step<D>(v, lane, up);
  if constexpr (D > 1) v = bitonic_tail<D / 2>(v, lane, up);
  return v;
}
// 64 values of a wave that rise and then fall (or any rotation): sorted downwards
template <typename V> __device__ __forceinline__ V bitonic_clean(V v, int lane) { return bitonic_tail<32>(v, lane, false); }
template <bool UP, typename V> __device__ __forceinline__ V bitonic_sort(V v, int lane) {
  v = bitonic_tail<1>(v, lane, !(lane & 2) == UP);
  v = bitonic_tail<2>(v, lane, !(lane & 4) == UP);
  v = bitonic_tail<4>(v, lane, !(lane & 8) == UP);
  v = bitonic_tail<8>(v, lane, !(lane & 16) == UP);
  v = bitonic_tail<16>(v, lane, !(lane & 32) == UP);
  return bitonic_tail<32>(v, lane, UP);
}
// the 64 largest of two lists sorted downwards: the second is given reversed
__device__ __forceinline__ Key merge_lists(Key a, Key b_reversed, int lane) {
  return bitonic_clean(a > b_reversed ? a : b_reversed, lane);
}

// The statistics of G lanes together, in all of them.  The groups of a wave hold the same.  The first lane with the maximum keeps
// its term apart, the others' terms are summed.
template <int G> __device__ __forceinline__ Stat join(const Stat& st) {
  const float m = group_max<G>(st.m), d = fmaxf(st.m - m, -200.f), f = fast_exp(d), all = st.one + st.s;
  const bool keeps = __builtin_ctzll(__ballot(st.m == m)) == (int)(threadIdx.x & (G - 1));
  return Stat{m, group_sum<G>(keeps ? st.one : 0.f), group_sum<G>(keeps ? st.s : all * f), group_sum<G>(f * fmaf(d, all, st.t))};
}

// a block's statistics and list in the workspace: [row * segs + seg]
struct ScorePart { float m, one, s, t; };

template <typename T, int NW, bool TOP, bool MASK>
__global__ __launch_bounds__(NW * 64) void logprob_wave_rows(ScoreArgs a) {
  constexpr int VEC = Elem<T>::VEC, NV = 32 / VEC, PIECE = 64 * 32;
  __shared__ Key cand[TOP ? NW : 1][128];
  __shared__ Key lists[TOP ? NW : 1][64];
  __shared__ Stat stats[NW];
  __shared__ float seen[NW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = blockIdx.x / (unsigned)a.segs;
  const int seg = (int)(blockIdx.x % (unsigned)a.segs);
  const T* src = static_cast<const T*>(a.x) + row * a.stride;
  const uint8_t* mask = MASK ? a.allowed + row * a.allowed_stride : nullptr;
  // pieces begin at multiples of 16 bytes, `pad` elements before the row's first: rows of an odd length read at the rate of
  // the others (4096 x 50001 bf16 without a top list, when it was built: 93 us unaligned, 78 aligned)
  const int pad = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
  const int pieces = (int)(((int64_t)a.classes + pad + PIECE - 1) / PIECE);
  const int p0 = (int)((int64_t)pieces * seg / a.segs), p1 = (int)((int64_t)pieces * (seg + 1) / a.segs);

  // the wave's maximum (uniform), whether a term of it is apart, and each lane's sums relative to it
  float top = kLowest, one = 0.f, sum = 0.f, sum_t = 0.f, lost = 0.f, lost_t = 0.f;
  Key list = 0;
  // An element is offered to the list when it is at least thr.  A wave that has seen top_k elements of at least b takes the
  // next float above b: its later pieces hold higher indices, an equal value stays behind.  The other waves' b hold as they
  // are; they are read from LDS without a barrier, an old value only offers more.
  float thr = kLowest;
  if (TOP && NW > 1 && lane == 0) seen[wave] = kLowest;
  if (TOP && NW > 1) __syncthreads();
  auto raise = [&](float b) {
    const float t = next_above(b);
    if (t > thr) {
      thr = t;
      if (NW > 1 && lane == 0) *const_cast<volatile float*>(&seen[wave]) = b;
    }
  };
  int n = 0;                  // candidates waiting in cand[wave]

  auto flush = [&](int count) {   // the first 64 (count of them valid) into the list
    wave_lds_fence();
    const Key k = lane < count ? cand[wave][lane] : 0;
    const Key rest = cand[wave][64 + lane];
    list = merge_lists(list, bitonic_sort<true>(k, lane), lane);
    wave_lds_fence();
    cand[wave][lane] = rest;
    const Key kth = read_lane(list, a.top_k - 1);
    if (kth) raise(key_value(kth));
  };

  // whole pieces are requested one ahead: the next one's loads are in flight while this one is worked on
  const int first = pad ? 1 : 0, past = (a.classes + pad) / PIECE;
  auto whole = [&](int p) { return p >= first && p < past && p < p1; };
  Piece<T, MASK> raw[NV];
  auto request = [&](int p) {
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v].load(src, mask, (int64_t)p * PIECE - pad + (v * 64 + lane) * VEC);
  };
  if (whole(p0 + wave)) request(p0 + wave);
  for (int p = p0 + wave; p < p1; p += NW) {
    float x[NV][VEC];
    const int base = p * PIECE - pad;
    if (whole(p)) {
#pragma unroll
      for (int v = 0; v < NV; ++v) raw[v].expand(x[v]);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) load_tail<T, MASK>(src, mask, base + (v * 64 + lane) * VEC, a.classes, x[v]);
    }
    if (whole(p + NW)) request(p + NW);
    float vec_max[NV], lane_max = neg_inf();
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      vec_max[v] = x[v][0];
#pragma unroll
      for (int e = 1; e < VEC; ++e) vec_max[v] = fmaxf(vec_max[v], x[v][e]);
      lane_max = fmaxf(lane_max, vec_max[v]);
    }
    // A new maximum (about 4 of 25 pieces of a row in no order): what there was is taken relative to it, and its own term, in the
    // first lane that holds it and there in the first 16 bytes, is kept out of that lane's sum (+inf stays in and makes it NaN)
    int apart = -1;
    bool keeps = false;
    if (__ballot(lane_max > top)) {
      const float m = group_max<64>(lane_max), d = fmaxf(top - m, -200.f), f = fast_exp(d), all = sum + (lane == 0 ? one : 0.f);
      sum_t = f * fmaf(d, all, sum_t);
      lost_t = f * fmaf(d, lost, lost_t);
      sum = f * all;
      lost *= f;
      top = m;
      one = 1.f;
      keeps = m < __builtin_inff() && __builtin_ctzll(__ballot(lane_max == m)) == lane;
#pragma unroll
      for (int v = NV - 1; v >= 0; --v) apart = __ballot(keeps && vec_max[v] == m) ? v : apart;
    }
    uint32_t offers = 0;      // bit v VEC + e: the element is offered to the list
    float least = thr, bound = kLowest;
    bool some = false;
    if constexpr (TOP) {
      // at least top_k elements of this piece are not below the top_k-th largest of the lanes' maxima: a bound that keeps
      // the first piece from offering all of its elements, and a rising row from offering all of every piece
      if constexpr (NW > 1) {
#pragma unroll
        for (int w = 0; w < NW; ++w) least = fmaxf(least, *const_cast<volatile float*>(&seen[w]));
      }
      const Key over = __ballot(lane_max >= least);
      if (over) {
        some = true;
        if (__popcll(over) >= a.top_k) {
          bound = read_lane(bitonic_sort<false>(lane_max, lane), a.top_k - 1);
          least = fmaxf(least, bound);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          if (__ballot(vec_max[v] >= least)) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) offers |= x[v][e] >= least ? 1u << (v * VEC + e) : 0u;
          }
        }
      }
    }
    float s = 0.f, t = 0.f;
    const float out = keeps ? top : __builtin_nanf("");
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (v == apart) {      // uniform; equal elements of the 16 bytes go together, all but one come back as terms of 1
        s = keeps ? -1.f : 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          s += x[v][e] == out ? 1.f : 0.f;
          x[v][e] = x[v][e] == out ? neg_inf() : x[v][e];
        }
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float z = x[v][e] - top, p = fast_exp(z);
        s += p;
        t = fmaf(p, fmaxf(z, -200.f), t);
      }
      __builtin_amdgcn_sched_barrier(0);      // 8 exponentials in flight at a time: more would only cost registers, and waves
    }
    add_carried(sum, lost, s);
    add_carried(sum_t, lost_t, t);
    if constexpr (TOP) {
      if (some) {
        // a lane's only offer is its maximum; several are read again (a register cannot be chosen by a lane)
        const bool several = offers & (offers - 1);
        for (Key who = __ballot(offers != 0); who; who = __ballot(offers != 0)) {      // one element of every lane that has one
          if (offers) {
            const int bit = __builtin_ctz(offers);
            const int idx = base + ((bit / VEC) * 64 + lane) * VEC + bit % VEC;
            float f = lane_max;
            if (several) f = Elem<T>::load(src + idx);
            offers &= offers - 1;
            cand[wave][n + __popcll(who & ((1ull << lane) - 1))] = make_key(f, idx);
          }
          n += (int)__popcll(who);
          if (n >= 64) {
            flush(64);
            n -= 64;
          }
        }
        if (bound > kLowest) raise(bound);
      }
    }
  }
  if (TOP && n) flush(n);
  Stat st{top, one, group_sum<64>(sum - lost), group_sum<64>(sum_t - lost_t)};
  if (lane == 0) stats[wave] = st;
  if constexpr (TOP) lists[wave][lane] = list;
  __syncthreads();
  if constexpr (TOP) {
    for (int h = NW / 2; h > 0; h >>= 1) {
      if (wave < h) {
        list = merge_lists(list, lists[wave + h][63 - lane], lane);
        lists[wave][lane] = list;
      }
      __syncthreads();
    }
  }
  if (wave) return;
  if constexpr (NW > 1) st = join<NW>(stats[lane & (NW - 1)]);
  if (a.segs > 1) {
    ScorePart* part = static_cast<ScorePart*>(a.part);
    const int64_t slot = row * a.segs + seg;
    if (lane == 0) part[slot] = ScorePart{st.m, st.one, st.s, st.t};
    if constexpr (TOP) reinterpret_cast<Key*>(part + a.rows * a.segs)[slot * 64 + lane] = list;
    return;
  }
  const RowOut o = row_out(st);
  if (lane == 0) write_row<T>(a, row, o);
  if (TOP && lane < a.top_k) {
    a.top_ids[row * a.top_k + lane] = list == 0 || o.bad ? -1 : key_index(list);
    a.top_logprobs[row * a.top_k + lane] = row_logprob(o, list == 0 ? neg_inf() : key_value(list));
  }
}

// joins what the blocks of a row found: one block a row, four waves
template <typename T, bool TOP>
__global__ __launch_bounds__(256) void logprob_join(ScoreArgs a) {
  __shared__ Key lists[TOP ? 4 : 1][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const ScorePart* part = static_cast<const ScorePart*>(a.part) + row * a.segs;
  Key list = 0;
  if constexpr (TOP) {
    const Key* keys = reinterpret_cast<const Key*>(static_cast<const ScorePart*>(a.part) + a.rows * a.segs) + row * a.segs * 64;
    for (int s = wave; s < a.segs; s += 4) list = merge_lists(list, keys[s * 64 + 63 - lane], lane);
    lists[wave][lane] = list;
    __syncthreads();
    if (wave < 2) lists[wave][lane] = list = merge_lists(list, lists[wave + 2][63 - lane], lane);
    __syncthreads();
    if (wave == 0) list = merge_lists(list, lists[1][63 - lane], lane);
  }
  if (wave) return;
  Stat st{kLowest, 0.f, 0.f, 0.f};
  if (lane < a.segs) st = Stat{part[lane].m, part[lane].one, part[lane].s, part[lane].t};      // up to 64
  st = join<64>(st);
  const RowOut o = row_out(st);
  if (lane == 0) write_row<T>(a, row, o);
  if (TOP && lane < a.top_k) {
    a.top_ids[row * a.top_k + lane] = list == 0 || o.bad ? -1 : key_index(list);
    a.top_logprobs[row * a.top_k + lane] = row_logprob(o, list == 0 ? neg_inf() : key_value(list));
  }
}

// ---- gradient
// With p_j = e^(x_j - lse) (0 where not allowed), H the row's entropy, gl / ge / gt the gradients that arrive:
//   d loss / d x_j = G_j (1 - p_j) - p_j (W - G_j) - ge p_j (x_j - lse + H),
//   G_j = gl [j = label] + sum_i gt_i [j = id_i],  W = gl + sum_i gt_i
// 1 - p of a named class is taken from z = ln p without the difference.  z = x - lse is known to the rounding of lse, 2^-24 |lse|,
// which is all of 1 - p for a class that has nearly everything; a name that brings the log probability of the forward pass
// (relative to 2^-24) has that as its z and keeps its bits.
// One read of the logits and one write of the gradient.  A block owns whole rows, or a piece of one; the classes that its
// rows' labels and alternatives name, and what arrives for them, are put into LDS first, and every 16-byte piece is compared
// with its row's names while it is in registers: no element is written twice, equal names add up.
struct GradArgs {
  const void* x;
  int64_t rows, stride;
  int classes;
  const void* labels;
  int label64;
  const uint8_t* allowed;
  int64_t allowed_stride;
  const float *lse, *entropy, *d_logprob, *d_entropy;   // all but lse may be NULL; labels NULL: the label is no name
  const int32_t* top_ids;
  const float* d_top;
  int top_k;                                            // 0: the alternatives are no names
  const float *logprob, *top_logprobs;                  // ln p of the names, or NULL
  void* grad;
  int64_t grad_stride;
  // a block: 16-byte pieces of rows_per_block rows (vecs each), or vecs pieces of one row that takes `cuts` blocks
  int rows_per_block, vecs, cuts;
  uint32_t magic;      // ceil(2^20 / vecs): i / vecs = i magic >> 20 for i < 1024, vecs <= 1024
};

struct GradRow { float lse, w, ge, h; };   // w = gl + sum gt; empty rows have all of them 0

// 1 - e^z: the series of e^z - 1 where the difference would cancel (7 terms: 0.35^7 / 8! < 2^-25), the difference elsewhere
__device__ __forceinline__ float one_minus_exp(float z) {
  float s = 1.f / 5040.f;
  s = fmaf(s, z, 1.f / 720.f);
  s = fmaf(s, z, 1.f / 120.f);
  s = fmaf(s, z, 1.f / 24.f);
  s = fmaf(s, z, 1.f / 6.f);
  s = fmaf(s, z, 0.5f);
  s = fmaf(s, z, 1.f);
  return z > -0.35f ? -z * s : 1.f - fast_exp(z);
}
__device__ __forceinline__ float grad_dense(const GradRow& r, float w, float z) {
  const float p = fast_exp(z);
  // an underflowed p takes the entropy term with it (0 * -inf otherwise)
  return -p * fmaf(r.ge, fmaxf(z, -200.f) + r.h, w);
}

constexpr int kGradNames = 1024;      // names a block holds

// NI 16-byte pieces a thread, requested before the names are looked up
template <typename T, bool MASK, int NI>
__global__ __launch_bounds__(256) void logprob_grad(GradArgs a) {
  constexpr int VEC = Elem<T>::VEC;
  __shared__ GradRow prm[256];
  __shared__ int ids[kGradNames];
  __shared__ float gs[kGradNames];
  __shared__ float zs[kGradNames];      // ln p of a name, 1: not given
  const int64_t row0 = a.cuts > 1 ? (int64_t)(blockIdx.x / (unsigned)a.cuts) : (int64_t)blockIdx.x * a.rows_per_block;
  // the pieces of a long row begin at multiples of 16 bytes of the gradient, up to VEC - 1 elements before its first
  const int pad = a.cuts > 1 ? (int)((reinterpret_cast<uintptr_t>(static_cast<T*>(a.grad) + row0 * a.grad_stride) & 15) / sizeof(T)) : 0;
  const int c0 = a.cuts > 1 ? (int)(blockIdx.x % (unsigned)a.cuts) * a.vecs * VEC - pad : 0;
  const int c1 = a.cuts > 1 && a.classes - c0 > a.vecs * VEC ? c0 + a.vecs * VEC : a.classes;
  const int nr = a.cuts > 1 ? 1 : (int)(a.rows - row0 < a.rows_per_block ? a.rows - row0 : a.rows_per_block);
  const int names = a.top_k + (a.labels ? 1 : 0);
  const bool kept = a.logprob || a.top_logprobs;
  int rr[NI], cc[NI];
  Piece<T, MASK> raw[NI];
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int i = n * 256 + threadIdx.x;
    rr[n] = (int)(((uint32_t)i * a.magic) >> 20);
    cc[n] = c0 + (i - rr[n] * a.vecs) * VEC;
    if (rr[n] < nr && cc[n] >= 0 && cc[n] + VEC <= c1)
      raw[n].load(static_cast<const T*>(a.x) + (row0 + rr[n]) * a.stride,
                  MASK ? a.allowed + (row0 + rr[n]) * a.allowed_stride : nullptr, cc[n]);
  }
  for (int i = threadIdx.x; i < nr * names; i += 256) {
    const int r = i / names, n = i - r * names;
    const int64_t row = row0 + r;
    int64_t id;
    float g = 0.f, z = 1.f;
    if (n < a.top_k) {
      const int64_t at = row * a.top_k + n;
      id = a.top_ids[at];
      if (a.d_top) g = a.d_top[at];
      if (a.top_logprobs) z = a.top_logprobs[at];
    } else {
      id = a.label64 ? static_cast<const int64_t*>(a.labels)[row] : static_cast<const int32_t*>(a.labels)[row];
      if (a.d_logprob) g = a.d_logprob[row];
      if (a.logprob) z = a.logprob[row];
    }
    const bool known = id >= 0 && id < a.classes;
    ids[i] = known ? (int)id : -1;
    gs[i] = known ? g : 0.f;
    if (kept) zs[i] = z;
  }
  GradRow mine{0.f, 0.f, 0.f, 0.f};
  if ((int)threadIdx.x < nr) {
    const int64_t row = row0 + threadIdx.x;
    mine.lse = a.lse[row];
    if (a.d_entropy) {
      mine.ge = a.d_entropy[row];
      mine.h = a.entropy[row];
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < nr) {
    const int n0 = threadIdx.x * names;
    const bool empty = mine.lse == neg_inf();      // nothing is allowed: the row's gradient is 0
    if (empty) mine = GradRow{0.f, 0.f, 0.f, 0.f};
    for (int n = n0; n < n0 + names; ++n) {
      if (empty) ids[n] = -1;
      else mine.w += gs[n];
    }
    prm[threadIdx.x] = mine;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NI; ++n) {
    const int r = rr[n], c = cc[n];
    if (r >= nr || c >= c1) continue;
    const GradRow p = prm[r];
    float x[VEC], f[VEC];
    const bool inside = c >= 0 && c + VEC <= c1;
    if (inside) raw[n].expand(x);
    else load_tail<T, MASK>(static_cast<const T*>(a.x) + (row0 + r) * a.stride,
                            MASK ? a.allowed + (row0 + r) * a.allowed_stride : nullptr, c, c1, x);
    float z[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      f[e] = 0.f;      // G_j first
      z[e] = x[e] - p.lse;
    }
    bool named = false;
    for (int k = r * names; k < (r + 1) * names; ++k) {
      const int d = ids[k] - c;
      if ((unsigned)d < (unsigned)VEC) {
        named = true;
        const float g = gs[k];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] += e == d ? g : 0.f;
        if (kept) {
          const float zk = zs[k];
#pragma unroll
          for (int e = 0; e < VEC; ++e) z[e] = e == d && zk <= 0.f ? zk : z[e];
        }
      }
    }
    if (named) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = fmaf(f[e], one_minus_exp(z[e]), grad_dense(p, p.w - f[e], z[e]));
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = grad_dense(p, p.w, z[e]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = x[e] == neg_inf() ? 0.f : f[e];
    T* dst = static_cast<T*>(a.grad) + (row0 + r) * a.grad_stride + c;
    if (inside) {
      stream16(dst, pack16<T>(f));
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (c + e >= 0 && c + e < c1) dst[e] = Elem<T>::from(f[e]);
    }
  }
}

}  // namespace pclseg

#endif  // PCLSEG_SCORE_H_
