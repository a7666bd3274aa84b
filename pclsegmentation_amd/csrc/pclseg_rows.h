// pclseg_rows.h — what the row operators (pclseg_score.h, pclseg_i8.h) share: element types, 16-byte accesses at any
// element alignment, lane exchanges.  gfx950, 64-lane waves.
#ifndef PCLSEG_ROWS_H_
#define PCLSEG_ROWS_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pclseg {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// the hardware takes a global access of any size at any 2-byte (16-bit types) or 4-byte (float) address: rows of an odd
// length need no other path, a 16-byte access that crosses a 128-byte line only costs a second tag look-up
typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2a2 __attribute__((ext_vector_type(2), aligned(2)));
struct __attribute__((packed, aligned(1))) Pack8a1 { uint64_t v; };
struct __attribute__((packed, aligned(1))) Pack4a1 { uint32_t v; };

template <typename T> struct Elem;
template <> struct Elem<float> {
  typedef u32x4a4 Pack;
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float get(const u32x4& v, int e) { return __uint_as_float(v[e]); }
  static __device__ __forceinline__ float load(const float* p) { return *p; }
  static __device__ __forceinline__ float from(float f) { return f; }
};
template <> struct Elem<__bf16> {
  typedef u32x4a2 Pack;
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(const u32x4& v, int e) {
    return __uint_as_float((e & 1) ? (v[e >> 1] & 0xffff0000u) : (v[e >> 1] << 16));
  }
  static __device__ __forceinline__ float load(const __bf16* p) { return (float)*p; }
  static __device__ __forceinline__ __bf16 from(float f) { return (__bf16)f; }   // nearest, ties to even
};
template <> struct Elem<_Float16> {
  typedef u32x4a2 Pack;
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(const u32x4& v, int e) {
    const uint32_t w = v[e >> 1];
    return (float)__builtin_bit_cast(_Float16, (uint16_t)((e & 1) ? (w >> 16) : (w & 0xffffu)));
  }
  static __device__ __forceinline__ float load(const _Float16* p) { return (float)*p; }
  static __device__ __forceinline__ _Float16 from(float f) { return (_Float16)f; }
};

// 16 bytes at element p (any element alignment)
template <typename T> __device__ __forceinline__ u32x4 load16(const T* p) {
  return *reinterpret_cast<const typename Elem<T>::Pack*>(p);
}
// Outputs that are written once and read by a later kernel pass the caches by: the lines they would push out are worth more
// than those a reader would find (ten passes of the same inputs in a graph: 131072x512 -> 1024 float32 with its
// quantisation 271 -> 205 us, a layer, its log probabilities and their gradient 553 -> 505 us; also where the output would fit:
// 8192x1024 -> 2048 bf16 34.7 -> 33.4 us.  The gradient of 4096x50001 bf16 by itself loses by it, 156 -> 160 us).
template <typename T> __device__ __forceinline__ void stream16(T* p, const u32x4& v) {
  typedef typename Elem<T>::Pack Pack;
  __builtin_nontemporal_store((Pack)v, reinterpret_cast<Pack*>(p));
}
template <typename T> __device__ __forceinline__ u32x4 pack16(const float* f) {
  u32x4 v;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(f[e]);
  } else {
    typedef T T2 __attribute__((ext_vector_type(2)));
    typedef float F2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(F2{f[2 * e], f[2 * e + 1]}, T2));
  }
  return v;
}

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// LDS traffic inside one wave is in order in the hardware; this keeps the compiler from reordering it
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The value of lane ^ D, in the vector pipe alone (DPP within rows of 16 lanes, row swaps beyond): a step of a reduction or
// of a sort takes tens of cycles, an exchange through the LDS crossbar more than a hundred.
template <int D> __device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  static_assert(D == 1 || D == 2 || D == 4 || D == 8 || D == 16 || D == 32, "a power of two below 64");
  if constexpr (D == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);        // quad_perm 1,0,3,2
  else if constexpr (D == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);   // quad_perm 2,3,0,1
  else if constexpr (D == 4) {      // ^ 7 (row_half_mirror), then ^ 3 (quad_perm 3,2,1,0)
    const int h = __builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true);
    return (uint32_t)__builtin_amdgcn_mov_dpp(h, 0x1B, 0xF, 0xF, true);
  } else if constexpr (D == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, true);   // row_ror 8
  else if constexpr (D == 16) {      // rows 0 0 2 2 and 1 1 3 3
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (threadIdx.x & 16) ? s[0] : s[1];
  } else {
    const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? s[0] : s[1];
  }
}
template <int D> __device__ __forceinline__ float lane_xor(float v) { return __uint_as_float(lane_xor<D>(__float_as_uint(v))); }
template <int D> __device__ __forceinline__ int lane_xor(int v) { return (int)lane_xor<D>((uint32_t)v); }
template <int D> __device__ __forceinline__ unsigned long long lane_xor(unsigned long long v) {
  return ((unsigned long long)lane_xor<D>((uint32_t)(v >> 32)) << 32) | lane_xor<D>((uint32_t)v);
}
// f(partner's value) over the lanes of a group of G
template <int G, typename V, typename F> __device__ __forceinline__ V group_reduce(V v, F f) {
  if constexpr (G > 1) v = f(v, lane_xor<1>(v));
  if constexpr (G > 2) v = f(v, lane_xor<2>(v));
  if constexpr (G > 4) v = f(v, lane_xor<4>(v));
  if constexpr (G > 8) v = f(v, lane_xor<8>(v));
  if constexpr (G > 16) v = f(v, lane_xor<16>(v));
  if constexpr (G > 32) v = f(v, lane_xor<32>(v));
  return v;
}

// Blocks are dealt round robin over the 8 XCDs: give each XCD one contiguous range of tiles, so neighbours share an L2.
// A bijection of [0, total) for every total.
__device__ __forceinline__ unsigned xcd_contiguous(unsigned block, unsigned total) {
  const unsigned q = total >> 3, r = total & 7, x = block & 7, i = block >> 3;
  return x * q + (x < r ? x : r) + i;
}

}  // namespace pclseg

#endif  // PCLSEG_ROWS_H_
