// Device helpers of the 4-bit cache (form: serve_kernels.h).
#pragma once

#include <hip/hip_fp16.h>

#include "serve_kernels.h"

namespace msh {

// offsets of a token's bytes inside its block; t = token in the block, m = groups
__device__ inline int kv4_key_at(int t, int g, int quarter, int m) {
  const int left = m - (g & ~3), of = left < 4 ? left : 4;
  return (t >> 4) * 256 * m + (g >> 2) * 1024 + ((quarter * 16 + (t & 15)) * of + (g & 3)) * 4;
}
__device__ inline int kv4_key_scale_at(int t, int g, int m) { return 512 * m + t * m + g; }
__device__ inline int kv4_value_at(int t, int g, int pair, int m) {
  const int left = m - (g & ~1), of = left < 2 ? left : 2;
  return 544 * m + (g >> 1) * 1024 + ((((t >> 2) & 3) * 16 + pair) * of + (g & 1)) * 8 + (t >> 4) * 4 + (t & 3);
}
__device__ inline int kv4_value_scale_at(int t, int g, int m) {
  return 1056 * m + (((t >> 2) & 3) * m + g) * 8 + (t >> 4) * 4 + (t & 3);
}

__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
// the power of byte B of a word in one instruction: left to itself the compiler shifts and masks
template <int B>
__device__ __forceinline__ float kv4_scale_of(uint32_t word) {
  uint32_t r;
  if constexpr (B == 0) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(23), "v"(word));
  else if constexpr (B == 1) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(23), "v"(word));
  else if constexpr (B == 2) asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(23), "v"(word));
  else asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(23), "v"(word));
  return __uint_as_float(r);
}

template <int BYTE>
__device__ __forceinline__ uint32_t kv4_pair_bf16(uint32_t codes, float scale) {   // exact: one significant bit, a power of two
  const auto v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <Elem E>
struct ElemOf;
template <>
struct ElemOf<Elem::f32> {
  typedef float T;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct ElemOf<Elem::bf16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(uint16_t x) { return bf16_to_f32(x); }
  static __device__ __forceinline__ uint16_t put(float x) { return (uint16_t)pack_bf16x2(x, 0.f); }
};
template <>
struct ElemOf<Elem::f16> {
  typedef uint16_t T;
  static __device__ __forceinline__ float get(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ uint16_t put(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};

// p aligned to N elements' size where ALIGNED
template <Elem E, int N>
__device__ __forceinline__ void load_elems(const typename ElemOf<E>::T* p, float* out) {
  typedef typename ElemOf<E>::T T;
  struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack { T v[N]; };
  const Pack x = *reinterpret_cast<const Pack*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = ElemOf<E>::get(x.v[i]);
}
template <Elem E, int N>
__device__ __forceinline__ void store_elems(typename ElemOf<E>::T* p, const float* in) {
  typedef typename ElemOf<E>::T T;
  struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack { T v[N]; } x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = ElemOf<E>::put(in[i]);
  *reinterpret_cast<Pack*>(p) = x;
}

}  // namespace msh
