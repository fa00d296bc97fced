// Elements of the three value types as fp32: pieces of 16 bytes, and single elements.
#pragma once
#include "lema_internal.h"

namespace lema {

struct Bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float to_f32(Bf16 v) {
  return __uint_as_float(static_cast<uint32_t>(v.bits) << 16);
}

// Round to nearest even (in bf16 gfx950's own conversion, a pair in one instruction).
template <typename T>
__device__ __forceinline__ T from_f32(float f);
template <>
__device__ __forceinline__ float from_f32<float>(float f) {
  return f;
}
template <>
__device__ __forceinline__ _Float16 from_f32<_Float16>(float f) {
  return static_cast<_Float16>(f);
}
template <>
__device__ __forceinline__ Bf16 from_f32<Bf16>(float f) {
  return Bf16{__builtin_bit_cast(uint16_t, static_cast<__bf16>(f))};
}

template <typename T>
constexpr int kPiece = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte piece

// A 16-byte piece as its elements.
template <typename T>
union Piece {
  u32x4 raw;
  T e[kPiece<T>];
};

// 16 bytes from or to memory, past the caches where kStream is set.
template <bool kStream>
__device__ __forceinline__ u32x4 get16(const void* p) {
  const u32x4* at = static_cast<const u32x4*>(p);
  if constexpr (kStream) return __builtin_nontemporal_load(at);
  return *at;
}
template <bool kStream>
__device__ __forceinline__ void put16(void* p, u32x4 v) {
  u32x4* at = static_cast<u32x4*>(p);
  if constexpr (kStream)
    __builtin_nontemporal_store(v, at);
  else
    *at = v;
}

// Calls f(T{}) with the element type of `dtype` (checked by the caller).
template <typename F>
inline void for_dtype(int32_t dtype, F f) {
  if (dtype == LEMA_F32)
    f(float{});
  else if (dtype == LEMA_F16)
    f(_Float16{});
  else
    f(Bf16{});
}

// Sum over the wavefront: every lane gets the same bits.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

}  // namespace lema
