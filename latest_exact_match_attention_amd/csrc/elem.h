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

// A grid of n workgroups or more, and a workgroup's index in it: a dimension takes fewer than 2^32
// threads, which rows of a few elements reach within the memory there is.
inline dim3 blocks_of(int64_t n) {
  const int64_t x = n < (1 << 21) ? n : 1 << 21;
  return dim3(static_cast<uint32_t>(x), static_cast<uint32_t>((n + x - 1) / x));
}
__device__ __forceinline__ int64_t block_index() {
  return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
}

template <typename T>
constexpr int kPiece = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte piece

// A 16-byte piece as its elements.
template <typename T>
union Piece {
  u32x4 raw;
  T e[kPiece<T>];
};

// 16 bytes of elements from or to memory, past the caches where kStream is set. The address may be any
// element's: gfx950 takes vector accesses at any alignment, by the same instructions.
template <typename T>
struct Unaligned;
template <>
struct Unaligned<float> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Unaligned<_Float16> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Unaligned<Bf16> : Unaligned<_Float16> {};

template <bool kStream = false, typename T>
__device__ __forceinline__ u32x4 get16(const T* p) {
  const auto* at = reinterpret_cast<const typename Unaligned<T>::type*>(p);
  if constexpr (kStream) return __builtin_nontemporal_load(at);
  return *at;
}
template <bool kStream = false, typename T>
__device__ __forceinline__ void put16(T* p, u32x4 v) {
  auto* at = reinterpret_cast<typename Unaligned<T>::type*>(p);
  if constexpr (kStream)
    __builtin_nontemporal_store(static_cast<typename Unaligned<T>::type>(v), at);
  else
    *at = v;
}

// How rows of D elements are read and written.
//   kWholeRows   16-byte pieces, D a multiple of 8.
//   kRaggedRows  16-bit types, D >= 8: pieces too. What would reach past the row is read as the row's
//                last whole piece instead and shifted into place once it is used, so that no load is
//                conditional: a branch around the last one made the kernels wait for every load where
//                it was issued (the gradient of 65,536 norms of 1535 in bf16: 489 us, 218 so).
//   kElements    element by element: fp32 rows, where 64 lanes' elements are whole lines anyway
//                and pieces that straddle lines cost more (18 us for the gradient of 4099 layer norms of
//                1001, 14 so), and rows shorter than a piece.
enum RowKind { kElements, kRaggedRows, kWholeRows };

inline RowKind row_kind(int32_t dtype, int64_t D) {
  return D % 8 == 0 ? kWholeRows : dtype == LEMA_F32 || D < 8 ? kElements : kRaggedRows;
}

// Calls f with the kind as a compile-time constant; fp32 rows are not ragged.
template <typename T, typename F>
inline void for_kind(RowKind kind, F f) {
  using std::integral_constant;
  if (kind == kWholeRows)
    f(integral_constant<int, kWholeRows>{});
  else if (kind == kElements || sizeof(T) == 4)
    f(integral_constant<int, kElements>{});
  else
    f(integral_constant<int, sizeof(T) == 4 ? kElements : kRaggedRows>{});
}

template <typename T, int kKind>
constexpr int kUnit = kKind == kElements ? 1 : kPiece<T>;

// N elements of a row, as they come from memory, in units of kUnit at the places at(i) of its elements
// i (multiples of the unit): all lanes fetch, settle before they look, and store.
template <typename T, int kKind, int N>
struct RowPart {
  static constexpr int n = kUnit<T, kKind>, kPerPiece = kPiece<T>;
  Piece<T> q[N / kPerPiece];

  template <bool kStream, typename At>
  __device__ __forceinline__ void fetch(const T* row, int64_t D, At at) {
#pragma unroll
    for (int i = 0; i < N; i += n) {
      const auto e = at(i);
      if constexpr (kKind == kElements)
        q[i / kPerPiece].e[i % kPerPiece] = e < D ? row[e] : T{};
      else if constexpr (kKind == kWholeRows)
        q[i / n].raw = e < D ? get16<kStream>(row + e) : u32x4{0, 0, 0, 0};
      else
        q[i / n].raw = get16<kStream>(row + (e < D - n ? e : D - n));
    }
  }
  template <typename At>
  __device__ __forceinline__ void settle(int64_t D, At at) {
    if constexpr (kKind == kRaggedRows) {
#pragma unroll
      for (int i = 0; i < N; i += n) {
        const int64_t past = at(i) - (D - n);  // elements to shift out
        const int s = past <= 0 ? 0 : past >= n ? 128 : static_cast<int>(past) * 16;
        u32x4& v = q[i / n].raw;
        const uint64_t lo = static_cast<uint64_t>(v.y) << 32 | v.x, hi = static_cast<uint64_t>(v.w) << 32 | v.z;
        const uint64_t top = s >= 64 ? 0 : hi >> (s & 63);
        const uint64_t low = s >= 128  ? 0
                             : s >= 64 ? hi >> (s & 63)
                             : s > 0   ? lo >> s | hi << (64 - s)
                                       : lo;
        v = u32x4{static_cast<uint32_t>(low), static_cast<uint32_t>(low >> 32), static_cast<uint32_t>(top),
                  static_cast<uint32_t>(top >> 32)};
      }
    }
  }
  template <bool kStream, typename At>
  __device__ __forceinline__ void store(T* row, int64_t D, At at) const {
#pragma unroll
    for (int i = 0; i < N; i += n) {
      const auto e = at(i);
      if constexpr (kKind == kElements) {
        if (e < D) row[e] = q[i / kPerPiece].e[i % kPerPiece];
      } else if (kKind == kWholeRows ? e < D : e + n <= D) {
        put16<kStream>(row + e, q[i / n].raw);
      } else if constexpr (kKind == kRaggedRows) {
#pragma unroll
        for (int k = 0; k < n - 1; ++k)
          if (e + k < D) row[e + k] = q[i / n].e[k];
      }
    }
  }
  __device__ __forceinline__ float get(int k) const { return to_f32(q[k / kPerPiece].e[k % kPerPiece]); }
  __device__ __forceinline__ void set(int k, float v) {
    q[k / kPerPiece].e[k % kPerPiece] = from_f32<T>(v);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < N / kPerPiece; ++i) q[i].raw = u32x4{0, 0, 0, 0};
  }
};

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
