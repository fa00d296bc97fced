// The matrix product behind gated.hip and fp8.hip: out = A . B over tiles in LDS, on the matrix
// cores, with an epilogue on the fp32 sums.
//
// An operand is K-major (rows along the sum: x and W of x . W^T) or M-major (rows across it, for the
// products of a backward: W of dg . W, both of dg^T . x). Either way a stage of a tile, 64 bytes of
// the sum deep, goes from memory to LDS as it lies (buffer_load ... lds, 16 bytes a lane); a K-major
// fragment is then read with ds_read_b128 and an M-major one with ds_read_b64_tr_b16, which hands a
// lane four k of one column: no operand is transposed in memory.
//
//   K-major   row r of 64 bytes, its 16-byte chunk c in slot c ^ (r / 4 % 4)
//   M-major   k-row of the tile's columns, chunk c in slot c ^ 4 (k % 4): the four k-rows of a
//             transposed read lie 64 bytes apart in the banks
//
// (no bank conflicts by counter in either). Buffer loads return 0 past the descriptor's end, which is the
// end of the tensor: rows past M or N give sums that nobody stores, k past the end gives zeros (in a
// K-major row by an offset past the end). The offset of a lane is all in its own register: the check
// leaves out the scalar one.
//
// Workgroups walk the tiles of their XCD (consecutive in an order that takes gm row tiles across all
// column tiles), and `splits` parts of the sum where the tiles are few: their fp32 sums go to a
// workspace, and a second kernel adds them up in order.
//
// A wave multiplies one stage's fragments while it reads the next one's from LDS and sends for two stages
// of A, or of B, four and five ahead: a line of a K-major row holds both. A barrier every two stages
// says that the next two have landed and that the ones that B's replace were read by all. The
// pipeline runs on across tiles. At [65536, 1536] x 6144 the forward takes 2048 us (1.21 PFLOP/s), the
// gradient's products 1944 us (dg . W, 1.27) and 2120 us (dg^T . x, 1.17; 2324 with the splits of an earlier
// choice, which the following had). Two stages of twice the depth, with the two waves of a SIMD taking turns at
// reading and multiplying, took 2110, 2683 and 2784 us: a stage had to arrive within the time of its
// predecessor's products. Sending for one stage at a time, half a line, took 2185, 2106 and 2384; 128 x 256
// tiles, two workgroups to a CU, 2711, 2583 and 2503.
#pragma once
#include "elem.h"

namespace lema {
namespace gemm {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

struct Fp8 {
  uint8_t bits;
};

// What the sums are stored as.
enum Form : int32_t {
  kPlain,   // out = sum over segments i of A_i . B_i
  kGated,   // out = silu(A . B_0) * (A . B_1), and its derivatives where asked for
  kWeights  // out_i = A_i . B, segment after segment of the output's rows
};

struct Args {
  const uint8_t* a[2];
  const uint8_t* b[2];
  void* out[2];      // kGated: out[0]; kWeights: one of each segment
  uint8_t* slopes;       // kGated: out's derivatives (see Slopes), or null
  float* part;       // splits > 1: [splits][planes][M][N] sums
  const uint8_t* sa;     // 8 bits: scales of A, [stages][lds_a] by row
  const uint8_t* sb[2];  // of B, [blocks of 128 rows][stages]
  int64_t lda, ldb, ldo;  // row strides, a's and b's in bytes, out's in elements
  int64_t lds_a;
  int32_t M, N, K;   // of the output (a segment's rows in kWeights), and a segment's sum
  int32_t nk;        // a segment's stages
  int32_t segs;      // kPlain: segments of the sum; kWeights: of the rows
  int32_t tiles_m, tiles_n, gm, splits, per;  // per: stages of a split
};

__device__ __forceinline__ uint32_t pack2(Bf16, float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
}
__device__ __forceinline__ uint32_t pack2(_Float16, float a, float b) {
  return __builtin_bit_cast(uint32_t, f16x2_t{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}

// y = q u with q = silu(g) = g s and s = 1 / (1 + e^-g), whose derivative is s (1 + g (1 - s)) = s + q (1 - s);
// e^-g overflows to infinity at most, where s is 0. (The reciprocal is off by one step; an IEEE
// division is 10 instructions.)
__device__ __forceinline__ float silu(float g, float& s) {
  s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));
  return g * s;
}
__device__ __forceinline__ float gated_value(float g, float u) {
  float s;
  return silu(g, s) * u;
}
__device__ __forceinline__ float gate_slope(float u, float q, float s) { return u * (s + q * (1.0f - s)); }

// dy/dg and dy/du of [M, N] results, as the gradient reads them, in 20 bits. In 16 they would add a rounding of
// their own to that of their product with y's gradient, which goes into the matrix products in 16 bits,
// and to the result's (gradients off by 0.0031 in bf16 where g and u are kept rounded, by 0.0024 so, against
// 0.0017 of fp32 sums rounded once; in f16 0.00030 against 0.00021).
//
// Pieces of 8 columns lie in blocks of 32 rows x 64 columns, in the order in which a wave has them: 16
// bytes of upper halves of dy/dg, as many of dy/du, and 8 bytes of both next 4 bits, so that a wave
// stores whole lines (rows of bytes, 64 at a time, took 530 us more of a [65536, 6144] forward).
struct Slopes {
  u32x4* hi[2];
  u32x2* lo;
  int64_t wide;  // blocks of 64 columns
  Slopes() = default;
  __host__ __device__ Slopes(uint8_t* p, int64_t M, int64_t N) {
    const int64_t n = pieces(M, N);
    hi[0] = reinterpret_cast<u32x4*>(p);
    hi[1] = hi[0] + n;
    lo = reinterpret_cast<u32x2*>(hi[1] + n);
    wide = (N + 63) / 64;
  }
  static __host__ __device__ int64_t pieces(int64_t M, int64_t N) { return (M + 31) / 32 * ((N + 63) / 64) * 256; }
  static __host__ __device__ int64_t bytes(int64_t M, int64_t N) { return pieces(M, N) * 40; }
  __device__ __forceinline__ int64_t at(int64_t m, int64_t n8) const {
    return ((m >> 5) * wide + (n8 >> 3)) * 256 + ((n8 & 7) >> 1) * 64 + (n8 & 1) * 32 + (m & 31);
  }
};
// A slope in the upper 20 bits of a number (the lower 12 are left over). For bf16 they are fp32's, rounded to 11
// bits of mantissa. f16 needs a 12th (with 11 its gradients are off by 0.00031), but no slope of f16 numbers
// lies beyond 2^53 or matters below 2^-41 (2^16, the largest gradient, times it is the least f16): there the
// number is 2^-64 of the slope and its exponent 7 bits, whose 127 stands for infinities and NaN.
__device__ __forceinline__ uint32_t to_slope(Bf16, float v) { return __float_as_uint(v) + 0x800u; }
__device__ __forceinline__ uint32_t to_slope(_Float16, float v) {
  const uint32_t b = __float_as_uint(v * 0x1p-64f) + 0x400u;
  return (b & 0x80000000u) | (b << 1 & 0x7FFFFFFFu);
}
__device__ __forceinline__ float from_slope(Bf16, uint32_t x) { return __uint_as_float(x); }
__device__ __forceinline__ float from_slope(_Float16, uint32_t x) {
  const uint32_t b = x >> 1 & 0x3FFFFFFFu;
  return __uint_as_float((x & 0x80000000u) | b | (b >= 0x3F800000u ? 0x40000000u : 0u)) * 0x1p64f;
}

__device__ __forceinline__ void wait_vm0() { __builtin_amdgcn_s_waitcnt(0x0F70); }
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xC07F); }
template <int N>
__device__ __forceinline__ void wait_vm() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);
}
__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// A fragment of one matrix instruction: 16 bytes of 16-bit values (k = 8 (l / 32) + j), or 32 bytes
// of 8-bit ones.
template <typename T>
struct Frag;
template <>
struct Frag<Bf16> {
  bf16x8_t v;
};
template <>
struct Frag<_Float16> {
  f16x8_t v;
};
template <>
struct Frag<Fp8> {
  i32x8_t v;
};

__device__ __forceinline__ f32x16_t mfma(Frag<Bf16> b, Frag<Bf16> a, f32x16_t c, int, int) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(b.v, a.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma(Frag<_Float16> b, Frag<_Float16> a, f32x16_t c, int, int) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(b.v, a.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma(Frag<Fp8> b, Frag<Fp8> a, f32x16_t c, int sb, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b.v, a.v, c, 0, 0, 0, sb, 0, sa);
}

// 2^e by its e8m0 byte, e + 127.
__device__ __forceinline__ float power_of(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }

// Eight 8-bit values of a lane's 32 (the c-th eight) times a power of two, as bf16: exact, 4 of its 8 bits of mantissa,
// down to bf16's least number, 2^-133.
__device__ __forceinline__ Frag<Bf16> widen(i32x8_t v, int c, float scale) {
  union {
    bf16x2_t h[4];
    Frag<Bf16> f;
  } u;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    u.h[2 * x] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * c + x], scale, false);
    u.h[2 * x + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * c + x], scale, true);
  }
  return u.f;
}

// A byte at an address that all lanes share, by a scalar load of its word: a vector load would make the
// compiler wait for the stages that are on their way.
__device__ __forceinline__ int uniform_byte(const uint8_t* p) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  const auto* w = (const __attribute__((address_space(4))) uint32_t*)(at & ~uint64_t(3));
  return static_cast<int>(*w >> (8 * (at & 3)) & 0xFFu);
}

__device__ __forceinline__ u32x4 descriptor(uint64_t p, int32_t bytes) {
  return u32x4{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(p))),
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(p >> 32))) & 0xFFFF,
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(bytes)), 0x00020000u};
}

// Sends for kSize bytes of each lane, to LDS at `lds` and on, lane after lane. Nothing waits for them but
// wait_vm. In assembly (it has no result that could be used too soon): of the builtin's loads hipcc
// waits for all before every ds_read_b64_tr, whichever part of LDS that reads. Its own counts of
// loads then only make it wait for more. Five idle states cover descriptors that a VALU wrote; nothing
// else here uses m0.
template <int kSize>
__device__ __forceinline__ void to_lds(u32x4 r, uint8_t* lds, uint32_t at) {
  const uint32_t to = __builtin_amdgcn_readfirstlane(
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds)));
  if constexpr (kSize == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(to), "v"(at), "s"(r)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(to), "v"(at), "s"(r)
                 : "memory");
}

// What a lane does to bring its 16-byte chunks of an operand's stage to LDS: blocks of 1024 bytes,
// one of a wave's instructions each, w + kWaves x for wave w.
template <int kRows, bool kT, int kWaves>
struct Loader {
  static constexpr int kChunks = kT ? kRows / 8 : 4;   // of a row of LDS
  static constexpr int kBlockRows = 64 / kChunks;      // rows of LDS in a block
  static constexpr int kBlocks = kRows / 16 / kWaves;  // blocks of each wave
  static constexpr int kBytes = kRows * 64;
  static constexpr uint32_t kPast = 0x40000000;        // an offset past every descriptor's end
  static_assert(kBlocks >= 1 && (!kT || kChunks >= 16), "a wave has whole blocks");

  static __device__ __forceinline__ int swizzle(int row) { return kT ? 4 * (row & 3) : (row >> 2) & 3; }
  static __device__ __forceinline__ int chunk(int w, int l) { return (l % kChunks) ^ swizzle(w * kBlockRows + l / kChunks); }
  // offset of the lane's chunk in block w, from the tile's first element of the stage
  static __device__ __forceinline__ uint32_t offset(int w, int l, uint32_t ld) {
    return static_cast<uint32_t>(w * kBlockRows + l / kChunks) * ld + chunk(w, l) * 16;
  }
  // Two stages, block by block: the halves of a K-major row's 128-byte line one after the other.
  static __device__ __forceinline__ void load(uint64_t base, int32_t bytes0, int32_t bytes1, uint32_t at0, uint32_t at1,
                                              uint32_t ld, uint64_t apart, uint8_t* lds0, uint8_t* lds1, int w) {
    const u32x4 r0 = descriptor(base, bytes0), r1 = descriptor(base + apart, bytes1);
    const uint32_t step = ld * (kWaves * kBlockRows);
    asm volatile("" : "+v"(at0), "+v"(at1));  // the blocks' offsets are added up here, not held in registers
#pragma unroll
    for (int x = 0; x < kBlocks; ++x) {
      to_lds<16>(r0, lds0 + (w + kWaves * x) * 1024, at0 + x * step);
      to_lds<16>(r1, lds1 + (w + kWaves * x) * 1024, at1 + x * step);
    }
  }
  // the fragment of 32 of the operand's rows from `first` on, kk-th of the stage
  template <typename T>
  static __device__ __forceinline__ Frag<T> frag(const uint8_t* lds, int first, int kk, int l) {
    Frag<T> f;
    if constexpr (kT) {
      const int q = (l & 15) >> 2;
      const int ch = first / 8 + 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
      const int k = kk * 16 + 8 * (l >> 5) + q;
      union {
        s16x4_t h[2];
        Frag<T> f;
      } u;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint8_t* p = lds + (k + 4 * t) * (kRows * 2) + (ch ^ swizzle(q)) * 16 + 8 * (l & 1);
        u.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_t*)(p));
      }
      f = u.f;
    } else {
      const int fr = l & 31;
      const uint8_t* row = lds + (first + fr) * 64;
      if constexpr (sizeof(T) == 2) {
        f = *reinterpret_cast<const Frag<T>*>(row + (((2 * kk + (l >> 5)) ^ swizzle(fr)) << 4));
      } else {
        union {
          i32x4_t h[2];
          Frag<T> f;
        } u;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          u.h[t] = *reinterpret_cast<const i32x4_t*>(row + (((2 * (l >> 5) + t) ^ swizzle(fr)) << 4));
        f = u.f;
      }
    }
    return f;
  }
};

template <typename T_, typename O_, int kBM_, int kBN_, int kWaves_, bool kAT_, bool kBT_, Form kForm_>
struct Tile {
  using T = T_;
  using O = O_;  // the output's type
  static constexpr int kBM = kBM_, kBN = kBN_, kWaves = kWaves_;
  static constexpr bool kAT = kAT_, kBT = kBT_, kScaled = sizeof(T_) == 1;
  static constexpr Form kForm = kForm_;
  // 8 bits into 32-bit results: multiplied as bf16 (see multiply)
  static constexpr bool kWide = kScaled && sizeof(O_) == 4;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int I = kBM / (kWaves / 2) / 32, J = kBN / 2 / 32;  // a wave's 32 x 32 tiles
  static constexpr int KK = kScaled ? 1 : 2;                      // fragments deep a stage
  static constexpr int kCols = kForm_ == kGated ? kBN / 2 : kBN;  // output columns of a tile
  // Rings of stages in LDS. A's next two stages go in while half of the ring is still to be read, B's
  // once two stages have been read by all. With a sixth stage of A, what A's replace was read before the
  // last barrier, and one barrier does for two stages; in 8 bits the scales leave room for five.
  static constexpr int kStageA = kBM * 64, kStageB = kBN * 64;
  static constexpr int kSlotsA = kScaled ? 5 : 6, kSlotsB = 4;
  static constexpr int kB = kSlotsA * kStageA, kScale = kB + kSlotsB * kStageB;  // then 3 steps' scales of A
  static constexpr int kLds = kScale + (kScaled ? 3 * 256 : 0);
  static constexpr int kElems = 64 / static_cast<int>(sizeof(T_));  // of the sum, a stage
  static_assert(kLds <= 160 * 1024, "LDS");
};

// Where a workgroup is in its list of (tile, split): step k of [k, end) of the sum, two stages each, at an
// output tile.
struct Cursor {
  int it, k, end, m0, n0, seg;
  int split;
};

template <typename C>
__device__ __forceinline__ void open_item(const Args& g, Cursor& c, int items) {
  if (c.it >= items) return;
  const int tiles = g.tiles_m * g.tiles_n;
  c.split = c.it / tiles;
  const int t = c.it - c.split * tiles;
  const int wide = g.gm * g.tiles_n, band = t / wide, in = t - band * wide;
  const int rows = min(g.gm, g.tiles_m - band * g.gm);
  int tm = band * g.gm + in % rows;
  c.n0 = in / rows * C::kCols;
  c.seg = 0;
  if (C::kForm == kWeights) {
    const int per = g.tiles_m / g.segs;
    c.seg = tm / per;
    tm -= c.seg * per;
  }
  c.m0 = tm * C::kBM;
  const int total = C::kForm == kPlain ? g.nk * g.segs : g.nk;
  c.k = c.split * g.per;
  c.end = min(total, c.k + g.per);
}

template <typename C>
__global__ __launch_bounds__(C::kThreads, C::kWaves == 8 || C::kLds <= 80 * 1024 ? 2 : 1) void tile_kernel(Args g) {
  using T = typename C::T;
  constexpr int W = C::kWaves;
  using LA = Loader<C::kBM, C::kAT, W>;
  constexpr int kBRows = C::kForm == kGated ? C::kBN / 2 : C::kBN;  // of each of B's tensors in a tile
  using LB = Loader<C::kBT ? C::kBN : kBRows, C::kBT, W>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int t = threadIdx.x, l = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wr = (wave >> 1) * (32 * C::I);
  // the wave's column tiles start here; a gated wave has J / 2 of each half of B's rows
  const int wc = (wave & 1) * (C::kForm == kGated ? 16 * C::J : 32 * C::J);
  auto bcol = [&](int j) __attribute__((always_inline)) {
    if (C::kForm == kGated) return (j / (C::J / 2)) * (C::kBN / 2) + wc + (j % (C::J / 2)) * 32;
    return wc + j * 32;
  };

  const int n_all = g.tiles_m * g.tiles_n * g.splits;
  const int xcd = blockIdx.x % kNumXcd;
  const int lo = static_cast<int>(static_cast<int64_t>(n_all) * xcd / kNumXcd);
  const int items = static_cast<int>(static_cast<int64_t>(n_all) * (xcd + 1) / kNumXcd);
  const int stride = gridDim.x / kNumXcd;
  Cursor c{}, d{}, f{};  // multiplied, sent for, read (8 bits: its scales)
  c.it = lo + blockIdx.x / kNumXcd;
  if (c.it >= items) return;
  open_item<C>(g, c, items);
  d = f = c;
  auto advance = [&](Cursor& q) __attribute__((always_inline)) {
    if (++q.k == q.end) {
      q.it += stride;
      --q.k;  // past the last one it stays where it was
      open_item<C>(g, q, items);
    }
  };

  const uint32_t lda = static_cast<uint32_t>(g.lda), ldb = static_cast<uint32_t>(g.ldb);
  const uint32_t oa = LA::offset(wave, l, lda), ob = LB::offset(wave, l, ldb);
  const int ca = LA::chunk(wave, l) * 16, cb = LB::chunk(wave, l) * 16;
  // What is sent for next: where each operand's stage starts, and how much of the sum is left, in bytes of a
  // K-major row and in k. ends: of a K-major operand's tile rows, from there on; in an M-major one
  // the widths of a k-row's rest.
  constexpr int kBs = C::kForm == kGated ? 2 : 1;
  uint64_t pa = 0, pb[kBs] = {}, psa = 0;
  int left = 0, width_a = 0, width_b = 0;
  auto feed = [&]() __attribute__((always_inline)) {
    int kb = d.k, sg = C::kForm == kWeights ? d.seg : 0;
    if (C::kForm == kPlain && g.segs > 1 && kb >= g.nk) {
      kb -= g.nk;
      sg = 1;
    }
    const int64_t k0 = static_cast<int64_t>(kb) * 2 * C::kElems;
    left = d.it < items ? static_cast<int>(g.K - k0) : 0;
    pa = reinterpret_cast<uint64_t>(sg ? g.a[1] : g.a[0]) +
         (C::kAT ? k0 * g.lda + static_cast<int64_t>(d.m0) * 2 : static_cast<int64_t>(d.m0) * g.lda + kb * 128);
    width_a = C::kAT ? (g.M - d.m0) * 2 : (min(g.M - d.m0, C::kBM) - 1) * static_cast<int>(lda);
#pragma unroll
    for (int h = 0; h < kBs; ++h)
      pb[h] = reinterpret_cast<uint64_t>(h || (C::kForm == kPlain && sg) ? g.b[1] : g.b[0]) +
              (C::kBT ? k0 * g.ldb + static_cast<int64_t>(d.n0) * 2 : static_cast<int64_t>(d.n0) * g.ldb + kb * 128);
    width_b = C::kBT ? (g.N - d.n0) * 2 : (min(g.N - d.n0, kBRows) - 1) * static_cast<int>(ldb);
    if (C::kScaled) psa = reinterpret_cast<uint64_t>(g.sa) + static_cast<int64_t>(kb) * g.lds_a + d.m0;
  };
  int slot_da = 0, slot_db = 0, slot_ds = 0;  // the places in LDS that are sent to next
  auto next_of = [](int slot, int slots, int by) __attribute__((always_inline)) {
    return slot + by >= slots ? slot + by - slots : slot + by;
  };
  // Both stages of a step of A, then of B. What lies past the sum's end, or past the last tile, is sent for
  // with nothing in range, so that every step is the same number of loads; a chunk of a K-major row
  // that starts past the sum's end is read as zeros.
  auto send_a = [&]() __attribute__((always_inline)) {
    uint8_t *to0 = smem + slot_da * C::kStageA, *to1 = smem + next_of(slot_da, C::kSlotsA, 1) * C::kStageA;
    slot_da = next_of(slot_da, C::kSlotsA, 2);
    const int left1 = left - C::kElems;
    if constexpr (C::kAT) {
      LA::load(pa, left > 0 ? (min(left, C::kElems) - 1) * static_cast<int>(lda) + width_a : 0,
               left1 > 0 ? (min(left1, C::kElems) - 1) * static_cast<int>(lda) + width_a : 0, oa, oa, lda,
               static_cast<uint64_t>(g.lda) * C::kElems, to0, to1, wave);
      pa += static_cast<uint64_t>(g.lda) * (2 * C::kElems);
    } else {
      const int bytes = left * static_cast<int>(sizeof(T)), bytes1 = bytes - 64;
      LA::load(pa, bytes > 0 ? width_a + bytes : 0, bytes1 > 0 ? width_a + bytes1 : 0, ca < bytes ? oa : LA::kPast,
               ca < bytes1 ? oa : LA::kPast, lda, 64, to0, to1, wave);
      pa += 128;
    }
    if constexpr (C::kScaled) {
      // a byte of each row, the rows side by side: every wave brings all of them, so that all send the
      // same number of loads
      const u32x4 r = descriptor(psa, left > 0 ? static_cast<int>(min(g.lds_a - d.m0, int64_t(C::kBM))) : 0);
      to_lds<4>(r, smem + C::kScale + slot_ds * 256, l * 4);
      slot_ds = next_of(slot_ds, 3, 1);
    }
  };
  auto send_b = [&]() __attribute__((always_inline)) {
    uint8_t *to0 = smem + C::kB + slot_db * C::kStageB, *to1 = to0 + C::kStageB;  // slots 0 and 1, or 2 and 3
    slot_db ^= 2;
    const int left1 = left - C::kElems;
    const int bytes = left * static_cast<int>(sizeof(T)), bytes1 = bytes - 64;
#pragma unroll
    for (int h = 0; h < kBs; ++h) {
      const int at = h * LB::kBytes;
      if constexpr (C::kBT) {
        LB::load(pb[h], left > 0 ? (min(left, C::kElems) - 1) * static_cast<int>(ldb) + width_b : 0,
                 left1 > 0 ? (min(left1, C::kElems) - 1) * static_cast<int>(ldb) + width_b : 0, ob, ob, ldb,
                 static_cast<uint64_t>(g.ldb) * C::kElems, to0 + at, to1 + at, wave);
        pb[h] += static_cast<uint64_t>(g.ldb) * (2 * C::kElems);
      } else {
        LB::load(pb[h], bytes > 0 ? width_b + bytes : 0, bytes1 > 0 ? width_b + bytes1 : 0, cb < bytes ? ob : LB::kPast,
                 cb < bytes1 ? ob : LB::kPast, ldb, 64, to0 + at, to1 + at, wave);
        pb[h] += 128;
      }
    }
    left -= 2 * C::kElems;
  };
  auto next_step = [&]() __attribute__((always_inline)) {  // both operands have been sent for
    const int was = d.it;
    advance(d);
    if (C::kScaled) psa += g.lds_a;
    if (d.it != was || (C::kForm == kPlain && g.segs > 1 && d.k == g.nk)) feed();
  };

  // two sets of fragments: one is multiplied while the other is read
  Frag<T> fa[2][C::KK][C::I], fb[2][C::KK][C::J];
  int sa[2][C::I], sb[2][2];
  f32x16_t acc[C::I][C::J];
  auto zero_acc = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < C::I; ++i)
#pragma unroll
      for (int j = 0; j < C::J; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  };
  int slot_fa = 0, slot_fb = 0, slot_fs = 0;  // the places in LDS that are read next
  auto fetch = [&](int set) __attribute__((always_inline)) {
    const uint8_t* s = smem + slot_fa * C::kStageA;
    const uint8_t* sb_at = smem + C::kB + slot_fb * C::kStageB;
    const uint8_t* ss = smem + C::kScale + slot_fs * 256;
    slot_fa = next_of(slot_fa, C::kSlotsA, 1);
    slot_fb = (slot_fb + 1) % C::kSlotsB;
    if (C::kScaled && set == 1) slot_fs = next_of(slot_fs, 3, 1);
    if constexpr (C::kScaled) {
      // the wave's columns lie in one block of 128 rows of B (two for a gated wave, one of each tensor)
      const int64_t at = static_cast<int64_t>(min(f.n0 + wc, g.N - 1) >> 7) * g.nk + f.k;
      sb[set][0] = uniform_byte(g.sb[0] + at);
      sb[set][1] = C::kForm == kGated ? uniform_byte(g.sb[1] + at) : sb[set][0];
#pragma unroll
      for (int i = 0; i < C::I; ++i) sa[set][i] = ss[wr + i * 32 + (l & 31)];
    }
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk) {
#pragma unroll
      for (int i = 0; i < C::I; ++i) fa[set][kk][i] = LA::template frag<T>(s, wr + i * 32, kk, l);
#pragma unroll
      for (int j = 0; j < C::J; ++j)
        fb[set][kk][j] = Loader<C::kBN, C::kBT, W>::template frag<T>(sb_at, bcol(j), kk, l);
    }
  };
  // with B's fragment first, lane l holds row l % 32 of a tile and its columns 8 q + 4 (l / 32) + e
  // in acc[i][j][4 q + e]
  // 8 bits into 32-bit results: the scaled instruction cuts products off 2^-13 below the largest of eight, so
  // the values are widened to bf16, scales and all, which holds them exactly, and multiplied by the bf16
  // instruction, 16 deep, in fp32. (Both operands' fragments hold the same k in the same place: which 16 go together
  // does not matter.)
  auto multiply = [&](int set) __attribute__((always_inline)) {
    if constexpr (C::kWide) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        Frag<Bf16> a[C::I], b[C::J];
#pragma unroll
        for (int i = 0; i < C::I; ++i) a[i] = widen(fa[set][0][i].v, c, power_of(sa[set][i]));
#pragma unroll
        for (int j = 0; j < C::J; ++j)
          b[j] = widen(fb[set][0][j].v, c, power_of(sb[set][C::kForm == kGated && j >= C::J / 2]));
#pragma unroll
        for (int i = 0; i < C::I; ++i)
#pragma unroll
          for (int j = 0; j < C::J; ++j) acc[i][j] = mfma(b[j], a[i], acc[i][j], 0, 0);
      }
      return;
    }
#pragma unroll
    for (int kk = 0; kk < C::KK; ++kk)
#pragma unroll
      for (int i = 0; i < C::I; ++i)
#pragma unroll
        for (int j = 0; j < C::J; ++j) {
          if constexpr (C::kScaled && !C::kWide)
            acc[i][j] = mfma(fb[set][kk][j], fa[set][kk][i], acc[i][j], sb[set][C::kForm == kGated && j >= C::J / 2],
                             sa[set][i]);
          else if constexpr (!C::kScaled)
            acc[i][j] = mfma(fb[set][kk][j], fa[set][kk][i], acc[i][j], 0, 0);
        }
  };

  int h = 0, row = 0;  // set by the epilogue
  // Where a tile goes: from its first element to the tensor's end, so that rows past M are dropped;
  // a lane's offset of a column past N lies past that end too.
  auto target = [&](void* out, int64_t ld, int size, int m0, int n0) __attribute__((always_inline)) {
    const int64_t bytes = (static_cast<int64_t>(g.M - 1 - m0) * ld + (g.N - n0)) * size;
    return __builtin_amdgcn_make_buffer_rsrc(
        static_cast<uint8_t*>(out) + (static_cast<int64_t>(m0) * ld + n0) * size, 0,
        static_cast<int32_t>(bytes < LA::kPast ? bytes : LA::kPast), 0x00020000);
  };
  // 16 sums of a tile's row (at column n of the output tile) as fp32, 4 columns a lane and store
  auto store_f32 = [&](__amdgpu_buffer_rsrc_t r, uint32_t row_at, int n, const f32x16_t& v) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = n + 8 * q + 4 * h, left = g.N - c.n0 - col;
      const uint32_t at = row_at + col * 4;
      if (!C::kScaled || g.N % 4 == 0) {
        const f32x4_t x{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), r, left > 0 ? at : LA::kPast, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[4 * q + e]), r, e < left ? at + 4 * e : LA::kPast, 0, 0);
      }
    }
  };
  // 8 of them, of 16 columns from n on, as 16 bits, 8 columns a lane and store: the lane pair trades
  // halves (after the swap lane l < 32 has columns 0 to 7 of 16, lane l + 32 columns 8 to 15)
  auto store_eight = [&](__amdgpu_buffer_rsrc_t r, uint32_t row_at, int n, const float* v) __attribute__((always_inline)) {
    using O = std::conditional_t<sizeof(typename C::O) == 2, typename C::O, Bf16>;
    uint32_t w[2][2];
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int x = 0; x < 2; ++x) w[y][x] = pack2(O{}, v[4 * y + 2 * x], v[4 * y + 2 * x + 1]);
    u32x4 out;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const auto sw = __builtin_amdgcn_permlane32_swap(w[0][x], w[1][x], false, false);
      out[x] = sw[0];
      out[2 + x] = sw[1];
    }
    const int col = n + 8 * h, left = g.N - c.n0 - col;
    const uint32_t at = row_at + col * 2;
    if (!C::kScaled || g.N % 8 == 0) {
      __builtin_amdgcn_raw_buffer_store_b128(out, r, left > 0 ? at : LA::kPast, 0, 0);
    } else {
      // rows of an even number of columns start at multiples of 4 bytes, which is what a wide store asks for:
      // 777 rows of 1000 columns into 1234 13.7 us with single values, 10.8 so
      const bool wide = g.N % 2 == 0;
      if (wide) __builtin_amdgcn_raw_buffer_store_b128(out, r, left >= 8 ? at : LA::kPast, 0, 0);
      if (left <= 0 || (wide && left >= 8)) return;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        __builtin_amdgcn_raw_buffer_store_b16(static_cast<uint16_t>(out[e / 2] >> (16 * (e & 1))), r,
                                              e < left ? at + 2 * e : LA::kPast, 0, 0);
    }
  };
  auto store_row = [&](__amdgpu_buffer_rsrc_t r, uint32_t row_at, int n, const f32x16_t& v) __attribute__((always_inline)) {
    if constexpr (sizeof(typename C::O) == 4) {
      store_f32(r, row_at, n, v);
    } else {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = v[8 * p + e];
        store_eight(r, row_at, n + 16 * p, x);
      }
    }
  };
  auto epilogue = [&]() __attribute__((always_inline)) {
    int lane = l;
    asm volatile("" : "+v"(lane));  // nothing of the epilogue is computed before the loop
    h = lane >> 5;
    row = wr + (lane & 31);
    if (g.splits > 1) {
      const int planes = C::kForm == kGated ? 2 : C::kForm == kWeights ? g.segs : 1;
      const int64_t plane = static_cast<int64_t>(g.M) * g.N;
      float* part = g.part + (static_cast<int64_t>(c.split) * planes + c.seg) * plane;
#pragma unroll
      for (int j = 0; j < C::J; ++j) {
        const bool second = C::kForm == kGated && j >= C::J / 2;
        const __amdgpu_buffer_rsrc_t r = target(part + (second ? plane : 0), g.N, 4, c.m0, c.n0);
#pragma unroll
        for (int i = 0; i < C::I; ++i)
          store_f32(r, static_cast<uint32_t>(row + i * 32) * g.N * 4, wc + (second ? j - C::J / 2 : j) * 32, acc[i][j]);
      }
      return;
    }
    constexpr int kSize = sizeof(typename C::O);
    const uint32_t ld = static_cast<uint32_t>(g.ldo) * kSize;
    if constexpr (C::kForm == kGated && kSize == 4) {
      const __amdgpu_buffer_rsrc_t r = target(g.out[0], g.ldo, kSize, c.m0, c.n0);
#pragma unroll
      for (int i = 0; i < C::I; ++i)
#pragma unroll
        for (int j = 0; j < C::J / 2; ++j) {
          f32x16_t y;
#pragma unroll
          for (int x = 0; x < 16; ++x) y[x] = gated_value(acc[i][j][x], acc[i][j + C::J / 2][x]);
          store_f32(r, static_cast<uint32_t>(row + i * 32) * ld, wc + j * 32, y);
        }
    } else if constexpr (C::kForm == kGated) {
      if (g.slopes) {
        const __amdgpu_buffer_rsrc_t r = target(g.out[0], g.ldo, kSize, c.m0, c.n0);
        // the tile's first block, to the tensor's end
        const Slopes to(g.slopes, g.M, g.N);
        const int64_t first = to.at(c.m0, c.n0 / 8), rest = Slopes::pieces(g.M, g.N) - first;
        auto pieces = [&](void* p, int size) __attribute__((always_inline)) {
          return __builtin_amdgcn_make_buffer_rsrc(static_cast<uint8_t*>(p) + first * size, 0,
                                                   static_cast<int32_t>(min(rest * size, int64_t(LA::kPast))), 0x00020000);
        };
        const __amdgpu_buffer_rsrc_t hi0 = pieces(to.hi[0], 16), hi1 = pieces(to.hi[1], 16), lo = pieces(to.lo, 8);
        const uint32_t wide = static_cast<uint32_t>(to.wide);
#pragma unroll
        for (int i = 0; i < C::I; ++i)
#pragma unroll
          for (int j = 0; j < C::J / 2; ++j) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              float y[8], d[8], q[8];
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                float s;
                const float u = acc[i][j + C::J / 2][8 * p + x];
                q[x] = silu(acc[i][j][8 * p + x], s);
                y[x] = q[x] * u;
                d[x] = gate_slope(u, q[x], s);
              }
              store_eight(r, static_cast<uint32_t>(row + i * 32) * ld, wc + j * 32 + 16 * p, y);
              uint32_t w[2][2][2], b[2];  // [slope][columns 4 y on][pair]
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                uint32_t x[2][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  x[0][e] = to_slope(typename C::O{}, d[4 * y + e]);
                  x[1][e] = to_slope(typename C::O{}, q[4 * y + e]);
                }
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                  w[f][y][0] = __builtin_amdgcn_perm(x[f][1], x[f][0], 0x07060302);
                  w[f][y][1] = __builtin_amdgcn_perm(x[f][3], x[f][2], 0x07060302);
                }
                // the bytes below the upper halves, whose upper halves are the next 4 bits
                uint32_t n[2];
#pragma unroll
                for (int f = 0; f < 2; ++f)
                  n[f] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(x[f][3], x[f][2], 0x05010501),
                                               __builtin_amdgcn_perm(x[f][1], x[f][0], 0x05010501), 0x05040100);
                b[y] = (n[0] >> 4 & 0x0F0F0F0Fu) | (n[1] & 0xF0F0F0F0u);
              }
              const int col = wc + j * 32 + 16 * p;  // of the tile, 8 h beyond
              const uint32_t at = (static_cast<uint32_t>(wr / 32 + i) * wide + (col >> 6)) * 256 + (col >> 4 & 3) * 64 + lane;
              const bool in = col + 8 * h < g.N - c.n0;
#pragma unroll
              for (int f = 0; f < 2; ++f) {
                u32x4 out;
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  const auto sw = __builtin_amdgcn_permlane32_swap(w[f][0][x], w[f][1][x], false, false);
                  out[x] = sw[0];
                  out[2 + x] = sw[1];
                }
                __builtin_amdgcn_raw_buffer_store_b128(out, f ? hi1 : hi0, in ? at * 16 : LA::kPast, 0, 0);
              }
              const auto sw = __builtin_amdgcn_permlane32_swap(b[0], b[1], false, false);
              __builtin_amdgcn_raw_buffer_store_b64(u32x2{sw[0], sw[1]}, lo, in ? at * 8 : LA::kPast, 0, 0);
              __builtin_amdgcn_sched_barrier(0);  // one piece after another: the registers are full
            }
          }
        return;
      }
      const __amdgpu_buffer_rsrc_t r = target(g.out[0], g.ldo, kSize, c.m0, c.n0);
#pragma unroll
      for (int i = 0; i < C::I; ++i)
#pragma unroll
        for (int j = 0; j < C::J / 2; ++j) {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            float y[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) y[x] = gated_value(acc[i][j][8 * p + x], acc[i][j + C::J / 2][8 * p + x]);
            store_eight(r, static_cast<uint32_t>(row + i * 32) * ld, wc + j * 32 + 16 * p, y);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
    } else {
      const __amdgpu_buffer_rsrc_t r = target(c.seg ? g.out[1] : g.out[0], g.ldo, kSize, c.m0, c.n0);
#pragma unroll
      for (int i = 0; i < C::I; ++i)
#pragma unroll
        for (int j = 0; j < C::J; ++j) store_row(r, static_cast<uint32_t>(row + i * 32) * ld, wc + j * 32, acc[i][j]);
    }
  };

  zero_acc();
  constexpr int kLoadsA = 2 * LA::kBlocks + C::kScaled, kLoadsB = 2 * kBs * LB::kBlocks;  // a step's, of a wave
  feed();
#pragma unroll 1
  for (int s = 0; s < 2; ++s) {
    send_a();
    send_b();
    next_step();
  }
  wait_vm<kLoadsA + kLoadsB>();
  barrier();
  fetch(0);
  while (true) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __builtin_amdgcn_sched_barrier(0);
      wait_lgkm0();  // this stage's fragments are here
      if (half == 0) {
        if (C::kSlotsA < 6) barrier();
        send_a();
      } else {
        // The next step has landed when no more than A of the one after it is on its way (loads return in
        // order; stores in between only make the wait longer), and every wave is done with B's stages.
        if (C::kScaled) advance(f);
        wait_vm<kLoadsA>();
        barrier();
        send_b();
      }
      fetch(half ^ 1);  // after the last stage of all: what is there, for nothing
      multiply(half);
      // reads between the matrix instructions
      constexpr int kMul = (C::kWide ? 4 : C::KK) * C::I * C::J;
      constexpr int kReads = C::kScaled ? 3 * C::I + 2 * C::J : C::KK * (C::I * (C::kAT ? 2 : 1) + C::J * (C::kBT ? 2 : 1));
      constexpr int kEach = (kReads + kMul - 1) / kMul;
#pragma unroll
      for (int n = 0; n < kMul; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kEach, 0);
      }
      asm volatile("" ::: "memory");  // the reads stay here, and so do the products
#pragma unroll
      for (int i = 0; i < C::I; ++i)
#pragma unroll
        for (int j = 0; j < C::J; ++j) asm volatile("" : "+v"(acc[i][j]));
      __builtin_amdgcn_sched_barrier(0);
      if (half) next_step();
    }
    if (c.k + 1 == c.end) {
      epilogue();
      zero_acc();
    }
    advance(c);
    if (c.it >= items) break;
  }
  wait_vm0();  // no load still writing this workgroup's LDS at its end
}

// Adds up the splits' sums in order and stores them. A thread has 4 columns of a row where the rows
// are whole fours, else one.
template <typename O, Form kForm, int W>
__global__ __launch_bounds__(256) void join_kernel(Args g, int64_t count) {
  const int64_t i = (block_index() * 256 + threadIdx.x) * W;
  if (i >= count) return;
  const int64_t plane = static_cast<int64_t>(g.M) * g.N;
  const int planes = kForm == kGated ? 2 : kForm == kWeights ? g.segs : 1;
  float v[2][W];
#pragma unroll
  for (int p = 0; p < (kForm == kGated ? 2 : 1); ++p) {
#pragma unroll
    for (int e = 0; e < W; ++e) v[p][e] = 0.f;
    for (int s = 0; s < g.splits; ++s) {
      const float* at = g.part + static_cast<int64_t>(s) * planes * plane + p * plane + i;
      if constexpr (W == 4) {
        const f32x4_t q = *reinterpret_cast<const f32x4_t*>(at);
#pragma unroll
        for (int e = 0; e < W; ++e) v[p][e] += q[e];
      } else {
        v[p][0] += at[0];
      }
    }
  }
  const int64_t in = kForm == kWeights ? i % plane : i;
  const int seg = kForm == kWeights ? static_cast<int>(i / plane) : 0;
  const int64_t to = in / g.N * g.ldo + in % g.N;
  auto put = [&](void* out, const float* f) {
    O* o = static_cast<O*>(out) + to;
    if constexpr (W == 1) {
      *o = from_f32<O>(f[0]);
    } else if constexpr (sizeof(O) == 4) {
      *reinterpret_cast<f32x4_t*>(o) = f32x4_t{f[0], f[1], f[2], f[3]};
    } else {
      *reinterpret_cast<u32x2*>(o) = u32x2{pack2(O{}, f[0], f[1]), pack2(O{}, f[2], f[3])};
    }
  };
  if constexpr (kForm == kGated) {
    if constexpr (sizeof(O) == 2) if (g.slopes) {
      const Slopes to(g.slopes, g.M, g.N);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        float s;
        const float q = silu(v[0][e], s);
        const uint32_t x[2] = {to_slope(O{}, gate_slope(v[1][e], q, s)), to_slope(O{}, q)};
        const int64_t n = in % g.N + e, piece = to.at(in / g.N, n / 8);
#pragma unroll
        for (int f = 0; f < 2; ++f) reinterpret_cast<uint16_t*>(to.hi[f] + piece)[n % 8] = static_cast<uint16_t>(x[f] >> 16);
        reinterpret_cast<uint8_t*>(to.lo + piece)[n % 8] = static_cast<uint8_t>((x[0] >> 12 & 15) | (x[1] >> 8 & 0xF0));
      }
    }
#pragma unroll
    for (int e = 0; e < W; ++e) v[0][e] = gated_value(v[0][e], v[1][e]);
    put(g.out[0], v[0]);
  } else {
    put(kForm == kWeights && seg ? g.out[1] : g.out[0], v[0]);
  }
}

}  // namespace gemm
}  // namespace lema

// ------------------------------------------------------------------------------------ host

namespace lema {
namespace gemm {

// One of the tiles that a product can take, as the choice sees it: rows and output columns, the
// workgroups that a CU holds, and what a stage (128 bytes of the sum) and a tile's first loads and its
// epilogue take there, in us.
//
// The shapes' numbers, and the three below, are fitted to the times of every tile and number of splits for
// 33 to 16,384 rows of widths 256 to 6144. Over those 256 products the choice takes 0.2 % longer than the
// best one on average, 7 % at most; without kAlone 3 % and 38 %, without splits 17 % and 4 times as long, the
// large tile alone 80 % and 7 times. Over 72 products of other sizes it takes 1 % and 15 % longer. The two
// sides of it at 1536 columns into 6144 (gated, bf16): 96 rows 17 us in 64 x 64 tiles and 20 in 128 x 64;
// 400 rows 31 and 28; 777 rows 42 in 128 x 64 and 37 in 256 x 128; 48 rows 15.2 in two splits and 16.5 in one.
struct Shape {
  int bm, cols, per_cu;
  float stage_us, tile_us;
};

struct Plan {
  int shape, splits, per;
  int64_t part_bytes;  // of the splits' sums
};

constexpr float kAlone = 0.7f;    // the time of a workgroup that has a CU for two to itself
constexpr float kJoinUs = 4.0f;   // the second launch
constexpr float kJoinRate = 3e6f; // bytes/us of the splits' sums, written and read

int num_cus();

// The tile and the number of splits with the least modelled time: rounds of workgroups over the
// CUs, stages in each, and the splits' traffic. `rows` and `segs`: of the output, `stages` of the
// whole sum.
inline Plan make_plan(const Shape* shapes, int count, int64_t rows, int64_t cols, int segs, int planes, int64_t stages) {
  Plan best{-1, 1, static_cast<int>(stages), 0};
  double least = 0;
  for (int i = 0; i < count; ++i) {
    const Shape& s = shapes[i];
    const int64_t tiles = (rows + s.bm - 1) / s.bm * ((cols + s.cols - 1) / s.cols) * segs;
    const int64_t slots = static_cast<int64_t>(num_cus()) * s.per_cu;
    for (int64_t splits = 1; splits <= 32 && splits <= stages; ++splits) {
      const int64_t per = (stages + splits - 1) / splits;
      if (splits > 1 && (per < 4 || (splits - 1) * per >= stages)) continue;
      if (splits > 1 && tiles * (splits - 1) >= 4 * slots) break;
      const int64_t rounds = (tiles * splits + slots - 1) / slots;
      const int64_t bytes = splits > 1 ? splits * planes * rows * cols * 4 : 0;
      const bool alone = s.per_cu > 1 && tiles * splits - (rounds - 1) * slots <= num_cus();
      const double us = (rounds - 1 + (alone ? kAlone : 1.f)) * (per * static_cast<double>(s.stage_us) + s.tile_us) +
                        (splits > 1 ? kJoinUs + 2.0 * bytes / kJoinRate : 0.0);
      if (best.shape < 0 || us < least) {
        least = us;
        best = Plan{i, static_cast<int>(splits), static_cast<int>(per), bytes};
      }
    }
  }
  return best;
}

template <typename C>
int launch_tiles(Args g, const Plan& p, int per_cu, hipStream_t st) {
  g.splits = p.splits;
  g.per = p.per;
  const int segs = C::kForm == kWeights ? g.segs : 1;
  const int64_t tm = static_cast<int64_t>((g.M + C::kBM - 1) / C::kBM) * segs;
  const int64_t tn = (g.N + C::kCols - 1) / C::kCols;
  LEMA_REQUIRE(tm * tn * p.splits < (int64_t(1) << 31), "the product has too many tiles");
  g.tiles_m = static_cast<int32_t>(tm);
  g.tiles_n = static_cast<int32_t>(tn);
  g.gm = 4;
  LEMA_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(tile_kernel<C>),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::kLds));
  const int64_t slots = static_cast<int64_t>(num_cus()) / kNumXcd * kNumXcd * per_cu;
  const int64_t items = (tm * tn * p.splits + kNumXcd - 1) / kNumXcd * kNumXcd;
  tile_kernel<C><<<dim3(static_cast<uint32_t>(items < slots ? items : slots)), dim3(C::kThreads), C::kLds, st>>>(g);
  const int rc = launch_status("tile_kernel");
  if (rc != LEMA_OK || p.splits == 1) return rc;
  const int64_t count = static_cast<int64_t>(g.M) * g.N * segs;
  if (g.N % 4 == 0)
    join_kernel<typename C::O, C::kForm, 4><<<blocks_of((count / 4 + 255) / 256), dim3(256), 0, st>>>(g, count);
  else
    join_kernel<typename C::O, C::kForm, 1><<<blocks_of((count + 255) / 256), dim3(256), 0, st>>>(g, count);
  return launch_status("join_kernel");
}

}  // namespace gemm
}  // namespace lema
