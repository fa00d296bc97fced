// A token of each row of logits z from a given random number u in [0, 1), after a temperature T, top-k,
// top-p and min-p (the decoder's pick, code/lema/decode.py:71-93, with the filters it lacks).
//
// With w_i = e^((z_i - max) / T) and the tokens in the order of their logits (equal ones by index):
//   top-k   keeps the first k;
//   top-p   keeps of those with mass M each whose predecessors' mass is below p M (the first always);
//   min-p   keeps w_i >= m (the largest w is 1);
// each keeps a head of that order. The token is the first in vocabulary order whose running sum of
// kept w exceeds u times their sum. The log-probability is (z_i - max) / T - log sum of all w.
//
// One workgroup of 1024 threads a row. A row of up to 128 KB is held in LDS and read once from memory, one of up
// to 256 KB in registers for the passes that every row takes; otherwise it is read again in each pass, from
// the caches. A single CU's arithmetic is what bounds a row
// (an instruction for each of 50,304 logits takes 0.33 us), so the passes over it are few and short:
//   1  the maximum, of the row and of each thread's part of it;
//   2  the sum of all w, and a list of those tokens that can be kept: not below min-p's border, nor below
//      the k-th largest of the threads' maxima (k of the row's tokens are no smaller). For top-p alone
//      the 320 largest of those maxima are tried, which hold the nucleus of a peaked row. The list is
//      ranked, cut and drawn from alone, without another look at the row.
//   Otherwise (a nucleus or a k that reaches further, more candidates than the list holds) a histogram of
//   the distances to the maximum finds the bin of a border, a pass lists that bin's tokens, and a last
//   one draws.
// Measured, bf16 logits: 50,304 with top-k 50 14 us for one row, 26 for 64 rows with settings of their own,
// 18 without a filter; 13 rows of 32,003 fp32 logits with a nucleus of thousands of tokens 38 us; 1024 rows of
// 131,072 with min-p 136 us (reading them 50): four rows a CU, one after another, each bound by its passes.
// Sums of w: of a list in 2^-44 fixed point, elsewhere fp32 within 8 logits and fp64 beyond; all in a fixed
// order (a histogram's are whole numbers, and only say where to look).
#include "elem.h"

namespace lema {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kList = 2048;     // candidates that are sorted
constexpr int kBins = 1536;     // of a logit's distance to the maximum: 128 to an octave from 2^-5 to 2^7
constexpr int kFirstBin = 0x3D00;
constexpr int64_t kMaxVocab = 1 << 20;
// A row that LDS holds beside the list. Registers, which take the next lengths, hold it in the first passes only:
// 17.2 us a row (LDS 15.0) and 68 for a late nucleus (60); from memory in each pass, 131,072 f16 logits take 112 us
// for a late nucleus and 103 from registers.
constexpr int64_t kRowBytes = 128 * 1024;

// A setting: one for all rows, or one of each.
struct Setting {
  const void* each;  // fp32 (int64 for top-k), or null
  float one;
  int32_t k;
};

struct SampleArgs {
  const void* logits;
  int64_t V, inner, so, si;  // row r starts at (r / inner) * so + (r % inner) * si
  const float* u;
  Setting temperature, top_k, top_p, min_p;
  int64_t* tokens;
  float* logprobs;  // or null
  int64_t seg_bytes;
};

// Order-preserving bits of a number that is no NaN; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

template <typename T>
constexpr int kKeyShift = 0;  // low bits of a key that go with its sign
template <>
constexpr int kKeyShift<Bf16> = 16;
template <>
constexpr int kKeyShift<_Float16> = 13;

struct Shared {
  double part[kWaves];
  uint64_t part64[kWaves];
  uint32_t part32[kWaves];
  int found;
  int count;
  double before;
  uint64_t mass;
};

// A value of the lane that a DPP control names.
template <int kCtrl, typename V>
__device__ __forceinline__ V moved(V v) {
  union {
    V v;
    int w[sizeof(V) / 4];
  } u{v};
#pragma unroll
  for (unsigned i = 0; i < sizeof(V) / 4; ++i) u.w[i] = __builtin_amdgcn_mov_dpp(u.w[i], kCtrl, 0xF, 0xF, true);
  return u.v;
}
// f over all lanes of a wave, f associative and commutative: pairs, quads, halves of rows and rows by
// DPP, then rows by swaps.
template <typename V, typename F>
__device__ __forceinline__ V wave_reduce(V v, F f) {
  v = f(v, moved<0xB1>(v));
  v = f(v, moved<0x4E>(v));
  v = f(v, moved<0x141>(v));
  v = f(v, moved<0x140>(v));
  union U {
    V v;
    int w[sizeof(V) / 4];
  } a{v}, b;
#pragma unroll
  for (unsigned i = 0; i < sizeof(V) / 4; ++i) {
    const auto q = __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
    a.w[i] = q[0], b.w[i] = q[1];
  }
  a.v = f(a.v, b.v);
#pragma unroll
  for (unsigned i = 0; i < sizeof(V) / 4; ++i) {
    const auto q = __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false);
    a.w[i] = q[0], b.w[i] = q[1];
  }
  return f(a.v, b.v);
}

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* part, F f) {
  v = wave_reduce(v, f);
  __syncthreads();  // the parts of an earlier call are read
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v = f(v, part[w]);
  return v;
}
__device__ __forceinline__ double block_sum(double v, Shared& s) {
  return block_reduce(v, s.part, [](double a, double b) { return a + b; });
}

// A value of the lane that a DPP control names, 0 where there is none (and in rows that the mask leaves out).
template <int kCtrl, int kRows, typename V>
__device__ __forceinline__ V moved_or_zero(V v) {
  union {
    V v;
    int w[sizeof(V) / 4];
  } u{v};
#pragma unroll
  for (unsigned i = 0; i < sizeof(V) / 4; ++i) u.w[i] = __builtin_amdgcn_update_dpp(0, u.w[i], kCtrl, kRows, 0xF, false);
  return u.v;
}
// The sum of a wave's lower lanes' values and one's own: within rows of 16, then row 0 into 1 and 2 into 3,
// then the lower half into the upper.
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
  v += moved_or_zero<0x111, 0xF>(v);
  v += moved_or_zero<0x112, 0xF>(v);
  v += moved_or_zero<0x114, 0xF>(v);
  v += moved_or_zero<0x118, 0xF>(v);
  v += moved_or_zero<0x142, 0xA>(v);
  v += moved_or_zero<0x143, 0xC>(v);
  return v;
}

// The sum of the lower threads' values and one's own; the block's total in `total`.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* part, V& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) part[wave] = v;
  __syncthreads();
  V add = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w == wave) add = total;
    total += part[w];
  }
  return v + add;
}

// The largest of a thread's logits, and whether one is a NaN. 16-bit types are compared as they lie: as
// whole numbers positive ones order as they are, negative ones the other way, and NaN lie beyond the
// infinity of their sign.
template <typename T>
struct Largest {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  static constexpr uint16_t kInf = std::is_same<T, Bf16>::value ? 0x7F80 : 0x7C00, kNegInf = kInf | 0x8000;
  s16x2 most = {static_cast<short>(kNegInf), static_cast<short>(kNegInf)};
  u16x2 least = {kNegInf, kNegInf}, last = {kNegInf, kNegInf};
  __device__ __forceinline__ void take(const Piece<T>& p) {
    two(p.raw.x), two(p.raw.y), two(p.raw.z), two(p.raw.w);
  }
  __device__ __forceinline__ void two(uint32_t w) {
    most = __builtin_elementwise_max(most, __builtin_bit_cast(s16x2, w));
    least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, w));
    last = __builtin_elementwise_max(last, __builtin_bit_cast(u16x2, w));
  }
  __device__ __forceinline__ float value() const {
    const short m = max(most[0], most[1]);
    const uint16_t bits = m >= 0 ? static_cast<uint16_t>(m) : min(least[0], least[1]);
    return to_f32(__builtin_bit_cast(T, bits));
  }
  __device__ __forceinline__ bool nan() const { return max(most[0], most[1]) > kInf || max(last[0], last[1]) > kNegInf; }
};
template <>
struct Largest<float> {
  float most = -INFINITY;
  bool any = false;
  __device__ __forceinline__ void take(const Piece<float>& p) {
    one(p.e[0]), one(p.e[1]), one(p.e[2]), one(p.e[3]);
  }
  __device__ __forceinline__ void one(float v) {
    most = __builtin_fmaxf(most, v);
    any |= v != v;
  }
  __device__ __forceinline__ float value() const { return most; }
  __device__ __forceinline__ bool nan() const { return any; }
};

// A row as its pieces of 16 bytes, piece t + 1024 j for thread t: in LDS, in memory, or in registers for
// the passes that every row takes (and in memory for the others, whose code would be 16 times as long).
// What lies behind the row reads as -inf, a token without mass.
enum Place { kInMemory, kInLds, kInRegisters };

template <typename T, Place kPlace>
struct Row {
  static constexpr int N = kPiece<T>;
  static constexpr bool kLds = kPlace == kInLds;
  static constexpr int kHeld = kPlace == kInRegisters ? 16 : 1;
  Piece<T> q[kHeld];
  const T* at;
  u32x4* lds;
  int64_t V;
  int tiles;
  bool infinite;  // the maximum is +inf: such tokens share the mass, no other has any

  __device__ __forceinline__ Piece<T> fetch(int j) const {
    const int64_t e = (static_cast<int64_t>(j) * kThreads + threadIdx.x) * N;
    Piece<T> p;
    if (e + N <= V) {
      p.raw = get16(at + e);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p.e[i] = e + i < V ? at[e + i] : from_f32<T>(-INFINITY);
    }
    if (infinite) level(p);
    return p;
  }
  // A row with +inf: 0 in its place, -inf for all else.
  static __device__ __forceinline__ void level(Piece<T>& p) {
#pragma unroll
    for (int i = 0; i < N; ++i) p.e[i] = from_f32<T>(to_f32(p.e[i]) == INFINITY ? 0.f : -INFINITY);
  }
  __device__ __forceinline__ void level() {
    infinite = true;
    if constexpr (kLds)
      for (int j = 0; j < tiles; ++j) {
        Piece<T> p = piece(j);
        level(p);
        lds[j * kThreads + threadIdx.x] = p.raw;
      }
    if constexpr (kPlace == kInRegisters)
#pragma unroll
      for (int j = 0; j < kHeld; ++j) level(q[j]);
  }
  // The first look, in which LDS gets the row.
  __device__ __forceinline__ Largest<T> open(const T* row, int64_t n, u32x4* to) {
    at = row;
    V = n;
    lds = to;
    infinite = false;
    tiles = static_cast<int>((n + kThreads * N - 1) / (kThreads * N));
    Largest<T> most;
    auto take = [&](int j, const Piece<T>& p) __attribute__((always_inline)) {
      most.take(p);
      if (kLds) lds[j * kThreads + threadIdx.x] = p.raw;
    };
    if constexpr (kPlace == kInRegisters) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) q[j] = fetch(j);
#pragma unroll
      for (int j = 0; j < kHeld; ++j) most.take(q[j]);
      return most;
    }
    constexpr int kAhead = 4;
    Piece<T> p[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) p[i] = fetch(min(i, tiles - 1));
    for (int j = 0; j < tiles; j += kAhead)
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (j + i < tiles) {
          take(j + i, p[i]);
          if (j + i + kAhead < tiles) p[i] = fetch(j + i + kAhead);
        }
    return most;  // a thread reads what it wrote itself
  }
  __device__ __forceinline__ float value(const Piece<T>& p, int i) const { return to_f32(p.e[i]); }
  __device__ __forceinline__ Piece<T> piece(int j) const {
    if constexpr (kLds) {
      Piece<T> p;
      p.raw = lds[j * kThreads + threadIdx.x];
      return p;
    }
    return fetch(j);
  }
  // f(tile, piece) of every piece of the thread; from memory with three on their way.
  template <typename F>
  __device__ __forceinline__ void pieces(F f) const {
    if constexpr (kLds) {
      for (int j = 0; j < tiles; ++j) f(j, piece(j));
    } else {
      Piece<T> p = fetch(0), q = fetch(min(1, tiles - 1)), r = fetch(min(2, tiles - 1));
#pragma unroll 1
      for (int j = 0; j < tiles; ++j) {
        const Piece<T> next = fetch(min(j + 3, tiles - 1));
        f(j, p);
        p = q, q = r, r = next;
      }
    }
  }
  // f(tile, piece) of the pieces in `marks`, a bit for each: a lane's first one, then its second and so on, so
  // that a wave runs f as often as its lane with the most: one row of 50,304 logits with 54 candidates 14.2 us, 15.0
  // where the pass itself calls f, as it does for a row in memory.
  static constexpr bool kMarks = kPlace != kInMemory;
  template <typename F>
  __device__ __forceinline__ void marked(uint32_t marks, F f) const {
    while (marks) {
      const int j = __ffs(marks) - 1;
      marks &= marks - 1;
      f(j, piece(j));
    }
  }
  // f of every piece, as pieces, in the passes that every row takes
  template <typename F>
  __device__ __forceinline__ void often(F f) const {
    if constexpr (kPlace == kInRegisters) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j)
        if (j < tiles) f(j, q[j]);
    } else {
      pieces(f);
    }
  }
  // f(index, value) of every logit of the thread
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    pieces([&](int j, const Piece<T>& p) __attribute__((always_inline)) {
      const uint32_t e = (static_cast<uint32_t>(j) * kThreads + threadIdx.x) * N;
#pragma unroll
      for (int i = 0; i < N; ++i) f(e + i, value(p, i));
    });
  }
};

// The first index at which the running sum of weight(index, value) exceeds of(total). `segs`: one
// double for 64 pieces of each tile, which may hold their sums already.
template <typename T, Place kPlace, typename W, typename F>
__device__ __forceinline__ uint32_t first_past(const Row<T, kPlace>& row, bool summed, double* segs, Shared& s, W weight, F of) {
  constexpr int N = kPiece<T>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = row.tiles * kWaves;
  auto mine = [&](int j, const Piece<T>& p) __attribute__((always_inline)) {
    const uint32_t e = (static_cast<uint32_t>(j) * kThreads + threadIdx.x) * N;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += weight(e + i, row.value(p, i));
    return static_cast<double>(sum);
  };
  __syncthreads();
  if (!summed)
    row.pieces([&](int j, const Piece<T>& p) __attribute__((always_inline)) {
      double sum = mine(j, p);
      if (__ballot(sum != 0.0) != 0) sum = wave_reduce(sum, [](double a, double b) { return a + b; });
      if (lane == 0) segs[j * kWaves + wave] = sum;
    });
  if (threadIdx.x == 0) s.found = 0x7FFFFFFF;
  __syncthreads();
  // a thread adds up `per` consecutive segments
  const int per = (n + kThreads - 1) / kThreads;
  double own = 0.0, total;
  for (int i = 0; i < per; ++i) {
    const int at = threadIdx.x * per + i;
    if (at < n) own += segs[at];
  }
  const double upto = block_scan(own, s.part, total);
  const double target = of(total);
  double run = upto - own;
  // the border's thread finds its segment; where rounding hides it, the last one with any weight does
  int seg = -1, last = -1;
  double before = 0.0, last_before = 0.0;
  for (int i = 0; i < per; ++i) {
    const int at = threadIdx.x * per + i;
    if (at >= n) break;
    const double w = segs[at];
    if (w > 0.0) last = at, last_before = run;
    if (seg < 0 && w > 0.0 && run + w > target) seg = at, before = run;
    run += w;
  }
  if (seg >= 0) atomicMin(&s.found, seg);
  __syncthreads();
  if (s.found == 0x7FFFFFFF) {
    __syncthreads();
    if (threadIdx.x == 0) s.found = -1;
    __syncthreads();
    if (last >= 0) atomicMax(&s.found, last);
    __syncthreads();
    seg = last;
    before = last_before;
  }
  if (seg >= 0 && seg == s.found) s.before = before;
  __syncthreads();
  const int at = s.found;
  if (at >= 0 && wave == at % kWaves) {
    const Piece<T> p = row.piece(at / kWaves);
    const double sum = mine(at / kWaves, p);
    const double inc = wave_scan(sum);
    double prev = __shfl_up(inc, 1);
    if (lane == 0) prev = 0.0;
    const uint64_t past = __ballot(sum > 0.0 && s.before + inc > target), any = __ballot(sum > 0.0);
    const int who = past ? __ffsll(static_cast<unsigned long long>(past)) - 1 : 63 - __clzll(any);
    if (lane == who) {
      const uint32_t e = (static_cast<uint32_t>(at / kWaves) * kThreads + threadIdx.x) * N;
      float sub = 0.f;
      int pick = -1;
      for (int i = 0; i < N; ++i) {
        const float w = weight(e + i, row.value(p, i));
        if (w > 0.f) {
          const bool done = pick >= 0 && s.before + prev + sub > target;
          if (!done) pick = i;
        }
        sub += w;
      }
      s.count = static_cast<int>(e + pick);
    }
  }
  __syncthreads();
  return at < 0 ? 0xFFFFFFFFu : static_cast<uint32_t>(s.count);
}

// Sorts n <= kList numbers of `list`, the largest first, behind them zeros up to the next power of two. A
// wave has 128 neighbours, so that only steps of 128 and more meet another wave's.
__device__ __forceinline__ void sort_list(uint64_t* list, int n) {
  int size = 128;
  while (size < n) size *= 2;
  for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = 0;
  __syncthreads();
  const int i = threadIdx.x;
#pragma unroll 1
  for (int width = 2; width <= size; width *= 2)
#pragma unroll 1
    for (int step = width / 2; step > 0; step /= 2) {
      if (step >= 128) __syncthreads();
      if (i < size / 2) {
        const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const uint64_t x = list[lo], y = list[hi];
        const bool turn = (x < y) == ((lo & width) == 0);
        list[lo] = turn ? y : x;
        list[hi] = turn ? x : y;
      }
      // a wave's accesses to LDS are in order; the compiler keeps them so
      asm volatile("" ::: "memory");
      if (step == 128) __syncthreads();
    }
  __syncthreads();
}

// The thread's candidates of a piece: those of its elements that `in` takes, behind the others' in `list`
// (kList at most; s.count counts on).
template <int N, typename In, typename Value>
__device__ __forceinline__ void append(uint64_t* list, Shared& s, uint32_t e, In in, Value value) {
  int many = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) many += in(i) ? 1 : 0;
  if (many == 0) return;
  int to = atomicAdd(&s.count, many);
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (in(i)) {
      if (to < kList) list[to] = static_cast<uint64_t>(key_of(value(i))) << 32 | (0xFFFFFFFFu - (e + i));
      ++to;
    }
}

__device__ __forceinline__ float setting(const Setting& s, int64_t r) {
  return s.each ? static_cast<const float*>(s.each)[r] : s.one;
}

// Choices, each with the times of both sides for 64 rows of 50,304 bf16 logits (measured at that size alone).
// Candidates that are ranked by counting: 54 of them (top-k 50, one row) 15.1 us, sorted 20.3; about 250 of them
// take the same both ways.
constexpr int kFew = 256;
// top-k up to which the threads' maxima bound the candidates, from there the pieces' (7 times as many counts, fewer
// candidates): k = 300 24.8 us with the threads' and 26.4 with the pieces', k = 400 28.1 and 26.9
constexpr int kByThread = 350;
// top-p alone: the threads' maxima that are tried. A nucleus among the first 380 or so tokens takes 29 us (with
// 640 maxima 39, without the try 43); one that ends later loses 2 us by it.
constexpr uint32_t kGuess = 320;

template <typename T, Place kPlace>
__global__ __launch_bounds__(kThreads, kPlace == kInMemory ? 8 : 4) void sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t dynamic[];  // segments of 64 pieces, then the row
  __shared__ Shared s;
  __shared__ __align__(16) uint64_t work[kList];  // the list, or bins
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x;
  double* segs = reinterpret_cast<double*>(dynamic);
  Row<T, kPlace> row;
  const T* const first_logit = static_cast<const T*>(a.logits) + r / a.inner * a.so + r % a.inner * a.si;
  // 1. the maximum
  const Largest<T> largest = row.open(first_logit, a.V, reinterpret_cast<u32x4*>(dynamic + a.seg_bytes));
  float mine = largest.value();
  const auto least_of = [](uint32_t x, uint32_t y) { return min(x, y); };
  const auto most_of = [](uint32_t x, uint32_t y) { return max(x, y); };
  const uint32_t most = block_reduce(largest.nan() ? 0xFFFFFFFFu : key_of(mine), s.part32, most_of);
  auto finish = [&](uint32_t token, float logprob) {
    if (t == 0) {
      a.tokens[r] = token == 0xFFFFFFFFu ? -1 : static_cast<int64_t>(token);
      if (a.logprobs) a.logprobs[r] = logprob;
    }
  };
  if (most == key_of(-INFINITY)) return finish(0xFFFFFFFFu, NAN);
  const float temperature = setting(a.temperature, r);
  const bool nan = most == 0xFFFFFFFFu;
  if (!nan && most == key_of(INFINITY)) row.level();
  const float top = nan || row.infinite ? 0.f : value_of(most);
  if (nan || !(temperature > 0.f)) {  // a NaN is the largest of all, like argmax; T = 0: the limit, the maximum
    uint32_t first = 0xFFFFFFFFu;
    row.each([&](uint32_t i, float v) { first = (nan ? v != v : v == top) ? min(first, i) : first; });
    return finish(block_reduce(first, s.part32, least_of), nan ? NAN : 0.f);
  }
  if (row.infinite) mine = mine == INFINITY ? 0.f : -INFINITY;
  const double scale = 1.4426950408889634 / fmin(static_cast<double>(temperature), 3.4028234663852886e38);
  const float fscale = static_cast<float>(fmin(scale, 3.4028234663852886e38));
  int64_t k = a.top_k.each ? static_cast<const int64_t*>(a.top_k.each)[r] : a.top_k.k;
  if (k <= 0 || k >= a.V) k = 0;
  const double p = setting(a.top_p, r);
  const bool by_p = p < 1.0;
  const double m = setting(a.min_p, r);
  // min-p's border as a logit: the least fp32 with (z - top) / T >= log m
  uint32_t least = 0;
  if (m > 0.0) {
    const double border = top + fmin(static_cast<double>(temperature), 3.4028234663852886e38) * log(fmin(m, 1.0));
    float z = static_cast<float>(border);
    if (static_cast<double>(z) < border) z = nextafterf(z, INFINITY);
    least = key_of(fminf(z, top));
  }
  float un = a.u[r];
  un = un > 0.f ? fminf(un, 0x1.fffffep-1f) : 0.f;
  const double u = un;
  // of the difference, so that the maximum's is 1 and equal logits' sums are whole numbers
  auto weight = [&](float v) __attribute__((always_inline)) { return __builtin_amdgcn_exp2f((v - top) * fscale); };
  auto bin_of = [&](float v) __attribute__((always_inline)) {
    return min(max(static_cast<int>(__float_as_uint(top - v) >> 16) - kFirstBin, 0), kBins - 1);
  };
  auto logprob = [&](float z, double sum) { return static_cast<float>((static_cast<double>(z) - top) * 0.6931471805599453 * scale - log(sum)); };
  auto at_index = [&](uint32_t i) {
    const float v = to_f32(first_logit[i]);
    return row.infinite ? 0.f : v;
  };
  uint32_t* const bins = reinterpret_cast<uint32_t*>(work);
  // a thread's two bins, and what the earlier ones hold
  uint32_t own[2], prior[2];
  auto scan_bins = [&]() __attribute__((always_inline)) {
    __syncthreads();
    uint32_t total;
    own[0] = own[1] = 0;
    if (2 * t < kBins) own[0] = bins[2 * t], own[1] = bins[2 * t + 1];
    const uint32_t upto = block_scan(own[0] + own[1], s.part32, total);
    prior[0] = upto - own[0] - own[1];
    prior[1] = upto - own[1];
  };
  auto clear_bins = [&]() __attribute__((always_inline)) {
    __syncthreads();
    for (int i = t; i < kBins; i += kThreads) bins[i] = 0;
    if (t == 0) s.found = kBins - 1, s.count = 0;
    __syncthreads();
  };

  // 2. the sum of all, and the candidates. With top-k no token of a bin behind that of the k-th largest of
  // the threads' maxima is kept; top-p alone may reach further than its guess.
  // For a larger k it takes the pieces' maxima.
  const bool by_piece = k > kByThread;
  const uint32_t most_k = by_piece ? static_cast<uint32_t>(min(int64_t(1800), a.V / kPiece<T>)) : kByThread;
  const uint32_t reach = k > 0 ? (k <= most_k ? static_cast<uint32_t>(k) : 0) : by_p && least == 0 ? kGuess : 0;
  const bool guess = reach > 0 && k == 0;
  clear_bins();
  float cut = -INFINITY;
  if (reach > 0) {
    if (by_piece)
      row.often([&](int, const Piece<T>& q) __attribute__((always_inline)) {
        Largest<T> l;
        l.take(q);
        atomicAdd(&bins[bin_of(l.value())], 1u);
      });
    else
      atomicAdd(&bins[bin_of(mine)], 1u);
    scan_bins();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if ((own[i] != 0) & (prior[i] < reach) & (prior[i] + own[i] >= reach)) s.found = 2 * t + i;
    __syncthreads();
    // the bin's end as a logit, or one below (a distance rounds)
    const int bound = s.found;
    if (bound < kBins - 1) {
      const float z = top - __uint_as_float(static_cast<uint32_t>(kFirstBin + bound + 1) << 16);
      cut = nextafterf(z, -INFINITY);
    }
  }
  // top-p's mass is that of all top-k tokens, those below min-p's border among them
  if (least > 0 && !(by_p && k > 0)) cut = fmaxf(cut, value_of(least));
  const bool listed = reach > 0 || (least > 0 && !(by_p && k > 0));
  cut = listed ? fmaxf(cut, -3.4028234663852886e38f) : INFINITY;
  // with no filter the sums of 64 pieces are all it takes to draw
  const bool free = !listed && k == 0 && !by_p && least == 0;
  double sum = 0.0, high = 0.0;
  uint32_t marks = 0;
  auto add = [&](int j, const Piece<T>& q) __attribute__((always_inline)) {
    append<kPiece<T>>(work, s, (static_cast<uint32_t>(j) * kThreads + t) * kPiece<T>, [&](int i) { return row.value(q, i) >= cut; },
                      [&](int i) { return row.value(q, i); });
  };
  row.often([&](int j, const Piece<T>& q) __attribute__((always_inline)) {
    constexpr int N = kPiece<T>;
    float few = 0.f;
    bool any = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float v = row.value(q, i);
      few += weight(v);
      any |= v >= cut;
    }
    sum += few;
    if constexpr (Row<T, kPlace>::kMarks) marks |= any ? 1u << j : 0u;
    if (any & (guess | !Row<T, kPlace>::kMarks)) {
      if (guess) {
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) part += row.value(q, i) >= cut ? weight(row.value(q, i)) : 0.f;
        high += part;
      } else {
        add(j, q);
      }
    }
    if (free) {
      const double part = wave_reduce(static_cast<double>(few), [](double a, double b) { return a + b; });
      if ((t & 63) == 0) segs[j * kWaves + (t >> 6)] = part;
    }
  });
  if (!guess) row.marked(marks, add);
  const double all = block_sum(sum, s);
  // a guess is listed if the nucleus ends in it
  const bool hit = !guess || block_sum(high, s) >= p * all;
  if (guess && hit) {
    if constexpr (Row<T, kPlace>::kMarks)
      row.marked(marks, add);
    else
      row.pieces([&](int j, const Piece<T>& q) __attribute__((always_inline)) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < kPiece<T>; ++i) any |= row.value(q, i) >= cut;
        if (any) add(j, q);
      });
    __syncthreads();
  }
  const int n = s.count;
  auto fixed = [&](uint64_t c) __attribute__((always_inline)) {  // a candidate's weight in 2^-44
    const double y = fmax((static_cast<double>(value_of(static_cast<uint32_t>(c >> 32))) - top) * scale, -1000.0);
    const double whole = rint(y);
    const uint64_t mant = static_cast<uint64_t>(__builtin_amdgcn_exp2f(static_cast<float>(y - whole)) * 0x1p23f);
    const int shift = static_cast<int>(whole) + 21;  // 44 - 23
    return shift >= 0 ? mant << (shift & 31) : mant >> min(-shift, 63);
  };
  bool complete = listed && hit && n <= kList;
  if (complete && guess) {  // (in the list's own numbers too)
    uint64_t w = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) w += t + i * kThreads < n ? fixed(work[t + i * kThreads]) : 0;
    complete = static_cast<double>(block_reduce(w, s.part64, [](uint64_t x, uint64_t y) { return x + y; })) >= p * (all * 0x1p44);
  }
  if (complete && n <= kFew) {
    // a thread a candidate: its rank, and the mass in front of it, by looking at all
    struct Pair {
      uint64_t c, w;
    };
    Pair* const pair = reinterpret_cast<Pair*>(work) + kList / 4;  // behind the candidates
    if (t < n) pair[t] = Pair{work[t], fixed(work[t])};
    __syncthreads();
    const int lanes = n <= 64 ? 16 : n <= 128 ? 8 : 4, who = t / lanes;
    // over a candidate's lanes
    auto together = [&](uint64_t v) __attribute__((always_inline)) {
      v += moved<0xB1>(v);
      v += moved<0x4E>(v);
      if (lanes >= 8) v += moved<0x141>(v);
      if (lanes == 16) v += moved<0x140>(v);
      return v;
    };
    const Pair own_pair = who < n ? pair[who] : Pair{0, 0};
    const uint64_t c = own_pair.c, w = own_pair.w;
    uint64_t rank = 0, before = 0;
#pragma unroll 2
    for (int i = t % lanes; i < n; i += lanes) {
      const Pair q = pair[i];
      const uint64_t mask = q.c > c ? ~uint64_t(0) : 0;
      rank -= mask;
      before += q.w & mask;
    }
    rank = together(rank);
    before = together(before);
    const uint64_t last = k > 0 && k < n ? static_cast<uint64_t>(k) - 1 : n - 1;
    if ((who < n) & (rank == last)) s.mass = before + w;  // of the first k
    __syncthreads();
    const double mass = k > 0 ? static_cast<double>(s.mass) : all * 0x1p44;
    const uint32_t index = 0xFFFFFFFFu - static_cast<uint32_t>(c);
    const bool kept = (who < n) & ((k == 0) | (rank < static_cast<uint64_t>(k))) & (static_cast<uint32_t>(c >> 32) >= least) &
                      (!by_p | (rank == 0) | (static_cast<double>(before) < p * mass));
    const uint64_t kept_w = w & (kept ? ~uint64_t(0) : 0);
    if ((who < n) & (t % lanes == 0)) pair[who] = Pair{index, kept_w};
    __syncthreads();
    uint64_t upto = 0, total = 0;
#pragma unroll 2
    for (int i = t % lanes; i < n; i += lanes) {
      const Pair q = pair[i];
      upto += q.c <= index ? q.w : 0;
      total += q.w;
    }
    upto = together(upto);
    total = together(total);
    const uint64_t target = static_cast<uint64_t>(u * static_cast<double>(total));  // running sums above it
    if ((t % lanes == 0) & (kept_w != 0) & (upto > target) & (upto - kept_w <= target)) {
      a.tokens[r] = index;
      if (a.logprobs) a.logprobs[r] = logprob(at_index(index), all);
    }
    return;
  }
  if (complete) {
    sort_list(work, n);
    // a thread has two neighbours of the order
    uint64_t w[2];
    uint32_t index[2], keys[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint64_t c = 2 * t + i < n ? work[2 * t + i] : 0;
      keys[i] = static_cast<uint32_t>(c >> 32);
      index[i] = 0xFFFFFFFFu - static_cast<uint32_t>(c);
      w[i] = 2 * t + i < n ? fixed(c) : 0;
    }
    uint64_t total;
    const uint64_t upto = block_scan(w[0] + w[1], s.part64, total);
    const uint64_t before[2] = {upto - w[0] - w[1], upto - w[1]};
    double mass = all * 0x1p44;
    if (k > 0 && by_p) {
      uint64_t head = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) head += 2 * t + i < k ? w[i] : 0;
      mass = static_cast<double>(block_reduce(head, s.part64, [](uint64_t x, uint64_t y) { return x + y; }));
    }
    const uint32_t span = static_cast<uint32_t>((a.V + kThreads - 1) / kThreads);
    uint64_t* const segment = work + kList / 2;
    __syncthreads();
    segment[t] = 0;
    if (t == 0) s.found = 0x7FFFFFFF;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // without branches: with && and an if, hipcc of ROCm 7.2 lost the store of the 0 in some instances
      const int at = 2 * t + i;
      const bool kept = (at < n) & ((k == 0) | (at < k)) & (keys[i] >= least) &
                        (!by_p | (at == 0) | (static_cast<double>(before[i]) < p * mass));
      w[i] &= kept ? ~uint64_t(0) : 0;
      if (w[i]) atomicAdd(reinterpret_cast<unsigned long long*>(&segment[index[i] / span]), w[i]);
    }
    __syncthreads();
    const uint64_t part = segment[t];
    const uint64_t end = block_scan(part, s.part64, total);
    const uint64_t target = static_cast<uint64_t>(u * static_cast<double>(total));
    if ((part != 0) & (end > target) & (end - part <= target)) {
      s.found = t;
      s.mass = end - part;
    }
    // the border's span: the kept tokens in it, by place
    uint64_t* const place = work;
    __syncthreads();
    const uint32_t first = static_cast<uint32_t>(s.found) * span;
    for (uint32_t i = t; i < span; i += kThreads) place[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (w[i] && index[i] / span == static_cast<uint32_t>(s.found)) place[index[i] - first] = w[i];
    __syncthreads();
    const uint64_t x = t < static_cast<int>(span) ? place[t] : 0;
    uint64_t unused;
    const uint64_t run = s.mass + block_scan(x, s.part64, unused);
    if ((x != 0) & (run > target) & (run - x <= target)) {
      const uint32_t token = first + t;
      a.tokens[r] = token;
      if (a.logprobs) a.logprobs[r] = logprob(at_index(token), all);
    }
    return;
  }

  // 3. otherwise. What is kept: (key, index) from `border` on. Stage 0 finds top-k's border, 1 top-p's, 2 adds
  // min-p's and draws.
  auto composite = [](uint32_t key, uint32_t i) __attribute__((always_inline)) {
    return static_cast<uint64_t>(key) << 32 | (0xFFFFFFFFu - i);
  };
  constexpr int kShift = kKeyShift<T>;
  uint64_t border = 0;
  double mass = all;  // of the first k
#pragma unroll 1
  for (int stage = k > 0 ? 0 : by_p ? 1 : 2;; ++stage) {
    if (stage == 1 && !by_p) stage = 2;
    if (stage == 2) border = max(border, static_cast<uint64_t>(least) << 32);
    uint32_t key = 0;
    bool tie = false;
    double take = 0.0;
    if (stage < 2) {
      const bool by_mass = stage == 1;
      const double goal = by_mass ? fmax(p, 0.0) * mass : static_cast<double>(k);
      // bins of the distances in whole numbers: tokens, or mass in 2^-31 of the row's
      const float unit = by_mass ? static_cast<float>(0x1p31 / all) : 0.f;
      auto amount = [&](float v) __attribute__((always_inline)) { return by_mass ? weight(v) : 1.f; };
      clear_bins();
      row.each([&](uint32_t, float v) __attribute__((always_inline)) {
        atomicAdd(&bins[bin_of(v)], by_mass ? static_cast<uint32_t>(weight(v) * unit) : 1u);
      });
      scan_bins();
      const uint32_t aim = static_cast<uint32_t>(by_mass ? goal * (0x1p31 / all) : goal);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if ((own[i] != 0) & (prior[i] <= aim) & (prior[i] + own[i] >= aim)) atomicMin(&s.found, 2 * t + i);
      __syncthreads();
      // the bin in which the running amount reaches the goal, by exact sums (up, then down: each way at most
      // once over the bins, whatever the sums round to), and its tokens
      int bin = s.found, held;
      double above;
      for (bool down = false;;) {
        // a bin's distances, from the upper half of its number
        const float from = bin > 0 ? __uint_as_float(static_cast<uint32_t>(kFirstBin + bin) << 16) : -1.f;
        const float to = bin < kBins - 1 ? __uint_as_float(static_cast<uint32_t>(kFirstBin + bin + 1) << 16) : NAN;
        double x = 0.0, y = 0.0;
        __syncthreads();
        if (t == 0) s.count = 0;
        __syncthreads();
        auto list = [&](int j, const Piece<T>& q) __attribute__((always_inline)) {
          append<kPiece<T>>(work, s, (static_cast<uint32_t>(j) * kThreads + t) * kPiece<T>,
                            [&](int i) { return !(top - row.value(q, i) < from || top - row.value(q, i) >= to); },
                            [&](int i) { return row.value(q, i); });
        };
        uint32_t found = 0;
        row.pieces([&](int j, const Piece<T>& q) __attribute__((always_inline)) {
          constexpr int N = kPiece<T>;
          float front = 0.f, here = 0.f;
          bool any = false;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float v = row.value(q, i), d = top - v;
            const float w = d >= to ? 0.f : amount(v);
            front += d < from ? w : 0.f;
            here += d < from ? 0.f : w;
            any |= !(d < from || d >= to);
          }
          x += front;
          y += here;
          if constexpr (Row<T, kPlace>::kMarks)
            found |= any ? 1u << j : 0u;
          else if (any)
            list(j, q);
        });
        row.marked(found, list);
        above = block_sum(x, s);
        const double in = block_sum(y, s);
        held = s.count;
        if (!down && above + in < goal && bin < kBins - 1) {
          ++bin;
        } else if (bin > 0 && (in == 0.0 || above >= goal)) {
          --bin;
          down = true;
        } else {
          break;
        }
      }
      if (held <= kList) {
        // in their order, the last one with less than the goal in front of it
        sort_list(work, held);
        uint64_t c[2];
        double w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          c[i] = 2 * t + i < held ? work[2 * t + i] : 0;
          w[i] = 2 * t + i < held ? amount(value_of(static_cast<uint32_t>(c[i] >> 32))) : 0.f;
        }
        double total;
        const double upto = above + block_scan(w[0] + w[1], s.part, total);
        // (the bin's first token always: the sums may round past the goal)
        uint64_t lowest = ~uint64_t(0);
        if ((2 * t < held) & ((t == 0) | (upto - w[0] - w[1] < goal))) lowest = c[0];
        if ((2 * t + 1 < held) & (upto - w[1] < goal)) lowest = c[1];
        border = max(border, block_reduce(lowest, s.part64, [](uint64_t x, uint64_t y) { return min(x, y); }));
      } else {
        // too many, most of them equal: the largest key whose tokens and those above reach the goal, by
        // bisection, and of the tokens with that key as many as it takes, by index
        uint32_t lo = 0xFFFFFFFFu, hi = 0;
        row.each([&](uint32_t, float v) __attribute__((always_inline)) {
          if (bin_of(v) == bin) lo = min(lo, key_of(v) >> kShift), hi = max(hi, key_of(v) >> kShift);
        });
        lo = block_reduce(lo, s.part32, least_of);
        hi = block_reduce(hi, s.part32, most_of);
        double over;
        for (;;) {
          const uint32_t from = lo < hi ? lo + (hi - lo + 1) / 2 : lo + 1;
          double x = 0.0;
          row.each([&](uint32_t, float v) __attribute__((always_inline)) {
            if (bin_of(v) == bin && key_of(v) >> kShift >= from) x += amount(v);
          });
          over = above + block_sum(x, s);
          if (lo >= hi) break;
          if (over >= goal)
            lo = from;
          else
            hi = from - 1;
        }
        uint32_t ties = 0;
        row.each([&](uint32_t, float v) __attribute__((always_inline)) {
          if (key_of(v) >> kShift == lo) key = key_of(v), ++ties;
        });
        key = block_reduce(key, s.part32, most_of);
        ties = block_reduce(ties, s.part32, [](uint32_t x, uint32_t y) { return x + y; });
        take = fmax(1.0, ceil((goal - over) / amount(value_of(key))));
        border = max(border, static_cast<uint64_t>(key) << 32);
        tie = take < ties;
      }
    }
    if (stage == 2 || tie) {
      // the border's logit, and the last index that is kept of those with it (the border 0 keeps all)
      const float equal = tie ? value_of(key) : border ? value_of(static_cast<uint32_t>(border >> 32)) : -INFINITY;
      const uint32_t upto_index = 0xFFFFFFFFu - static_cast<uint32_t>(border);
      const uint32_t i = first_past(
          row, free, segs, s,
          [&](uint32_t at, float v) __attribute__((always_inline)) {
            if (tie) return v == equal ? 1.f : 0.f;
            return ((v >= equal) & !((v == equal) & (at > upto_index))) ? weight(v) : 0.f;
          },
          [&](double total) { return tie ? take - 0.5 : u * total; });
      if (stage == 2) return finish(i, i == 0xFFFFFFFFu ? NAN : logprob(at_index(i), all));
      border = max(border, composite(key, i));
    }
    if (stage == 0 && by_p) {
      double x = 0.0;
      row.each([&](uint32_t i, float v) __attribute__((always_inline)) {
        if (composite(key_of(v), i) >= border) x += weight(v);
      });
      mass = block_sum(x, s);
    }
  }
}

}  // namespace
}  // namespace lema

using namespace lema;

extern "C" int lema_sample(const void* logits, int32_t dtype, int64_t rows, int64_t inner, int64_t V, int64_t so,
                           int64_t si, const float* u, const float* temperatures, float temperature,
                           const int64_t* top_ks, int64_t top_k, const float* top_ps, float top_p,
                           const float* min_ps, float min_p, int64_t* tokens, float* logprobs, void* stream) {
  clear_error();
  const int size = dtype_size(dtype);
  LEMA_REQUIRE(size != 0, "unknown type %d", dtype);
  LEMA_REQUIRE(V > 0 && V <= kMaxVocab, "a vocabulary of %lld: 1 to %lld", (long long)V, (long long)kMaxVocab);
  LEMA_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && inner > 0, "bad number of rows %lld", (long long)rows);
  if (rows == 0) return LEMA_OK;
  LEMA_REQUIRE(logits && u && tokens && aligned(logits, size) && aligned(tokens, 8), "bad pointer");
  const int64_t pieces = (V * size + 15) / 16, tiles = (pieces + kThreads - 1) / kThreads;
  const SampleArgs a{logits, V, inner, so, si, u,
                     {temperatures, temperature, 0},
                     {top_ks, 0.f, static_cast<int32_t>(top_k < 0 || top_k > V ? 0 : top_k)},
                     {top_ps, top_p, 0},
                     {min_ps, min_p, 0},
                     tokens, logprobs, tiles * kWaves * 8};
  const int64_t row_bytes = tiles * kThreads * 16;
  const Place place = row_bytes <= kRowBytes ? kInLds : tiles <= 16 ? kInRegisters : kInMemory;
  const uint32_t lds = static_cast<uint32_t>(a.seg_bytes + (place == kInLds ? row_bytes : 0));
  const dim3 grid(static_cast<uint32_t>(rows)), threads(kThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto kernel) -> int {
    LEMA_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(lds)));
    kernel<<<grid, threads, lds, st>>>(a);
    return launch_status("sample_kernel");
  };
  auto of = [&](auto t) {
    using T = decltype(t);
    return place == kInLds       ? go(sample_kernel<T, kInLds>)
           : place == kInRegisters ? go(sample_kernel<T, kInRegisters>)
                                   : go(sample_kernel<T, kInMemory>);
  };
  return dtype == LEMA_F32 ? of(0.f) : dtype == LEMA_F16 ? of(_Float16{}) : of(Bf16{});
}
