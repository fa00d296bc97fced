// Embedding lookup with a scale, and its gradient by sorted tokens.
//
// Forward: out row i = round(scale * table row ids[i]); a copy of the bits where scale is 1.
//
// Backward: gw row v = round(scale * sum of gy row i over the positions i with ids[i] = v), every row
// of the table written, zeros where a token does not occur. Positions are first put in the order
// of (token, position), which makes the sums' order fixed, without atomics on values:
//   count    per span of positions, how many fall into each of up to 1024 buckets of tokens
//            (the token's high bits);
//   scatter  each span puts its positions, in order, into the buckets;
//   order    each bucket orders its positions by token, and notes where each token's start. Of up to
//            7168 positions each bucket picks its own, and there is no count and no scatter;
//   sum      a wavefront per (token, 512 columns) adds up to 32 rows. A longer list would
//            keep one wavefront busy while the others end, so its whole tiles of 16 or 64 positions are
//            summed by wavefronts of their own, in the same launch, in fp32;
//   join     a workgroup per (long list, 512 columns) adds its tiles and its ragged ends.
// A wavefront keeps its own cursors, so a place is a ballot per bit of the digit and needs no
// atomics. gy is read once and the table's gradient written once, which bounds the work (HBM);
// the ordering costs one or three short launches.
#include "elem.h"

namespace lema {
namespace {

constexpr int kBuckets = 1024;      // at most, of 1 << row_bits tokens each
constexpr int kMaxRowBits = 10;     // so at most 2^20 tokens
constexpr int kSpanStep = 1024;     // a span is a multiple of it: 16 wavefronts of 64
constexpr int kLong = 32;           // positions of a token that one wavefront adds up
// Up to this many positions every bucket reads all of them, 15 a lane at once: 5003 of a table of 32,003
// took 12 us so and 16 in three launches, whose host side is 5 us longer (a pass with its gradient 87
// and 95 us). It is what leaves a bucket's items and cursors within 64 KB; the two do not cross below: the
// whole gradient took 5.6 to 7.6 us less in one launch of 200 to 7168 positions of a table of 256, 2.2 to
// 3.6 of 50,304, and 0.8 to 2.7 of 2^20, whose 1024 buckets each read all positions.
constexpr int64_t kShort = 7168;
constexpr int kCols = 512;          // columns of a wavefront, 8 a lane

__device__ __forceinline__ int wave_index() {
  return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
}

// C slices of 512 columns of a row, as they come from memory, a load's units next to each other.
template <typename T, int C, int kKind>
struct RawSlices : RowPart<T, kKind, C * 8> {
  typedef RowPart<T, kKind, C * 8> Part;
  static __device__ __forceinline__ auto columns(int64_t c0, int lane) {
    return [=](int i) { return c0 + i * 64 + lane * kUnit<T, kKind>; };
  }
  template <bool kStream = false>
  __device__ __forceinline__ void fetch(const T* row, int64_t c0, int64_t D, int lane) {
    Part::template fetch<kStream>(row, D, columns(c0, lane));
  }
  __device__ __forceinline__ void settle(int64_t c0, int64_t D, int lane) { Part::settle(D, columns(c0, lane)); }
  template <bool kStream>
  __device__ __forceinline__ void store(T* row, int64_t c0, int64_t D, int lane) const {
    Part::template store<kStream>(row, D, columns(c0, lane));
  }
  __device__ __forceinline__ float at(int k) const { return this->get(k); }
};

// fp32 sums of C slices as a row's elements.
template <typename T, int C, int kKind, bool kStream>
__device__ __forceinline__ void store_slices(T* row, int64_t c0, int64_t D, int lane, const float (&v)[C * 8]) {
  RawSlices<T, C, kKind> r;
#pragma unroll
  for (int k = 0; k < C * 8; ++k) r.set(k, v[k]);
  r.template store<kStream>(row, c0, D, lane);
}

// One wavefront per (position, 512 columns).
template <typename T, int kKind, bool kScale, bool kStream>
__global__ __launch_bounds__(256) void embed_kernel(const T* table, int64_t vocab, int64_t D,
                                                    const int64_t* ids, int64_t n, int slices,
                                                    float scale, T* out) {
  const int lane = threadIdx.x & 63;
  const int64_t u = block_index() * 4 + wave_index();
  const int64_t i = u / slices;
  if (i >= n) return;
  const int64_t c0 = (u - i * slices) * kCols, id = ids[i];
  const bool ok = id >= 0 && id < vocab;
  RawSlices<T, 1, kKind> r;
  r.fetch(table + (ok ? id : 0) * D, c0, D, lane);
  r.settle(c0, D, lane);
  if constexpr (kScale) {
#pragma unroll
    for (int k = 0; k < 8; ++k) r.set(k, r.at(k) * scale);
  }
  if (!ok) r.clear();
  r.template store<kStream>(out + i * D, c0, D, lane);
}

struct Order {            // what the ordering kernels share
  const int64_t* ids;
  int64_t n, vocab, padding;
  int row_bits, buckets, spans, tile;
  int64_t span;
  uint32_t* counts;       // [spans, kBuckets]
  uint32_t* bucket_at;    // [kBuckets + 1]: where a bucket's positions start
  uint32_t* item_pos;     // [n] positions by bucket
  uint32_t* item_id;      // [n] their tokens
  uint32_t* perm;         // [n] positions by (token, position)
  uint32_t* token;        // [n] their tokens
  uint32_t* start;        // [vocab + 1]
  bool pick;              // n is up to kShort: what follows is not filled
  uint32_t* long_count;   // lists of more than kLong
  uint32_t* long_list;    // their tokens, starts and ends, in no order
};

// Token of position i, or -1 for one that takes no part.
__device__ __forceinline__ int64_t token_of(const Order& o, int64_t i, int64_t end) {
  const int64_t id = i < end ? o.ids[i] : -1;
  return id >= 0 && id < o.vocab && id != o.padding ? id : -1;
}

// Lanes whose `bits`-bit digit equals this lane's, among the lanes of `live`.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, uint64_t live) {
  uint64_t m = live;
  for (int b = 0; b < bits; ++b) {
    const bool one = (digit >> b) & 1;
    const uint64_t s = __ballot(one);
    m &= one ? s : ~s;
  }
  return m;
}

// The place of each live lane's item from its digit's cursor, lanes in order; every lane of the
// wavefront calls it.
__device__ __forceinline__ uint32_t take_place(uint32_t* cursors, uint32_t digit, bool live, int bits,
                                               int lane) {
  const uint64_t m = same_digit(digit, bits, __ballot(live));
  const uint32_t rank = __popcll(m & ((uint64_t(1) << lane) - 1));
  uint32_t at = 0;
  if (live) at = cursors[digit] + rank;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // every lane has read before one writes
  if (live && rank == 0) cursors[digit] = at + __popcll(m);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return at;
}

// Batches of 64 items that a wavefront has on their way while it works on as many. More make the
// kernels' code longer than what they save: they are short, and run cold.
constexpr int kHeld = 4;

__global__ __launch_bounds__(1024) void embed_count_kernel(Order o) {
  __shared__ uint32_t hist[kBuckets];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t at = blockIdx.x * o.span, end = min(at + o.span, o.n);
  for (int64_t i = at + threadIdx.x; i < end; i += 1024) {
    const int64_t id = token_of(o, i, end);
    if (id >= 0) atomicAdd(&hist[id >> o.row_bits], 1u);
  }
  __syncthreads();
  o.counts[static_cast<int64_t>(blockIdx.x) * kBuckets + threadIdx.x] = hist[threadIdx.x];
}

// Exclusive sum over a workgroup's threads (kWaves wavefronts); `red` holds kWaves words.
template <int kWaves>
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t* red) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t t = __shfl_up(s, d);
    if (lane >= d) s += t;
  }
  if (lane == 63) red[w] = s;
  __syncthreads();
  uint32_t base = 0;
  for (int i = 0; i < w; ++i) base += red[i];
  return base + s - v;
}

// A span's positions into the buckets: 16 wavefronts on consecutive sixteenths of it.
__global__ __launch_bounds__(1024) void embed_scatter_kernel(Order o) {
  __shared__ uint32_t cur[16][kBuckets];
  __shared__ uint32_t red[16];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int64_t part = o.span / 16;
  const int64_t at = blockIdx.x * o.span + w * part;
  const int64_t end = min(at + part, o.n);
  // A batch's tokens, kNone where there is none; f(i0, tokens) for each batch in order.
  constexpr uint32_t kNone = ~0u;
  const auto fetch = [&](int64_t i0, uint32_t (&id)[kHeld]) {
#pragma unroll
    for (int u = 0; u < kHeld; ++u) id[u] = static_cast<uint32_t>(token_of(o, i0 + u * 64 + lane, end));
  };
  const auto each = [&](auto f) {
    uint32_t id[kHeld], next[kHeld];
    fetch(at, next);
    for (int64_t i0 = at; i0 < end; i0 += kHeld * 64) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u) id[u] = next[u];
      fetch(i0 + kHeld * 64, next);
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (i0 + u * 64 < end) f(i0 + u * 64, id[u]);
    }
  };
  for (int k = 0; k < 16; ++k) cur[k][t] = 0;
  __syncthreads();
  each([&](int64_t, uint32_t id) {
    if (id != kNone) atomicAdd(&cur[w][id >> o.row_bits], 1u);
  });
  // thread t: bucket t's positions in all spans, and in the spans before this one
  uint32_t all = 0, before = 0;
  for (int s0 = 0; s0 < o.spans; s0 += 32) {
    uint32_t c[32];
#pragma unroll
    for (int u = 0; u < 32; ++u)
      c[u] = o.counts[static_cast<int64_t>(s0 + u < o.spans ? s0 + u : s0) * kBuckets + t];
#pragma unroll
    for (int u = 0; u < 32; ++u) {
      if (s0 + u < o.spans) all += c[u];
      if (s0 + u < static_cast<int>(blockIdx.x)) before += c[u];
    }
  }
  uint32_t base = group_scan<16>(all, red);  // its barrier also ends the counting above
  if (blockIdx.x == 0) {
    if (t == 0) *o.long_count = 0;
    o.bucket_at[t] = base;
    if (t == kBuckets - 1) o.bucket_at[kBuckets] = base + all;
  }
  base += before;
  for (int k = 0; k < 16; ++k) {
    const uint32_t c = cur[k][t];
    cur[k][t] = base;
    base += c;
  }
  __syncthreads();
  each([&](int64_t i0, uint32_t id) {
    const bool live = id != kNone;
    const uint32_t to = take_place(cur[w], live ? id >> o.row_bits : 0u, live, 10, lane);
    if (live) {
      o.item_pos[to] = static_cast<uint32_t>(i0 + lane);
      o.item_id[to] = id;
    }
  });
}

// One workgroup per bucket: its positions ordered by token, and where each token's start. With
// kPick it first picks them out of all positions, in order, each wavefront out of an eighth.
template <bool kPick>
__global__ __launch_bounds__(512) void embed_order_kernel(Order o) {
  extern __shared__ uint32_t cursors[];  // [8][rows]
  __shared__ uint32_t red[8], inside[8], below[8];
  __shared__ uint32_t items[kPick ? kShort : 1];  // position, the token's low bits above 16
  const int t = threadIdx.x, lane = t & 63, w = wave_index();
  const int rows = 1 << o.row_bits;
  uint32_t* const cur = cursors + w * rows;
  const uint32_t first = static_cast<uint32_t>(blockIdx.x) << o.row_bits;  // the bucket's first token
  uint32_t b0, b1;
  if constexpr (kPick) {
    constexpr int kBatches = kShort / 512;
    const int64_t eighth = (o.n / 512 + 1) * 64, from = min(w * eighth, o.n), to = min(from + eighth, o.n);
    uint32_t id[kBatches + 1];
#pragma unroll
    for (int u = 0; u <= kBatches; ++u) id[u] = static_cast<uint32_t>(token_of(o, from + u * 64 + lane, to));
    uint32_t mine = 0, less = 0;
#pragma unroll
    for (int u = 0; u <= kBatches; ++u) {
      mine += __popcll(__ballot(id[u] - first < static_cast<uint32_t>(rows)));
      less += __popcll(__ballot(id[u] < first));
    }
    if (lane == 0) {
      inside[w] = mine;
      below[w] = less;
    }
    __syncthreads();
    uint32_t at = 0;
    b0 = 0, b1 = 0;
    for (int k = 0; k < 8; ++k) {
      if (k < w) at += inside[k];
      b0 += below[k];
      b1 += inside[k];
    }
    b1 += b0;
#pragma unroll
    for (int u = 0; u <= kBatches; ++u) {
      const bool in = id[u] - first < static_cast<uint32_t>(rows);
      const uint64_t m = __ballot(in);
      if (in)
        items[at + __popcll(m & ((uint64_t(1) << lane) - 1))] =
            static_cast<uint32_t>(from + u * 64 + lane) | (id[u] - first) << 16;
      at += __popcll(m);
    }
  } else {
    b0 = o.bucket_at[blockIdx.x], b1 = o.bucket_at[blockIdx.x + 1];
  }
  const uint32_t part = ((b1 - b0) / 512 + 1) * 64;  // 8 parts cover the bucket
  const uint32_t at = min(b0 + w * part, b1), end = min(at + part, b1);
  // f(i0, tokens, positions) for each batch in order
  const auto each = [&](auto f) {
    uint32_t id[kHeld], pos[kHeld], next_id[kHeld], next_pos[kHeld];
    const auto fetch = [&](uint32_t i0) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        const uint32_t i = min(i0 + u * 64 + lane, end - 1);
        if constexpr (kPick) {
          next_id[u] = first + (items[i - b0] >> 16);
          next_pos[u] = items[i - b0] & 0xffff;
        } else {
          next_id[u] = o.item_id[i];
          next_pos[u] = o.item_pos[i];
        }
      }
    };
    if (at < end) fetch(at);
    for (uint32_t i0 = at; i0 < end; i0 += kHeld * 64) {
#pragma unroll
      for (int u = 0; u < kHeld; ++u) {
        id[u] = next_id[u];
        pos[u] = next_pos[u];
      }
      fetch(i0 + kHeld * 64);
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (i0 + u * 64 < end) f(i0 + u * 64, id[u], pos[u]);
    }
  };
  for (int k = t; k < 8 * rows; k += 512) cursors[k] = 0;
  __syncthreads();
  // counted a digit at a time: 64 lanes of one frequent token would queue for its word
  each([&](uint32_t i0, uint32_t id, uint32_t) {
    const bool live = i0 + lane < end;
    const uint64_t m = same_digit(id & (rows - 1), o.row_bits, __ballot(live));
    if (live && (m & ((uint64_t(1) << lane) - 1)) == 0) cur[id & (rows - 1)] += __popcll(m);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  });
  __syncthreads();
  uint32_t mine[2] = {0, 0};  // tokens 2 t and 2 t + 1 of the bucket
  for (int j = 0; j < 2; ++j)
    if (2 * t + j < rows)
      for (int k = 0; k < 8; ++k) mine[j] += cursors[k * rows + 2 * t + j];
  uint32_t base = b0 + group_scan<8>(mine[0] + mine[1], red);
  for (int j = 0; j < 2; ++j) {
    const int r = 2 * t + j;
    if (r >= rows) break;
    const int64_t v = (static_cast<int64_t>(blockIdx.x) << o.row_bits) + r;
    if (v < o.vocab) {
      o.start[v] = base;
      if (v == o.vocab - 1) o.start[o.vocab] = b1;
      if (!kPick && mine[j] > kLong) {
        uint32_t* entry = o.long_list + 3 * atomicAdd(o.long_count, 1u);
        entry[0] = static_cast<uint32_t>(v);
        entry[1] = base;
        entry[2] = base + mine[j];
      }
    }
    for (int k = 0; k < 8; ++k) {
      const uint32_t c = cursors[k * rows + r];
      cursors[k * rows + r] = base;
      base += c;
    }
  }
  __syncthreads();
  each([&](uint32_t i0, uint32_t id, uint32_t pos) {
    const bool live = i0 + lane < end;
    const uint32_t to = take_place(cur, id & (rows - 1), live, o.row_bits, lane);
    if (live) {
      o.perm[to] = pos;
      o.token[to] = id;
    }
  });
}

// acc += gy rows perm[j], j in [j0, j1), in order: 64 positions read at once, 4 or 8 rows in flight.
template <typename T, int C, int kKind, bool kStream>
__device__ __forceinline__ void add_rows(const T* gy, const uint32_t* perm, uint32_t j0, uint32_t j1,
                                         int64_t c0, int64_t D, int lane, float (&acc)[C * 8]) {
  for (uint32_t j = j0; j < j1; j += 64) {
    const int m = min(64u, j1 - j);
    const uint32_t pos = perm[j + min(lane, m - 1)];
    constexpr int kRows = C == 1 ? 8 : 4;
    for (int i = 0; i < m; i += kRows) {
      RawSlices<T, C, kKind> v[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const uint32_t p = __builtin_amdgcn_readlane(pos, min(i + u, m - 1));
        if (u == 0 || i + u < m) v[u].template fetch<kStream>(gy + static_cast<int64_t>(p) * D, c0, D, lane);
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u)
        if (u == 0 || i + u < m) {
          v[u].settle(c0, D, lane);
#pragma unroll
          for (int k = 0; k < C * 8; ++k) acc[k] += v[u].at(k);
        }
    }
  }
}

// A tile's sums: whole slices, a lane's eight where the lane finds them, whatever column they are of.
__host__ __device__ inline int64_t padded_cols(int64_t D) { return (D + kCols - 1) / kCols * kCols; }

// One wavefront per (tile or token, C slices of 512 columns): the tiles come first. partial: [tiles,
// padded_cols(D)].
template <typename T, int C, int kKind, bool kStream>
__global__ __launch_bounds__(256) void embed_sum_kernel(Order o, const T* gy, int64_t D, int slices,
                                                        int64_t tiles, float scale, float* partial,
                                                        T* gw) {
  const int lane = threadIdx.x & 63;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + wave_index();
  const int64_t item = u / slices, c0 = (u - item * slices) * C * kCols;
  if (item >= tiles + o.vocab) return;
  float acc[C * 8];
#pragma unroll
  for (int k = 0; k < C * 8; ++k) acc[k] = 0.0f;
  if (item < tiles) {
    const uint32_t j0 = static_cast<uint32_t>(item) * o.tile;
    if (j0 + o.tile > o.start[o.vocab]) return;
    const uint32_t v = o.token[j0];
    if (o.token[j0 + o.tile - 1] != v || o.start[v + 1] - o.start[v] <= kLong) return;
    add_rows<T, C, kKind, kStream>(gy, o.perm, j0, j0 + o.tile, c0, D, lane, acc);
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c0 + c * kCols < D) {
        u32x4* at = reinterpret_cast<u32x4*>(partial + item * padded_cols(D) + c0 + c * kCols) + lane;
        const float* a = acc + c * 8;
        Piece<float> lo, hi;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          lo.e[k] = a[k];
          hi.e[k] = a[4 + k];
        }
        at[0] = lo.raw;
        at[64] = hi.raw;
      }
  } else {
    const int64_t v = item - tiles;
    const uint32_t j0 = o.start[v], j1 = o.start[v + 1];
    if (j1 - j0 > kLong) return;
    add_rows<T, C, kKind, kStream>(gy, o.perm, j0, j1, c0, D, lane, acc);
#pragma unroll
    for (int k = 0; k < C * 8; ++k) acc[k] *= scale;
    store_slices<T, C, kKind, kStream>(gw + v * D, c0, D, lane, acc);
  }
}

// One workgroup per (long list, 512 columns): the positions before the first whole tile, the tiles'
// sums and the positions after the last one, each dealt out to the 16 wavefronts, the tiles 4 at a time
// in flight: the most frequent token of 65,536 has about 120. 64 registers, so that a CU holds two
// workgroups.
template <typename T, int kKind, bool kStream>
__global__ __launch_bounds__(1024, 8) void embed_join_kernel(Order o, const T* gy, int64_t D, float scale,
                                                          const float* partial, T* gw) {
  __shared__ float sums[16][8][64];
  const int lane = threadIdx.x & 63;
  const uint32_t w = wave_index(), lists = o.pick ? (o.start[o.vocab] + kLong - 1) / kLong : *o.long_count;
  const int64_t c0 = static_cast<int64_t>(blockIdx.y) * kCols;
  for (uint32_t list = blockIdx.x; list < lists; list += gridDim.x) {
    int64_t v;
    uint32_t j0, j1;
    if (o.pick) {  // the list that holds position kLong * list and none of the multiples before
      v = o.token[kLong * list];
      j0 = o.start[v], j1 = o.start[v + 1];
      if (j1 - j0 <= kLong || (j0 + kLong - 1) / kLong != list) continue;
    } else {
      const uint32_t* entry = o.long_list + 3 * list;
      v = entry[0], j0 = entry[1], j1 = entry[2];
    }
    const uint32_t tile = o.tile, t0 = (j0 + tile - 1) / tile, t1 = max(j1 / tile, t0);
    const uint32_t head = min(t0 * tile, j1), tail = max(t1 * tile, head);
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    // a wavefront's share of the ends, each shorter than a tile: as many rows in flight as the registers
    // hold, their positions read before (one behind the other in 16 bits: 16 us for a Zipf batch of
    // 65,536, now 14)
    constexpr int kRows = sizeof(T) == 4 || kKind == kElements ? 2 : 4;
    for (uint32_t i = 0; i < 2 * tile; i += 16 * kRows) {
      RawSlices<T, 1, kKind> r[kRows];
      uint32_t pos[kRows];
      bool live[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const uint32_t e = i + 16 * u, at = (e < tile ? j0 : tail) + (e & (tile - 1)) + w;
        live[u] = e < 2 * tile && at < (e < tile ? head : j1);
        pos[u] = o.perm[live[u] ? at : j0];
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u)
        if (live[u]) r[u].template fetch<kStream>(gy + static_cast<int64_t>(pos[u]) * D, c0, D, lane);
#pragma unroll
      for (int u = 0; u < kRows; ++u)
        if (live[u]) {
          r[u].settle(c0, D, lane);
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] += r[u].at(k);
        }
    }
    for (uint32_t t = t0 + w; t < t1; t += 16 * 4) {
      Piece<float> lo[4], hi[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t tile = t + 16 * u < t1 ? t + 16 * u : t;
        const u32x4* at = reinterpret_cast<const u32x4*>(partial + tile * padded_cols(D) + c0) + lane;
        lo[u].raw = at[0];
        hi[u].raw = at[64];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (t + 16 * u < t1) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            acc[k] += lo[u].e[k];
            acc[4 + k] += hi[u].e[k];
          }
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sums[w][k][lane] = acc[k];
    __syncthreads();
    // 8 wavefronts add up a column of each lane's eight each, then the first one writes them
    if (w < 8) {
      float s = sums[0][w][lane];
#pragma unroll
      for (int i = 1; i < 16; ++i) s += sums[i][w][lane];
      sums[0][w][lane] = s * scale;
    }
    __syncthreads();
    if (w == 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[k] = sums[0][k][lane];
      store_slices<T, 1, kKind, kStream>(gw + v * D, c0, D, lane, acc);
    }
    __syncthreads();
  }
}

int64_t span_of(int64_t n) {
  // about 64 spans of 1024 to 16384 positions, longer ones where that would make more than 1024:
  // every span reads the counts of all of them
  const auto whole = [](int64_t x) { return (x + kSpanStep - 1) / kSpanStep * kSpanStep; };
  const int64_t s = whole(n / 64), most = 16 * kSpanStep;
  if (n > 1024 * most) return whole((n + 1023) / 1024);
  return s < kSpanStep ? kSpanStep : s > most ? most : s;
}

// Fills `o` and the address of the tiles' sums for a workspace at `ws`; returns its bytes.
int64_t lay_out(Order& o, float*& partial, void* ws, int64_t n, int64_t vocab, int64_t D) {
  o.n = n;
  o.vocab = vocab;
  o.row_bits = 0;
  while (((vocab - 1) >> o.row_bits) >= kBuckets) ++o.row_bits;
  o.buckets = static_cast<int>((vocab - 1) >> o.row_bits) + 1;
  o.span = span_of(n);
  o.spans = static_cast<int>((n + o.span - 1) / o.span);
  if (o.spans < 1) o.spans = 1;
  // Short tiles end sooner, long ones leave fewer sums to add: with 64, 5003 positions of 771 columns in
  // fp32 took 30 us in the sums and 9 in the join, with 16 23 and 5; 65,536 of 1536 in bf16 65 and 15, with
  // 32 71 and 16. The whole gradient with 16 and with 64: 54.8 and 58.1 us of 16,384 positions, 62.5 and
  // 62.3 of 24,576, 70.7 and 66.4 of 32,768 (771 in fp32); 57.3 and 58.1, 63.9 and 61.1, 73.9 and 65.2 (1536
  // in bf16).
  o.tile = n <= 16384 ? 16 : 64;
  o.pick = n <= kShort;
  char* base = static_cast<char*>(ws);
  int64_t used = 0;
  const auto take = [&](int64_t count) {
    const int64_t at = used;
    used += (count * 4 + 255) / 256 * 256;
    return base == nullptr ? nullptr : base + at;
  };
  const auto words = [&](int64_t count) { return reinterpret_cast<uint32_t*>(take(count)); };
  o.counts = words(static_cast<int64_t>(o.spans) * kBuckets);
  o.bucket_at = words(kBuckets + 1);
  o.item_pos = words(n);
  o.item_id = words(n);
  o.perm = words(n);
  o.token = words(n);
  o.start = words(vocab + 1);
  o.long_count = words(1);
  o.long_list = words(3 * (n / kLong + 1));
  partial = reinterpret_cast<float*>(take(n / o.tile * padded_cols(D)));
  return used;
}

bool sizes_ok(int64_t n, int64_t vocab, int64_t D) {
  return n >= 0 && n < (int64_t(1) << 31) - 16384 && vocab >= 1 &&
         vocab <= int64_t(kBuckets) << kMaxRowBits && D >= 1 && D <= (int64_t(1) << 20);
}

}  // namespace

int embed_launch(const void* table, int32_t dtype, int64_t vocab, int64_t D, const int64_t* ids,
                 int64_t n, float scale, void* out, hipStream_t st) {
  const int64_t slices = (D + kCols - 1) / kCols, grid = (n * slices + 3) / 4;
  LEMA_REQUIRE(grid < (int64_t(1) << 31), "too many ids");
  const RowKind kind = row_kind(dtype, D);
  // many rows go past the Infinity Cache, and leave it to the table's frequent ones: 65,536 of 1536 in
  // bf16 took 40 us, not 60, and of 1535 with no frequent ones 66, not 77
  const bool past = n * D * dtype_size(dtype) > (int64_t(128) << 20);
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const auto launch = [&](auto kernel) {
      kernel<<<blocks_of(grid), dim3(256), 0, st>>>(static_cast<const T*>(table), vocab, D, ids, n,
                                               static_cast<int>(slices), scale, static_cast<T*>(out));
    };
    for_kind<T>(kind, [&](auto k) {
      constexpr int kKind = decltype(k)::value;
      constexpr bool kCan = kKind != kElements;
      if (kCan && past)
        launch(scale != 1.0f ? embed_kernel<T, kKind, true, kCan> : embed_kernel<T, kKind, false, kCan>);
      else
        launch(scale != 1.0f ? embed_kernel<T, kKind, true, false> : embed_kernel<T, kKind, false, false>);
    });
  });
  return launch_status("embed_kernel");
}

}  // namespace lema

using namespace lema;

extern "C" int lema_embedding(const void* table, int32_t dtype, int64_t vocab, int64_t D,
                              const int64_t* ids, int64_t n, float scale, void* out, void* stream) {
  clear_error();
  const int size = dtype_size(dtype);
  LEMA_REQUIRE(size != 0, "unknown dtype %d", dtype);
  LEMA_REQUIRE(vocab >= 1 && D >= 1 && D <= (int64_t(1) << 20) && n >= 0 && n < (int64_t(1) << 31),
               "bad sizes: %lld ids, table [%lld, %lld]", (long long)n, (long long)vocab, (long long)D);
  if (n == 0) return LEMA_OK;
  LEMA_REQUIRE(table && ids && out && aligned(table, size) && aligned(ids, 8) && aligned(out, size),
               "bad pointer");
  return embed_launch(table, dtype, vocab, D, ids, n, scale, out, static_cast<hipStream_t>(stream));
}

extern "C" int64_t lema_embedding_grad_workspace_bytes(int64_t n, int64_t vocab, int64_t D) {
  if (!sizes_ok(n, vocab, D)) return 0;
  Order o;
  float* partial;
  return lay_out(o, partial, nullptr, n, vocab, D);
}

extern "C" int lema_embedding_grad(const void* gy, int32_t dtype, const int64_t* ids, int64_t n,
                                   int64_t vocab, int64_t D, float scale, int64_t padding, void* gw,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  const int size = dtype_size(dtype);
  LEMA_REQUIRE(size != 0, "unknown dtype %d", dtype);
  LEMA_REQUIRE(sizes_ok(n, vocab, D),
               "bad sizes: %lld ids, table [%lld, %lld] (at most 2^20 tokens and columns)", (long long)n,
               (long long)vocab, (long long)D);
  LEMA_REQUIRE(gw && aligned(gw, size) && (n == 0 || (gy && ids && aligned(gy, size) && aligned(ids, 8))),
               "bad pointer");
  LEMA_REQUIRE(workspace && aligned(workspace, 256) &&
                   workspace_bytes >= lema_embedding_grad_workspace_bytes(n, vocab, D),
               "the gradient needs a workspace of %lld bytes",
               (long long)lema_embedding_grad_workspace_bytes(n, vocab, D));
  Order o;
  float* partial;
  lay_out(o, partial, workspace, n, vocab, D);
  o.ids = ids;
  o.padding = padding;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t cols = (D + kCols - 1) / kCols, tiles = n / o.tile;
  // long lists at most, or the places where one may be
  const int64_t longest = o.pick && n > kLong ? (n + kLong - 1) / kLong : n / (kLong + 1);
  // a wavefront takes up to 3 slices: its chain of reads (start, positions, rows) is then shared
  const int64_t per = cols < 3 ? cols : 3, slices = (cols + per - 1) / per;
  const int64_t grid = ((tiles + vocab) * slices + 3) / 4;
  LEMA_REQUIRE(grid < (int64_t(1) << 24), "table [%lld, %lld] is too large", (long long)vocab,
               (long long)D);
  if (o.pick) {
    embed_order_kernel<true><<<dim3(o.buckets), dim3(512), 8 * 4 << o.row_bits, st>>>(o);
  } else {
    embed_count_kernel<<<dim3(o.spans), dim3(1024), 0, st>>>(o);
    embed_scatter_kernel<<<dim3(o.spans), dim3(1024), 0, st>>>(o);
    embed_order_kernel<false><<<dim3(o.buckets), dim3(512), 8 * 4 << o.row_bits, st>>>(o);
  }
  const RowKind kind = row_kind(dtype, D);
  // rows in, and the table's gradient out, past the Infinity Cache where they are larger than it: 65,536
  // rows of 1536 and a table of 50,304 in bf16 took 71 us, not 85 (of 1535: 71, not 82)
  const bool past = (n + vocab) * D * size > (int64_t(256) << 20);
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const auto run = [&](auto k, auto stream) {
      constexpr int kKind = decltype(k)::value;
      constexpr bool kStream = decltype(stream)::value;
      const auto sum = per == 1   ? embed_sum_kernel<T, 1, kKind, kStream>
                       : per == 2 ? embed_sum_kernel<T, 2, kKind, kStream>
                                  : embed_sum_kernel<T, 3, kKind, kStream>;
      sum<<<dim3(grid), dim3(256), 0, st>>>(o, static_cast<const T*>(gy), D, static_cast<int>(slices),
                                            tiles, scale, partial, static_cast<T*>(gw));
      const int64_t at_once = longest < 256 ? longest : 256;
      if (longest > 0)
        embed_join_kernel<T, kKind, kStream><<<dim3(at_once, cols), dim3(1024), 0, st>>>(
            o, static_cast<const T*>(gy), D, scale, partial, static_cast<T*>(gw));
    };
    for_kind<T>(kind, [&](auto k) {
      constexpr bool kCan = decltype(k)::value != kElements;
      if (kCan && past)
        run(k, std::integral_constant<bool, kCan>{});
      else
        run(k, std::false_type{});
    });
  });
  return launch_status("the embedding gradient's kernels");
}
