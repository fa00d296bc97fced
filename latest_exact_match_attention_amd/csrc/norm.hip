// Layer norm, and the gradients of layer norm and RMS norm.
//
// Forward, per row of D: s = round(x + d), m = mean(s), r = rsqrt(mean((s - m)^2) + eps),
// h = (s - m) r w + b. The mean of squares is that of the centred elements, which the row in
// registers allows: no cancellation for rows far from zero.
//
// Backward, with z = (s - m) r and a = gh w (m = 0 for RMS norm):
//   gx = gs + r (a - mean(a) - z mean(a z))      (RMS norm has no mean(a))
//   gw = sum over rows of gh z,  gb = sum over rows of gh
// m and r are computed again from s, which is read anyway: saving them would add a tensor and
// spare one reduction in registers.
//
// Both are bound by HBM. A row is read once and stays in registers, 8 elements a lane and step,
// S steps: up to 2048 elements in one wavefront, longer rows over 4 or 16 wavefronts that meet in
// LDS. The weights' gradients are summed in fp32 in registers over the rows that a wavefront
// takes in turn, then over a workgroup's wavefronts, then over the workgroups by a second
// kernel, each in a fixed order.
#include "elem.h"

namespace lema {
namespace {

constexpr int64_t kMaxD = 16384;

// Where lane `lane` of a row's W wavefronts finds its element k of step s: a load's units next to
// each other.
template <typename T, int W, int kKind>
__device__ __forceinline__ int elem_at(int s, int k, int lane) {
  constexpr int n = kUnit<T, kKind>;
  return ((s * 8 + k) / n * W * 64 + lane) * n + k % n;
}

// A row's elements as they come from memory, so that a row can be on its way while the one before
// it is worked on.
template <typename T, int W, int S, int kKind>
struct RawRow : RowPart<T, kKind, S * 8> {
  template <bool kStream = false>
  __device__ __forceinline__ void fetch(const T* p, int D, int lane) {
    RowPart<T, kKind, S * 8>::template fetch<kStream>(p, D, [&](int i) { return elem_at<T, W, kKind>(0, i, lane); });
  }
  __device__ __forceinline__ void settle(int D, int lane) {
    RowPart<T, kKind, S * 8>::settle(D, [&](int i) { return elem_at<T, W, kKind>(0, i, lane); });
  }
  __device__ __forceinline__ float at(int k) const { return this->get(k); }
};

template <typename T, int W, int S, int kKind>
__device__ __forceinline__ void load_row(const T* p, int D, int lane, float (&v)[S * 8]) {
  RawRow<T, W, S, kKind> r;
  r.fetch(p, D, lane);
  r.settle(D, lane);
#pragma unroll
  for (int k = 0; k < S * 8; ++k) v[k] = r.at(k);
}

template <typename T, int W, int S, int kKind, bool kStream = false>
__device__ __forceinline__ void store_row(T* p, int D, int lane, const float (&v)[S * 8]) {
  RowPart<T, kKind, S * 8> r;
#pragma unroll
  for (int k = 0; k < S * 8; ++k) r.set(k, v[k]);
  r.template store<kStream>(p, D, [&](int i) { return elem_at<T, W, kKind>(0, i, lane); });
}

// Sums of N values over a row's W wavefronts, in every lane. `red` holds 2 * N * W floats, used
// in turn (`turn` flips), so that one barrier a sum is enough: a wavefront that is ahead writes
// the other half, and cannot be two sums ahead of one that still reads.
template <int W, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float* red, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (W > 1) {
    float* half = red + turn * N * W;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) half[i * W + (threadIdx.x >> 6)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = half[i * W];
#pragma unroll
      for (int w = 1; w < W; ++w) t += half[i * W + w];
      v[i] = t;
    }
  }
}

// Wavefronts of a workgroup: a row each where a row takes one, else all on one row.
constexpr int group_waves(int W) { return W > 1 ? W : 4; }

template <typename T, int W, int S, int kKind>
__global__ __launch_bounds__(64 * group_waves(W)) void layer_norm_kernel(
    const T* x, const T* d, const T* w, const T* b, float eps, int64_t rows, int D, T* s_out, T* h_out) {
  __shared__ float red[2 * W];
  constexpr int kSlots = group_waves(W) / W;
  const int lane = W > 1 ? threadIdx.x : threadIdx.x & 63;
  const int64_t row = block_index() * kSlots + (W > 1 ? 0 : threadIdx.x >> 6);
  if (row >= rows) return;
  int turn = 0;
  float v[S * 8], t[S * 8];
  load_row<T, W, S, kKind>(x + row * D, D, lane, v);
  if (d != nullptr) {
    load_row<T, W, S, kKind>(d + row * D, D, lane, t);
#pragma unroll
    for (int k = 0; k < S * 8; ++k) v[k] = to_f32(from_f32<T>(v[k] + t[k]));
    store_row<T, W, S, kKind>(s_out + row * D, D, lane, v);
  }
  float sum[1] = {0.0f};
#pragma unroll
  for (int k = 0; k < S * 8; ++k) sum[0] += v[k];
  row_sums<W, 1>(sum, red, turn);
  const float m = sum[0] / static_cast<float>(D);
  sum[0] = 0.0f;
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[s * 8 + k] -= m;
      if (elem_at<T, W, kKind>(s, k, lane) < D) sum[0] += v[s * 8 + k] * v[s * 8 + k];
    }
  row_sums<W, 1>(sum, red, turn);
  const float r = rsqrtf(sum[0] / static_cast<float>(D) + eps);
  if (w != nullptr) load_row<T, W, S, kKind>(w, D, lane, t);
#pragma unroll
  for (int k = 0; k < S * 8; ++k) v[k] *= w != nullptr ? r * t[k] : r;
  if (b != nullptr) {
    load_row<T, W, S, kKind>(b, D, lane, t);
#pragma unroll
    for (int k = 0; k < S * 8; ++k) v[k] += t[k];
  }
  store_row<T, W, S, kKind>(h_out + row * D, D, lane, v);
}

// Rows blockIdx.x * kSlots + slot, then on by gridDim.x * kSlots. partial: [2, gridDim.x, D] fp32,
// this workgroup's sums of gh z and of gh, where wanted.
template <typename T, int W, int S, int kKind, bool kCenter, bool kStream>
__global__ __launch_bounds__(64 * group_waves(W)) void norm_grad_kernel(
    const T* s_in, const T* w, const T* gh, const T* gs, float eps, int64_t rows, int D, T* gx,
    float* partial) {
  constexpr int kSlots = group_waves(W) / W;
  __shared__ float red[2 * 3 * W];
  __shared__ float comb[W > 1 ? 1 : kSlots * 512 * S];
  const int lane = W > 1 ? threadIdx.x : threadIdx.x & 63;
  const int slot = W > 1 ? 0 : threadIdx.x >> 6;
  const float inv_d = 1.0f / static_cast<float>(D);
  int turn = 0;
  float wv[S * 8], gw[S * 8], gb[S * 8];
#pragma unroll
  for (int k = 0; k < S * 8; ++k) gw[k] = gb[k] = 0.0f, wv[k] = 1.0f;
  if (w != nullptr) load_row<T, W, S, kKind>(w, D, lane, wv);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kSlots;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kSlots + slot;
  RawRow<T, W, S, kKind> next_v, next_g, next_gs;
  const bool add = gx != nullptr && gs != nullptr;
  const auto fetch = [&](int64_t r) {
    next_v.template fetch<kStream>(s_in + r * D, D, lane);
    next_g.template fetch<kStream>(gh + r * D, D, lane);
    if (add) next_gs.template fetch<kStream>(gs + r * D, D, lane);
  };
  constexpr bool kAhead = S == 1;  // with more, the registers of the row on its way spill
  if (kAhead && row < rows) fetch(row);
  for (; row < rows; row += step) {
    if (!kAhead) fetch(row);
    float v[S * 8], g[S * 8];
    RawRow<T, W, S, kKind> gs_row = next_gs;
    next_v.settle(D, lane);
    next_g.settle(D, lane);
#pragma unroll
    for (int k = 0; k < S * 8; ++k) {
      v[k] = next_v.at(k);
      g[k] = next_g.at(k);
    }
    if (kAhead && row + step < rows) fetch(row + step);
    if constexpr (kCenter) {
      float sum[1] = {0.0f};
#pragma unroll
      for (int k = 0; k < S * 8; ++k) sum[0] += v[k];
      row_sums<W, 1>(sum, red, turn);
      const float m = sum[0] * inv_d;
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          v[s * 8 + k] = elem_at<T, W, kKind>(s, k, lane) < D ? v[s * 8 + k] - m : 0.0f;
    }
    float sum[3] = {0.0f, 0.0f, 0.0f};  // of squares, of a v, of a
#pragma unroll
    for (int k = 0; k < S * 8; ++k) {
      const float a = g[k] * wv[k];
      sum[0] += v[k] * v[k];
      sum[1] += a * v[k];
      sum[2] += a;
    }
    row_sums<W, 3>(sum, red, turn);
    const float r = rsqrtf(sum[0] * inv_d + eps);
    const float c1 = kCenter ? sum[2] * inv_d : 0.0f, c2 = sum[1] * inv_d * r;
#pragma unroll
    for (int k = 0; k < S * 8; ++k) {
      const float z = v[k] * r;
      gw[k] += g[k] * z;
      if constexpr (kCenter) gb[k] += g[k];
      v[k] = r * (g[k] * wv[k] - c1 - z * c2);
    }
    if (gx != nullptr) {
      if (add) {
        gs_row.settle(D, lane);
#pragma unroll
        for (int k = 0; k < S * 8; ++k) v[k] += gs_row.at(k);
      }
      store_row<T, W, S, kKind, kStream>(gx + row * D, D, lane, v);
    }
  }
  if (partial == nullptr) return;
  for (int which = 0; which < (kCenter ? 2 : 1); ++which) {
    float* out = partial + (static_cast<int64_t>(which) * gridDim.x + blockIdx.x) * D;
    if constexpr (W == 1) {
      if (which) __syncthreads();
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int e = elem_at<T, W, kKind>(s, k, lane);
          comb[slot * 512 * S + e] = which ? gb[s * 8 + k] : gw[s * 8 + k];
        }
      __syncthreads();
      for (int e = threadIdx.x; e < D; e += 64 * kSlots) {
        float t = comb[e];
#pragma unroll
        for (int j = 1; j < kSlots; ++j) t += comb[j * 512 * S + e];
        out[e] = t;
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int e = elem_at<T, W, kKind>(s, k, lane);
          if (e < D) out[e] = which ? gb[s * 8 + k] : gw[s * 8 + k];
        }
    }
  }
}

// out[e] = sum over `parts` of partial[p, e]; blockIdx.y picks the weight's or the bias's. 64
// groups of 16 columns' threads each take every 64th part, 8 parts in flight: the partial sums
// are a few MB in L2 and the Infinity Cache, and a thread that waits for each of them in turn took
// 25 us for 1024 parts of 1536.
template <typename T>
__global__ __launch_bounds__(1024) void norm_weight_kernel(const float* partial, int parts, int D,
                                                           T* gw, T* gb) {
  __shared__ float sums[64][17];
  T* out = blockIdx.y ? gb : gw;
  if (out == nullptr) return;
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int e = blockIdx.x * 16 + c;
  const float* p = partial + static_cast<int64_t>(blockIdx.y) * parts * D + (e < D ? e : 0);
  float t = 0.0f;
  for (int i = q; i < parts; i += 64 * 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int at = i + u * 64;
      v[u] = p[static_cast<int64_t>(at < parts ? at : q) * D];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) t += i + u * 64 < parts ? v[u] : 0.0f;
  }
  sums[q][c] = t;
  __syncthreads();
  for (int half = 32; half > 0; half >>= 1) {
    if (q < half) sums[q][c] += sums[q + half][c];
    __syncthreads();
  }
  if (q == 0 && e < D) out[e] = from_f32<T>(sums[0][c]);
}

// Calls f with the wavefronts a row takes and its steps, as compile-time constants.
template <typename F>
inline void for_width(int64_t D, F f) {
  using std::integral_constant;
  if (D <= 512)
    f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (D <= 1024)
    f(integral_constant<int, 1>{}, integral_constant<int, 2>{});
  else if (D <= 1536)
    f(integral_constant<int, 1>{}, integral_constant<int, 3>{});
  else if (D <= 2048)
    f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (D <= 4096)
    f(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  else if (D <= 8192)
    f(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else
    f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
}

// The gradient's widths: 8 elements a lane where that is possible, because each element costs a lane
// five registers (row, gradient, weight, two sums), and the row on its way as much again.
template <typename F>
inline void for_grad_width(int64_t D, F f) {
  using std::integral_constant;
  if (D <= 512)
    f(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (D <= 1024)
    f(integral_constant<int, 2>{}, integral_constant<int, 1>{});
  else if (D <= 1536)
    f(integral_constant<int, 3>{}, integral_constant<int, 1>{});
  else if (D <= 2048)
    f(integral_constant<int, 4>{}, integral_constant<int, 1>{});
  else if (D <= 4096)
    f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  else if (D <= 8192)
    f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else
    f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
}

// Workgroups of the gradient: what the GPU holds at once (16 wavefronts a CU), no more than there are
// rows, and no more than 1024, because each leaves two rows of sums for the second kernel.
int64_t grad_groups(int64_t rows, int64_t D) {
  const int64_t slots = D <= 512 ? 4 : 1;
  const int64_t want = (rows + slots - 1) / slots, fit = D <= 2048 ? 1024 : D <= 4096 ? 512 : 256;
  return want < fit ? want : fit;
}

int check_rows(int32_t dtype, int64_t rows, int64_t D) {
  LEMA_REQUIRE(dtype_size(dtype) != 0, "unknown dtype %d", dtype);
  LEMA_REQUIRE(D > 0 && D <= kMaxD, "row length %lld must lie in [1, %lld]", (long long)D,
               (long long)kMaxD);
  LEMA_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31), "bad row count %lld", (long long)rows);
  return LEMA_OK;
}

}  // namespace
}  // namespace lema

using namespace lema;

extern "C" int lema_layer_norm(const void* x, const void* d, const void* w, const void* b,
                               int32_t dtype, float eps, int64_t rows, int64_t D, void* s_out,
                               void* h_out, void* stream) {
  clear_error();
  if (int rc = check_rows(dtype, rows, D)) return rc;
  if (rows == 0) return LEMA_OK;
  LEMA_REQUIRE(x && h_out && (d == nullptr || s_out != nullptr), "null pointer");
  const int size = dtype_size(dtype);
  for (const void* p : {x, d, w, b, static_cast<const void*>(s_out), static_cast<const void*>(h_out)})
    LEMA_REQUIRE(aligned(p, size), "pointers must be aligned to an element");
  const RowKind kind = row_kind(dtype, D);
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    for_width(D, [&](auto wc, auto sc) {
      constexpr int W = decltype(wc)::value, S = decltype(sc)::value;
      const int64_t slots = group_waves(W) / W, grid = (rows + slots - 1) / slots;
      for_kind<T>(kind, [&](auto k) {
        layer_norm_kernel<T, W, S, decltype(k)::value>
            <<<blocks_of(grid), dim3(64 * group_waves(W)), 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const T*>(x), static_cast<const T*>(d), static_cast<const T*>(w),
                static_cast<const T*>(b), eps, rows, static_cast<int>(D), static_cast<T*>(s_out),
                static_cast<T*>(h_out));
      });
    });
  });
  return launch_status("layer_norm_kernel");
}

extern "C" int64_t lema_norm_grad_workspace_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D <= 0 || D > kMaxD) return 0;
  return 2 * grad_groups(rows, D) * D * static_cast<int64_t>(sizeof(float));
}

extern "C" int lema_norm_grad(const void* s, const void* w, const void* gh, const void* gs,
                              int32_t dtype, int32_t center, float eps, int64_t rows, int64_t D,
                              void* gx, void* gw, void* gb, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int rc = check_rows(dtype, rows, D)) return rc;
  const bool sums = gw != nullptr || gb != nullptr;
  if (rows == 0 && !sums) return LEMA_OK;
  LEMA_REQUIRE(rows == 0 || (s && gh), "null pointer");
  LEMA_REQUIRE(center != 0 || gb == nullptr, "RMS norm has no bias");
  const int size = dtype_size(dtype);
  for (const void* p : {s, w, gh, gs, static_cast<const void*>(gx), static_cast<const void*>(gw),
                        static_cast<const void*>(gb)})
    LEMA_REQUIRE(aligned(p, size), "pointers must be aligned to an element");
  LEMA_REQUIRE(!sums || rows == 0 ||
                   (workspace && aligned(workspace, 256) &&
                    workspace_bytes >= lema_norm_grad_workspace_bytes(rows, D)),
               "the weights' gradients need a workspace of %lld bytes",
               (long long)lema_norm_grad_workspace_bytes(rows, D));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t groups = rows > 0 ? grad_groups(rows, D) : 0;
  float* partial = sums ? static_cast<float*>(workspace) : nullptr;
  const RowKind kind = row_kind(dtype, D);
  // Up to four tensors of rows pass through. Where they are far larger than the Infinity Cache they go
  // past it: the gradient of 65,536 rows of 1536 in bf16 took 137 us, not 159 (of 1535: 200, not 218),
  // and the norm that ran next 133, not 130. 8192 rows of 4096 in fp16 fit it and lost by it, 59 us
  // against 56 (and 49 against 44).
  const bool past = rows * D * size > (int64_t(128) << 20);
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (rows > 0)
      for_grad_width(D, [&](auto wc, auto sc) {
        constexpr int W = decltype(wc)::value, S = decltype(sc)::value;
        const auto launch = [&](auto kernel) {
          kernel<<<dim3(groups), dim3(64 * group_waves(W)), 0, st>>>(
              static_cast<const T*>(s), static_cast<const T*>(w), static_cast<const T*>(gh),
              static_cast<const T*>(gs), eps, rows, static_cast<int>(D), static_cast<T*>(gx), partial);
        };
        for_kind<T>(kind, [&](auto k) {
          constexpr int kKind = decltype(k)::value;
          constexpr bool kCan = kKind != kElements;
          if (kCan && past)
            launch(center ? norm_grad_kernel<T, W, S, kKind, true, kCan>
                          : norm_grad_kernel<T, W, S, kKind, false, kCan>);
          else
            launch(center ? norm_grad_kernel<T, W, S, kKind, true, false>
                          : norm_grad_kernel<T, W, S, kKind, false, false>);
        });
      });
    if (sums)
      norm_weight_kernel<T><<<dim3((D + 15) / 16, gb != nullptr ? 2 : 1), dim3(1024), 0, st>>>(
          partial, static_cast<int>(groups), static_cast<int>(D), static_cast<T*>(gw),
          static_cast<T*>(gb));
  });
  return launch_status("norm_grad_kernel");
}
