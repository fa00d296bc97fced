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

// Where lane `lane` of a row's W wavefronts finds its 8 elements of step s: next to each other in
// 16-byte pieces (kVec), or 64 * W apart, so that a wavefront's loads of single elements
// are contiguous too.
template <int W, bool kVec>
__device__ __forceinline__ int elem_at(int s, int k, int lane) {
  return kVec ? (s * W * 64 + lane) * 8 + k : (s * 8 + k) * W * 64 + lane;
}

template <typename T, int W, int S, bool kVec>
__device__ __forceinline__ void load_row(const T* p, int D, int lane, float (&v)[S * 8]) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (kVec) {
      const int e = elem_at<W, true>(s, 0, lane);
      constexpr int n = kPiece<T>;
      Piece<T> q[8 / n];
#pragma unroll
      for (int i = 0; i < 8 / n; ++i)
        q[i].raw = e < D ? *reinterpret_cast<const u32x4*>(p + e + i * n) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 8; ++k) v[s * 8 + k] = to_f32(q[k / n].e[k % n]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = elem_at<W, false>(s, k, lane);
        v[s * 8 + k] = e < D ? to_f32(p[e]) : 0.0f;
      }
    }
  }
}

template <typename T, int W, int S, bool kVec>
__device__ __forceinline__ void store_row(T* p, int D, int lane, const float (&v)[S * 8]) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (kVec) {
      const int e = elem_at<W, true>(s, 0, lane);
      constexpr int n = kPiece<T>;
      if (e < D) {
        Piece<T> q[8 / n];
#pragma unroll
        for (int k = 0; k < 8; ++k) q[k / n].e[k % n] = from_f32<T>(v[s * 8 + k]);
#pragma unroll
        for (int i = 0; i < 8 / n; ++i) *reinterpret_cast<u32x4*>(p + e + i * n) = q[i].raw;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = elem_at<W, false>(s, k, lane);
        if (e < D) p[e] = from_f32<T>(v[s * 8 + k]);
      }
    }
  }
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

template <typename T, int W, int S, bool kVec>
__global__ __launch_bounds__(64 * group_waves(W)) void layer_norm_kernel(
    const T* x, const T* d, const T* w, const T* b, float eps, int64_t rows, int D, T* s_out, T* h_out) {
  __shared__ float red[2 * W];
  constexpr int kSlots = group_waves(W) / W;
  const int lane = W > 1 ? threadIdx.x : threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kSlots + (W > 1 ? 0 : threadIdx.x >> 6);
  if (row >= rows) return;
  int turn = 0;
  float v[S * 8], t[S * 8];
  load_row<T, W, S, kVec>(x + row * D, D, lane, v);
  if (d != nullptr) {
    load_row<T, W, S, kVec>(d + row * D, D, lane, t);
#pragma unroll
    for (int k = 0; k < S * 8; ++k) v[k] = to_f32(from_f32<T>(v[k] + t[k]));
    store_row<T, W, S, kVec>(s_out + row * D, D, lane, v);
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
      if (elem_at<W, kVec>(s, k, lane) < D) sum[0] += v[s * 8 + k] * v[s * 8 + k];
    }
  row_sums<W, 1>(sum, red, turn);
  const float r = rsqrtf(sum[0] / static_cast<float>(D) + eps);
  if (w != nullptr) load_row<T, W, S, kVec>(w, D, lane, t);
#pragma unroll
  for (int k = 0; k < S * 8; ++k) v[k] *= w != nullptr ? r * t[k] : r;
  if (b != nullptr) {
    load_row<T, W, S, kVec>(b, D, lane, t);
#pragma unroll
    for (int k = 0; k < S * 8; ++k) v[k] += t[k];
  }
  store_row<T, W, S, kVec>(h_out + row * D, D, lane, v);
}

// Rows blockIdx.x * kSlots + slot, then on by gridDim.x * kSlots. partial: [2, gridDim.x, D] fp32,
// this workgroup's sums of gh z and of gh, where wanted.
template <typename T, int W, int S, bool kVec, bool kCenter>
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
  if (w != nullptr) load_row<T, W, S, kVec>(w, D, lane, wv);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kSlots + slot; row < rows;
       row += static_cast<int64_t>(gridDim.x) * kSlots) {
    float v[S * 8], g[S * 8];
    load_row<T, W, S, kVec>(s_in + row * D, D, lane, v);
    load_row<T, W, S, kVec>(gh + row * D, D, lane, g);
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
          v[s * 8 + k] = elem_at<W, kVec>(s, k, lane) < D ? v[s * 8 + k] - m : 0.0f;
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
      if (gs != nullptr) {
        load_row<T, W, S, kVec>(gs + row * D, D, lane, g);
#pragma unroll
        for (int k = 0; k < S * 8; ++k) v[k] += g[k];
      }
      store_row<T, W, S, kVec>(gx + row * D, D, lane, v);
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
          const int e = elem_at<W, kVec>(s, k, lane);
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
          const int e = elem_at<W, kVec>(s, k, lane);
          if (e < D) out[e] = which ? gb[s * 8 + k] : gw[s * 8 + k];
        }
    }
  }
}

// out[e] = sum over `parts` of partial[p, e]; blockIdx.y picks the weight's or the bias's. 16
// groups of 16 columns' threads each take every 16th part.
template <typename T>
__global__ __launch_bounds__(256) void norm_weight_kernel(const float* partial, int parts, int D,
                                                          T* gw, T* gb) {
  __shared__ float sums[16][17];
  T* out = blockIdx.y ? gb : gw;
  if (out == nullptr) return;
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int e = blockIdx.x * 16 + c;
  const float* p = partial + static_cast<int64_t>(blockIdx.y) * parts * D + e;
  float t = 0.0f;
  if (e < D)
    for (int i = q; i < parts; i += 16) t += p[static_cast<int64_t>(i) * D];
  sums[q][c] = t;
  __syncthreads();
  if (q == 0 && e < D) {
    for (int i = 1; i < 16; ++i) t += sums[i][c];
    out[e] = from_f32<T>(t);
  }
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

// Workgroups of the gradient: enough to fill the GPU a few times over, no more than there are rows.
int64_t grad_groups(int64_t rows, int64_t D) {
  const int64_t slots = D <= 2048 ? 4 : 1;
  const int64_t want = (rows + slots - 1) / slots;
  return want < 1024 ? want : 1024;
}

bool pieces_ok(int64_t D, std::initializer_list<const void*> ptrs) {
  bool ok = D % 8 == 0;
  for (const void* p : ptrs) ok = ok && aligned(p, 16);  // NULL counts as aligned
  return ok;
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
  const bool vec = pieces_ok(D, {x, d, w, b, s_out, h_out});
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    for_width(D, [&](auto wc, auto sc) {
      constexpr int W = decltype(wc)::value, S = decltype(sc)::value;
      const int64_t slots = group_waves(W) / W, grid = (rows + slots - 1) / slots;
      const auto kernel = vec ? layer_norm_kernel<T, W, S, true> : layer_norm_kernel<T, W, S, false>;
      kernel<<<dim3(grid), dim3(64 * group_waves(W)), 0, static_cast<hipStream_t>(stream)>>>(
          static_cast<const T*>(x), static_cast<const T*>(d), static_cast<const T*>(w),
          static_cast<const T*>(b), eps, rows, static_cast<int>(D), static_cast<T*>(s_out),
          static_cast<T*>(h_out));
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
  const bool vec = pieces_ok(D, {s, w, gh, gs, gx});
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (rows > 0)
      for_width(D, [&](auto wc, auto sc) {
        constexpr int W = decltype(wc)::value, S = decltype(sc)::value;
        const auto kernel = center ? (vec ? norm_grad_kernel<T, W, S, true, true>
                                          : norm_grad_kernel<T, W, S, false, true>)
                                   : (vec ? norm_grad_kernel<T, W, S, true, false>
                                          : norm_grad_kernel<T, W, S, false, false>);
        kernel<<<dim3(groups), dim3(64 * group_waves(W)), 0, st>>>(
            static_cast<const T*>(s), static_cast<const T*>(w), static_cast<const T*>(gh),
            static_cast<const T*>(gs), eps, rows, static_cast<int>(D), static_cast<T*>(gx), partial);
      });
    if (sums)
      norm_weight_kernel<T><<<dim3((D + 15) / 16, gb != nullptr ? 2 : 1), dim3(256), 0, st>>>(
          partial, static_cast<int>(groups), static_cast<int>(D), static_cast<T*>(gw),
          static_cast<T*>(gb));
  });
  return launch_status("norm_grad_kernel");
}
