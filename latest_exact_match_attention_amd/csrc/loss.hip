// Losses on the log-probabilities of given tokens, from logits, and their gradients.
//
// Per row of V logits x, with k = 1 / temperature:  M = max x,  S = sum of e^(k (x - M)),
//   lp = k (x_t - M) - log S                          t the row's target
//   d lp / d x_j = k ([j = t] - e^(k (x_j - M)) / S)
// so a loss needs lp and c = d loss / d lp of each row, and the logits' gradient is c k times the
// bracket. The forward kernel reads a row once, with a running maximum and a sum that is rescaled to
// it, and keeps (M, 1 / S); the gradient's kernel reads it once more and writes it. Both are bound
// by HBM. lp is formed in 64 bits by one thread, from fp32 differences and the fp32 sum: a
// preference adds up those of a whole answer.
//
//   policy      r = e^(lp - old), term = -min(r A, clip(r, 1 - lo, 1 + hi) A)
//                                        + kl (e^(ref - lp) - (ref - lp) - 1),
//               loss = mean of the counted rows' terms
//   preference  s = sum of an answer's counted (lp - ref), m = beta (s_chosen - s_rejected),
//               term = -(1 - e) log sigmoid(m) - e log sigmoid(-m), loss = mean over the pairs
//
// Rows that the mask leaves out are not read: their lp and gradient are zero whatever they hold.
#include <cfloat>
#include <cmath>

#include "elem.h"

namespace lema {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Row r of a tensor [outer, inner, V] with element strides (so, si, 1).
struct Rows {
  int64_t inner, so, si;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    const int64_t o = r / inner;
    return o * so + (r - o * inner) * si;
  }
};

// What a row's thread 0 needs for the policy loss; `old` NULL: log-probabilities only.
struct Policy {
  const float *old, *adv, *ref;
  float *term, *coef;
  float clip_low, clip_high, kl;
};

struct Running {
  float m, s;  // the maximum so far, -FLT_MAX at least, and the sum rescaled to it
};

// Adds n logits to r. -FLT_MAX for the maximum of nothing, or of -inf alone, keeps
// (-inf) - m = -inf, a zero, while a NaN stays one.
template <int N>
__device__ __forceinline__ void add_logits(Running& r, const float (&x)[N], float k2) {
  float bm = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) bm = fmaxf(bm, x[i]);
  if (bm > r.m) {
    r.s *= __builtin_amdgcn_exp2f((r.m - bm) * k2);
    r.m = bm;
  }
  float sa = 0.0f, sb = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    sa += __builtin_amdgcn_exp2f((x[i] - r.m) * k2);
    if (i + 1 < N) sb += __builtin_amdgcn_exp2f((x[i + 1] - r.m) * k2);
  }
  r.s += sa + sb;
}

__device__ __forceinline__ Running join(Running a, Running b, float k2) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * __builtin_amdgcn_exp2f((a.m - m) * k2) + b.s * __builtin_amdgcn_exp2f((b.m - m) * k2)};
}

// The elements of a row before its first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* row, int64_t V) {
  const int64_t h = ((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T);
  return h < V ? h : V;
}

// One workgroup per row.
template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void logprob_kernel(const T* logits, Rows rows, int64_t V,
                                                           const int64_t* target, const uint8_t* mask,
                                                           float k, float* lp_out, double* lp64_out,
                                                           float2* stats, Policy pol) {
  constexpr int kWaves = kThreads / 64, n = kPiece<T>;
  __shared__ Running part[kWaves];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  if (mask != nullptr && mask[row] == 0) {
    if (tid == 0) {
      lp_out[row] = 0.0f;
      if (lp64_out != nullptr) lp64_out[row] = 0.0;
      if (pol.old != nullptr) pol.term[row] = pol.coef[row] = 0.0f;
    }
    return;
  }
  const float k2 = k * kLog2e;
  const T* x = logits + rows.at(row);
  const int64_t head = head_of(x, V), pieces = (V - head) / n, tail = head + pieces * n;
  const u32x4* body = reinterpret_cast<const u32x4*>(x + head);
  Running r{-FLT_MAX, 0.0f};
  if (tid < head) {  // head < n <= 8 elements
    const float one[1] = {to_f32(x[tid])};
    add_logits<1>(r, one, k2);
  }
  if (tid < V - tail) {
    const float one[1] = {to_f32(x[tail + tid])};
    add_logits<1>(r, one, k2);
  }
  // two pieces in flight; the second of an odd last trip is missing
  for (int64_t p = tid; p < pieces; p += 2 * kThreads) {
    Piece<T> a, b;
    const bool two = p + kThreads < pieces;
    a.raw = body[p];
    b.raw = body[two ? p + kThreads : p];
    float v[n];
    if (two) {
      float w[2 * n];
#pragma unroll
      for (int i = 0; i < n; ++i) {
        w[i] = to_f32(a.e[i]);
        w[n + i] = to_f32(b.e[i]);
      }
      add_logits<2 * n>(r, w, k2);
    } else {
#pragma unroll
      for (int i = 0; i < n; ++i) v[i] = to_f32(a.e[i]);
      add_logits<n>(r, v, k2);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) r = join(r, Running{__shfl_xor(r.m, o), __shfl_xor(r.s, o)}, k2);
  if ((tid & 63) == 0) part[tid >> 6] = r;
  __syncthreads();
  if (tid != 0) return;
  r = part[0];
  for (int w = 1; w < kWaves; ++w) r = join(r, part[w], k2);
  const int64_t t = target[row];
  const float xt = t >= 0 && t < V ? to_f32(x[t]) : NAN;
  const double lp = static_cast<double>(xt - r.m) * k - log(static_cast<double>(r.s));
  lp_out[row] = static_cast<float>(lp);
  if (lp64_out != nullptr) lp64_out[row] = lp;
  if (stats != nullptr) stats[row] = make_float2(r.m, 1.0f / r.s);
  if (pol.old != nullptr) {
    const double a = pol.adv[row], ratio = exp(lp - pol.old[row]);
    const double lo = 1.0 - pol.clip_low, hi = 1.0 + pol.clip_high;
    // the smaller product is the clipped one where the ratio has left the interval on the side
    // that the advantage pushes to; there it does not depend on lp
    const bool live = a >= 0.0 ? !(ratio > hi) : !(ratio < lo);
    double term = -a * (live ? ratio : a >= 0.0 ? hi : lo), coef = live ? -a * ratio : 0.0;
    if (pol.ref != nullptr) {
      const double gap = pol.ref[row] - lp;
      term += pol.kl * (expm1(gap) - gap);
      coef -= pol.kl * expm1(gap);
    }
    pol.term[row] = static_cast<float>(term);
    pol.coef[row] = static_cast<float>(coef);
  }
}

// Sum over the wavefront in 64 bits.
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// loss = sum of the terms / counted rows (0 where there are none), in 64 bits; inv_n = 1 / rows.
__global__ __launch_bounds__(1024) void policy_mean_kernel(const float* term, const uint8_t* mask,
                                                           int64_t rows, float* loss, float* inv_n) {
  __shared__ double sums[2][16];
  double t = 0.0, n = 0.0;
  for (int64_t i = threadIdx.x; i < rows; i += 1024) {
    t += term[i];
    n += mask == nullptr || mask[i] != 0 ? 1.0 : 0.0;
  }
  t = wave_sum64(t);
  n = wave_sum64(n);
  if ((threadIdx.x & 63) == 0) {
    sums[0][threadIdx.x >> 6] = t;
    sums[1][threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) {
    t += sums[0][w];
    n += sums[1][w];
  }
  n = n > 0.0 ? 1.0 / n : 1.0;
  *loss = static_cast<float>(t * n);
  *inv_n = static_cast<float>(n);
}

// One workgroup, a wavefront a pair at a time: answers p and pairs + p of T rows each.
__global__ __launch_bounds__(1024) void preference_kernel(const double* lp, const float* ref,
                                                          const uint8_t* mask, int64_t pairs, int64_t T,
                                                          float beta, float smooth, float* loss,
                                                          float* margin, float* coef) {
  __shared__ double sums[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  double total = 0.0;
  for (int64_t p = w; p < pairs; p += 16) {
    double s[2] = {0.0, 0.0};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int64_t at = (side * pairs + p) * T;
      for (int64_t i = at + lane; i < at + T; i += 64)
        if (mask == nullptr || mask[i] != 0) s[side] += lp[i] - ref[i];
    }
    const double m = beta * wave_sum64(s[0] - s[1]);
    const double tail = log1p(exp(-fabs(m)));        // -log sigmoid(|m|)
    const double up = tail + (m < 0.0 ? -m : 0.0), down = tail + (m > 0.0 ? m : 0.0);
    total += (1.0 - smooth) * up + smooth * down;
    if (lane == 0) {
      // d term / d m = -(1 - smooth) sigmoid(-m) + smooth sigmoid(m)
      const double dm = -(1.0 - smooth) / (1.0 + exp(m)) + smooth / (1.0 + exp(-m));
      const float c = static_cast<float>(dm * beta / static_cast<double>(pairs));
      margin[p] = static_cast<float>(m);
      coef[p] = c;
      coef[pairs + p] = -c;
    }
  }
  if (lane == 0) sums[w] = total;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) total += sums[i];
  *loss = static_cast<float>(total / static_cast<double>(pairs));
}

// grad[row] = c k ([j = t] - e^(k (x_j - M)) / S), c = coef[row / per] * *scale0 * *scale1 (each
// NULL: 1). grad is contiguous [rows, V]. Rows of c = 0 are not read.
template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void logprob_grad_kernel(
    const T* logits, Rows rows, int64_t V, const int64_t* target, const uint8_t* mask, float k,
    const float2* stats, const float* coef, int64_t per, const float* scale0, const float* scale1, T* grad) {
  constexpr int n = kPiece<T>;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  T* g = grad + row * V;
  float c = 0.0f;
  if (mask == nullptr || mask[row] != 0) {
    c = coef[row / per] * k;
    if (scale0 != nullptr) c *= *scale0;
    if (scale1 != nullptr) c *= *scale1;
  }
  const int64_t head = head_of(g, V), pieces = (V - head) / n, tail = head + pieces * n;
  u32x4* out = reinterpret_cast<u32x4*>(g + head);
  if (c == 0.0f) {
    const T zero = from_f32<T>(0.0f);
    if (tid < head) g[tid] = zero;
    if (tid < V - tail) g[tail + tid] = zero;
    for (int64_t p = tid; p < pieces; p += kThreads) out[p] = u32x4{0, 0, 0, 0};
    return;
  }
  const float2 st = stats[row];
  const float k2 = k * kLog2e, cs = c * st.y;
  const int64_t t = target[row];
  const T* x = logits + rows.at(row);
  const auto one = [&](int64_t j, float v) {
    const float e = __builtin_amdgcn_exp2f((v - st.x) * k2);
    return from_f32<T>(j == t ? fmaf(-cs, e, c) : -cs * e);
  };
  if ((reinterpret_cast<uintptr_t>(x + head) & 15) != 0) {  // the rows' alignments differ
    for (int64_t j = tid; j < V; j += kThreads) g[j] = one(j, to_f32(x[j]));
    return;
  }
  if (tid < head) g[tid] = one(tid, to_f32(x[tid]));
  if (tid < V - tail) g[tail + tid] = one(tail + tid, to_f32(x[tail + tid]));
  const u32x4* body = reinterpret_cast<const u32x4*>(x + head);
  for (int64_t p = tid; p < pieces; p += 2 * kThreads) {
    Piece<T> a, b;
    const bool two = p + kThreads < pieces;
    a.raw = body[p];
    b.raw = body[two ? p + kThreads : p];
#pragma unroll
    for (int i = 0; i < n; ++i) {
      a.e[i] = one(head + p * n + i, to_f32(a.e[i]));
      b.e[i] = one(head + (p + kThreads) * n + i, to_f32(b.e[i]));
    }
    out[p] = a.raw;
    if (two) out[p + kThreads] = b.raw;
  }
}

int check_logits(const void* logits, int32_t dtype, int64_t rows, int64_t inner, int64_t V, int64_t so,
                 int64_t si, const int64_t* target, float temperature) {
  const int size = dtype_size(dtype);
  LEMA_REQUIRE(size != 0, "unknown dtype %d", dtype);
  LEMA_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31),
               "bad sizes: %lld rows of %lld logits", (long long)rows, (long long)V);
  LEMA_REQUIRE(inner >= 1 && so >= 0 && si >= 0, "bad strides");
  LEMA_REQUIRE(temperature > 0.0f && std::isfinite(temperature) &&
                   std::isfinite(kLog2e / temperature) && 1.0f / temperature > 0.0f,
               "the temperature must be a positive number");
  LEMA_REQUIRE(rows == 0 || (logits && target && aligned(logits, size) && aligned(target, 8)),
               "bad pointer");
  return LEMA_OK;
}

int logprob_launch(const void* logits, int32_t dtype, int64_t rows, int64_t inner, int64_t V, int64_t so,
                   int64_t si, const int64_t* target, const uint8_t* mask, float temperature, float* lp,
                   double* lp64, float* stats, const Policy& pol, hipStream_t st) {
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    logprob_kernel<T, 256><<<dim3(rows), dim3(256), 0, st>>>(
        static_cast<const T*>(logits), Rows{inner, so, si}, V, target, mask, 1.0f / temperature, lp, lp64,
        reinterpret_cast<float2*>(stats), pol);
  });
  return launch_status("logprob_kernel");
}

}  // namespace
}  // namespace lema

using namespace lema;

extern "C" int lema_token_logprobs(const void* logits, int32_t dtype, int64_t rows, int64_t inner,
                                   int64_t V, int64_t so, int64_t si, const int64_t* target,
                                   const uint8_t* mask, float temperature, float* lp, double* lp64,
                                   float* stats, void* stream) {
  clear_error();
  if (int rc = check_logits(logits, dtype, rows, inner, V, so, si, target, temperature)) return rc;
  if (rows == 0) return LEMA_OK;
  LEMA_REQUIRE(lp && aligned(lp, 4) && aligned(lp64, 8) && aligned(stats, 8), "bad pointer");
  return logprob_launch(logits, dtype, rows, inner, V, so, si, target, mask, temperature, lp, lp64, stats,
                        Policy{}, static_cast<hipStream_t>(stream));
}

extern "C" int lema_policy_loss(const void* logits, int32_t dtype, int64_t rows, int64_t inner, int64_t V,
                                int64_t so, int64_t si, const int64_t* target, const uint8_t* mask,
                                float temperature, const float* old_lp, const float* advantage,
                                const float* ref_lp, float clip_low, float clip_high, float kl,
                                float* lp, float* stats, float* term, float* coef, float* loss,
                                float* inv_n, void* stream) {
  clear_error();
  if (int rc = check_logits(logits, dtype, rows, inner, V, so, si, target, temperature)) return rc;
  LEMA_REQUIRE(loss && inv_n, "null pointer");
  LEMA_REQUIRE(rows == 0 || (old_lp && advantage && lp && stats && aligned(stats, 8) && term && coef),
               "null pointer");
  LEMA_REQUIRE(clip_low >= 0.0f && clip_high >= 0.0f, "the clip distances must not be negative");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    const Policy pol{old_lp, advantage, kl != 0.0f ? ref_lp : nullptr, term, coef, clip_low, clip_high, kl};
    if (int rc = logprob_launch(logits, dtype, rows, inner, V, so, si, target, mask, temperature, lp,
                                nullptr, stats, pol, st))
      return rc;
  }
  policy_mean_kernel<<<dim3(1), dim3(1024), 0, st>>>(term, mask, rows, loss, inv_n);
  return launch_status("policy_mean_kernel");
}

extern "C" int lema_preference_loss(const double* lp64, const float* ref_lp, const uint8_t* mask,
                                    int64_t pairs, int64_t T, float beta, float label_smoothing,
                                    float* loss, float* margin, float* coef, void* stream) {
  clear_error();
  LEMA_REQUIRE(pairs >= 1 && T >= 0 && pairs * 2 < (int64_t(1) << 31) && T < (int64_t(1) << 31),
               "bad sizes: %lld pairs of %lld tokens", (long long)pairs, (long long)T);
  LEMA_REQUIRE(loss && margin && coef && (T == 0 || (lp64 && ref_lp && aligned(lp64, 8))), "bad pointer");
  LEMA_REQUIRE(label_smoothing >= 0.0f && label_smoothing <= 1.0f,
               "label smoothing must lie in [0, 1]");
  preference_kernel<<<dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream)>>>(
      lp64, ref_lp, mask, pairs, T, beta, label_smoothing, loss, margin, coef);
  return launch_status("preference_kernel");
}

extern "C" int lema_token_logprobs_grad(const void* logits, int32_t dtype, int64_t rows, int64_t inner,
                                        int64_t V, int64_t so, int64_t si, const int64_t* target,
                                        const uint8_t* mask, float temperature, const float* stats,
                                        const float* coef, int64_t per, const float* scale0,
                                        const float* scale1, void* grad, void* stream) {
  clear_error();
  if (int rc = check_logits(logits, dtype, rows, inner, V, so, si, target, temperature)) return rc;
  if (rows == 0) return LEMA_OK;
  LEMA_REQUIRE(stats && aligned(stats, 8) && coef && per >= 1 && grad && aligned(grad, dtype_size(dtype)),
               "bad pointer");
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    logprob_grad_kernel<T, 256><<<dim3(rows), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const T*>(logits), Rows{inner, so, si}, V, target, mask, 1.0f / temperature,
        reinterpret_cast<const float2*>(stats), coef, per, scale0, scale1, static_cast<T*>(grad));
  });
  return launch_status("logprob_grad_kernel");
}
