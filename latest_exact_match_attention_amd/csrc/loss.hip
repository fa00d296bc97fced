// Losses on the log-probabilities of given tokens, from logits, and their gradients.
//
// Per row of V logits x, with k = 1 / temperature:  M = max x,  S = sum of e^(k (x - M)),
//   lp = k (x_t - M) - log S                          t the row's target
//   d lp / d x_j = k ([j = t] - e^(k (x_j - M)) / S)
// so a loss needs lp and c = d loss / d lp of each row, and the logits' gradient is c k times the
// bracket. The forward kernel reads a row once, with a running maximum and a sum that is rescaled to
// it, and keeps (M, 1 / S); the gradient's kernel reads it once more and writes it. Both are bound
// by HBM. lp is formed by one thread, in 64 bits from the fp32 difference and sum where it is not
// for a policy's row: a preference adds up those of a whole answer.
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

constexpr double kLog2e = 1.4426950408889634;

// e^(k d), d <= 0, as 2^(d log2(e) k), the factor in two parts: its rounding alone, 1.3e-8 of it and the
// same for every term, moved lp by 8e-8 on average, which adds up over an answer. hi is rounded down and
// lo above 0, so that both products of d = -inf are -inf, whose power is 0: with a lo below 0, as the
// nearest float leaves it at half of all temperatures, they would add up to NaN. `near` is that float.
struct Scale {
  float hi, lo, near;
  explicit Scale(float temperature) {
    const double k2 = kLog2e / temperature;
    near = hi = static_cast<float>(k2);
    while ((lo = static_cast<float>(k2 - hi)) <= 0.0f) hi = std::nextafter(hi, 0.0f);
  }
  __device__ __forceinline__ float exp(float d) const {
    return __builtin_amdgcn_exp2f(fmaf(d, hi, d * lo));
  }
};

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

// A row's term and coefficient from its lp, by one thread; returns the coefficient.
__device__ __forceinline__ float policy_row(const Policy& pol, int64_t row, float lp, float old, float a,
                                            float ref) {
  const float ratio = expf(lp - old), lo = 1.0f - pol.clip_low, hi = 1.0f + pol.clip_high;
  // the smaller product is the clipped one where the ratio has left the interval on the side
  // that the advantage pushes to; there it does not depend on lp
  const bool live = a >= 0.0f ? !(ratio > hi) : !(ratio < lo);
  float term = -a * (live ? ratio : a >= 0.0f ? hi : lo), coef = live ? -a * ratio : 0.0f;
  if (pol.ref != nullptr) {
    const float gap = ref - lp, grown = expm1f(gap);
    term += pol.kl * (grown - gap);
    coef -= pol.kl * grown;
  }
  pol.term[row] = term;
  pol.coef[row] = coef;
  return coef;
}

struct Running {
  float m;   // the maximum so far, -FLT_MAX at least
  double s;  // the sum rescaled to it: 64 bits, so that a likely token's 1 does not round the others off
};

// Adds n logits to r. -FLT_MAX for the maximum of nothing, or of -inf alone, keeps
// (-inf) - m = -inf, whose power is 0 at every temperature, while a NaN stays one.
template <int N>
__device__ __forceinline__ void add_logits(Running& r, const float (&x)[N], Scale k2) {
  float bm = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) bm = fmaxf(bm, x[i]);
  if (bm > r.m) {
    r.s *= k2.exp(r.m - bm);
    r.m = bm;
  }
  constexpr int kLines = N < 8 ? N : 8;  // short lines of additions, for the same reason
  float e[kLines];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float v = k2.exp(x[i] - r.m);
    e[i % kLines] = i < kLines ? v : e[i % kLines] + v;
  }
#pragma unroll
  for (int d = kLines / 2; d > 0; d /= 2)
#pragma unroll
    for (int i = 0; i < d; ++i) e[i] += e[i + d];
  r.s += e[0];
}

__device__ __forceinline__ Running join(Running a, Running b, Scale k2) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * k2.exp(a.m - m) + b.s * k2.exp(b.m - m)};
}

// The elements of a row before its first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* row, int64_t V) {
  const int64_t h = ((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T);
  return h < V ? h : V;
}

// Gradients larger than the Infinity Cache are stored past it: a batch's 16,384 rows of 50,304 in bf16
// took 468 us, not 496.
constexpr int64_t kStreamBytes = int64_t(256) << 20;

// A row of zeros: `head` elements, 16-byte pieces, `rest` elements from `tail` on.
template <typename T, int kThreads, bool kStream>
__device__ __forceinline__ void write_zeros(T* g, int64_t head, int64_t tail, int64_t rest, int64_t pieces) {
  const int tid = threadIdx.x;
  const T zero = from_f32<T>(0.0f);
  if (tid < head) g[tid] = zero;
  if (tid < rest) g[tail + tid] = zero;
  for (int64_t p = tid; p < pieces; p += kThreads) put16<kStream>(g + head + p * kPiece<T>, u32x4{0, 0, 0, 0});
}

// One workgroup per row.
template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void logprob_kernel(const T* logits, Rows rows, int64_t count,
                                                           int64_t V, const int64_t* target,
                                                           const uint8_t* mask,
                                                           float temperature, Scale k2, float* lp_out,
                                                           double* lp64_out, float2* stats, Policy pol) {
  constexpr int kWaves = kThreads / 64, n = kPiece<T>;
  __shared__ Running part[kWaves];
  const int64_t row = block_index();
  if (row >= count) return;
  const int tid = threadIdx.x;
  if (mask != nullptr && mask[row] == 0) {
    if (tid == 0) {
      lp_out[row] = 0.0f;
      if (lp64_out != nullptr) lp64_out[row] = 0.0;
      if (pol.old != nullptr) pol.term[row] = pol.coef[row] = 0.0f;
    }
    return;
  }
  const T* x = logits + rows.at(row);
  const int64_t head = head_of(x, V), pieces = (V - head) / n, tail = head + pieces * n;
  Running r{-FLT_MAX, 0.0};
  if (tid < head) {  // head < n <= 8 elements
    const float one[1] = {to_f32(x[tid])};
    add_logits<1>(r, one, k2);
  }
  if (tid < V - tail) {
    const float one[1] = {to_f32(x[tail + tid])};
    add_logits<1>(r, one, k2);
  }
  // kFlight pieces in flight; past the row the first again, for nothing
  constexpr int kFlight = 4;
  for (int64_t p0 = tid; p0 < pieces; p0 += kFlight * kThreads) {
    Piece<T> q[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int64_t p = p0 + u * kThreads;
      q[u].raw = get16(x + head + (p < pieces ? p : p0) * n);
    }
    if (p0 + (kFlight - 1) * kThreads < pieces) {
      float v[kFlight * n];
#pragma unroll
      for (int i = 0; i < kFlight * n; ++i) v[i] = to_f32(q[i / n].e[i % n]);
      add_logits<kFlight * n>(r, v, k2);
    } else {
#pragma unroll
      for (int u = 0; u < kFlight - 1; ++u) {
        if (p0 + u * kThreads >= pieces) break;
        float v[n];
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = to_f32(q[u].e[i]);
        add_logits<n>(r, v, k2);
      }
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
  const double lp = (static_cast<double>(xt) - r.m) / temperature - log(r.s);
  lp_out[row] = static_cast<float>(lp);
  if (lp64_out != nullptr) lp64_out[row] = lp;
  if (stats != nullptr) stats[row] = make_float2(r.m, static_cast<float>(1.0 / r.s));
  if (pol.old != nullptr)
    policy_row(pol, row, static_cast<float>(lp), pol.old[row], pol.adv[row],
               pol.ref != nullptr ? pol.ref[row] : 0.0f);
}

// Ends what the compiler knows of the pieces' elements, so that it forms them (and the exponentials)
// again from the pieces: kept as floats from one pass to the next they take twice the registers.
template <typename T, int P>
__device__ __forceinline__ void keep_packed(Piece<T> (&q)[P]) {
#pragma unroll
  for (int u = 0; u < P; ++u) asm volatile("" : "+v"(q[u].raw));
}

// The policy loss with its gradient for a gradient of 1 of the loss, in one pass: a row stays in the
// registers of its workgroup, P pieces a thread, between the maximum, the sum and the gradient, so
// that logits are read once. inv_n is known before.
template <typename T, int kThreads, int P, bool kStream>
__global__ __launch_bounds__(kThreads, P > 7 ? 4 : 8) void policy_grad_kernel(
    const T* logits, Rows rows, int64_t count, int64_t V, const int64_t* target, const uint8_t* mask,
    float k, Scale k2, float* lp_out, float2* stats, Policy pol, const float* inv_n, T* grad) {
  constexpr int kWaves = kThreads / 64, n = kPiece<T>;
  __shared__ float part[2][kWaves];
  __shared__ float coef;
  const int64_t row = block_index();
  if (row >= count) return;
  const int tid = threadIdx.x;
  T* g = grad + row * V;
  const int head = static_cast<int>(head_of(g, V)), pieces = static_cast<int>(V - head) / n;
  const int tail = head + pieces * n, rest = static_cast<int>(V) - tail;
  if (mask != nullptr && mask[row] == 0) {
    if (tid == 0) lp_out[row] = pol.term[row] = pol.coef[row] = 0.0f;
    write_zeros<T, kThreads, kStream>(g, head, tail, rest, pieces);
    return;
  }
  const T* x = logits + rows.at(row);
  Piece<T> q[P];
#pragma unroll
  for (int u = 0; u < P; ++u) {
    const int p = tid + u * kThreads;
    q[u].raw = p < pieces ? get16(x + head + p * n) : u32x4{0, 0, 0, 0};
  }
  // the ends' elements, -inf where this thread has none: e^-inf adds nothing
  const float xh = tid < head ? to_f32(x[tid]) : -INFINITY;
  const float xe = tid < rest ? to_f32(x[tail + tid]) : -INFINITY;
  float xt = 0.0f, old = 0.0f, adv = 0.0f, ref = 0.0f;
  const int64_t t = target[row];
  if (tid == 0) {
    xt = t >= 0 && t < V ? to_f32(x[t]) : NAN;
    old = pol.old[row];
    adv = pol.adv[row];
    if (pol.ref != nullptr) ref = pol.ref[row];
  }
  float m = fmaxf(fmaxf(xh, xe), -FLT_MAX);
#pragma unroll
  for (int u = 0; u < P; ++u)
    if (tid + u * kThreads < pieces) {
#pragma unroll
      for (int i = 0; i < n; ++i) m = fmaxf(m, to_f32(q[u].e[i]));
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) part[0][tid >> 6] = m;
  __syncthreads();
  m = part[0][tid & (kWaves - 1)];
#pragma unroll
  for (int o = kWaves / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  // 2^(x k2 - m k2) in one FMA: the rounding of m k2 is the same in every term, so it leaves the
  // softmax alone, and the sum is set right for it below
  const float mk = m * k2.near;
  const auto finish = [&](auto power, float off) {
    keep_packed(q);
    float s = power(xh) + power(xe);
#pragma unroll
    for (int u = 0; u < P; ++u)
      if (tid + u * kThreads < pieces) {
        float sa = 0.0f, sb = 0.0f;
#pragma unroll
        for (int i = 0; i < n; i += 2) {
          sa += power(to_f32(q[u].e[i]));
          sb += power(to_f32(q[u].e[i + 1]));
        }
        s += sa + sb;
      }
    s = wave_sum(s);
    if ((tid & 63) == 0) part[1][tid >> 6] = s;
    __syncthreads();
    s = part[1][tid & (kWaves - 1)];
#pragma unroll
    for (int o = kWaves / 2; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (tid == 0) {
      const float sum = s * __builtin_amdgcn_exp2f(-off);
      const float lp = fmaf(xt - m, k, -logf(sum));
      lp_out[row] = lp;
      stats[row] = make_float2(m, 1.0f / sum);
      coef = policy_row(pol, row, lp, old, adv, ref);
    }
    __syncthreads();
    const float c = coef * k * *inv_n, cs = c * (1.0f / s);
    if (c == 0.0f) {
      write_zeros<T, kThreads, kStream>(g, head, tail, rest, pieces);
      return;
    }
    keep_packed(q);
    const auto one = [&](float v) { return -cs * power(v); };
    const auto hit = [&](float v) { return fmaf(-cs, power(v), c); };
    if (tid < head) g[tid] = from_f32<T>(tid == t ? hit(xh) : one(xh));
    if (tid < rest) g[tail + tid] = from_f32<T>(tail + tid == t ? hit(xe) : one(xe));
    const int body_t = static_cast<int>(t) - head;  // the target's place in the body, if it is there
#pragma unroll
    for (int u = 0; u < P; ++u) {
      const int p = tid + u * kThreads;
      if (p < pieces) {
        Piece<T> o;
#pragma unroll
        for (int i = 0; i < n; ++i) o.e[i] = from_f32<T>(one(to_f32(q[u].e[i])));
        if (body_t >= 0 && p == body_t / n) {
#pragma unroll
          for (int i = 0; i < n; ++i)
            if (i == body_t % n) o.e[i] = from_f32<T>(hit(to_f32(q[u].e[i])));
        }
        put16<kStream>(g + head + p * n, o.raw);
      }
    }
  };
  if (fabsf(mk) < 1048576.0f)  // its rounding is then below 2^-4
    finish([&](float v) { return __builtin_amdgcn_exp2f(fmaf(v, k2.near, -mk)); }, fmaf(m, k2.near, -mk));
  else  // logits of any size, up to those whose product leaves fp32's range
    finish([&](float v) { return __builtin_amdgcn_exp2f((v - m) * k2.near); }, 0.0f);
}

// Sum over the wavefront in 64 bits.
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// inv_n = scale / counted rows (scale where there are none). 16 mask bytes a thread at a time where
// they are aligned to it.
__global__ __launch_bounds__(1024) void policy_count_kernel(const uint8_t* mask, int64_t rows, float scale,
                                                            float* inv_n) {
  __shared__ uint32_t sums[16];
  uint32_t n = 0;
  const bool pieces = (reinterpret_cast<uintptr_t>(mask) & 15) == 0;
  const int64_t body = mask != nullptr && pieces ? rows / 16 * 16 : 0;
  for (int64_t i = static_cast<int64_t>(threadIdx.x) * 16; i < body; i += 1024 * 16) {
    union {
      u32x4 raw;
      uint8_t b[16];
    } q;
    q.raw = *reinterpret_cast<const u32x4*>(mask + i);
#pragma unroll
    for (int k = 0; k < 16; ++k) n += q.b[k] != 0;
  }
  if (mask != nullptr)
    for (int64_t i = body + threadIdx.x; i < rows; i += 1024) n += mask[i] != 0;
  else if (threadIdx.x == 0)
    n = static_cast<uint32_t>(rows);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < 16; ++w) n += sums[w];
  *inv_n = n > 0 ? static_cast<float>(scale / static_cast<double>(n)) : scale;
}

// loss = sum of the terms * inv_n, in 64 bits; `term` starts at a 4-byte boundary of any kind.
__global__ __launch_bounds__(1024) void policy_mean_kernel(const float* term, int64_t rows,
                                                           const float* inv_n, float* loss) {
  __shared__ double sums[16];
  double t = 0.0;
  for (int64_t i = threadIdx.x; i < rows; i += 16 * 1024) {
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u)  // 16 rows in flight; past the end the first one again
      v[u] = term[i + u * 1024 < rows ? i + u * 1024 : i];
#pragma unroll
    for (int u = 0; u < 16; ++u) t += i + u * 1024 < rows ? v[u] : 0.0f;
  }
  t = wave_sum64(t);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  t = wave_sum64(threadIdx.x < 16 ? sums[threadIdx.x] : 0.0);
  if (threadIdx.x == 0) *loss = static_cast<float>(t * *inv_n);
}

// One workgroup: 16 / kTeams wavefronts (a team) a pair at a time, answers p and pairs + p of T rows
// each, 4 rows of either in flight.
template <int kTeams>
__global__ __launch_bounds__(1024) void preference_kernel(const double* lp, const float* ref,
                                                          const uint8_t* mask, int64_t pairs, int64_t T,
                                                          float beta, float smooth, float* loss,
                                                          float* margin, float* coef) {
  constexpr int kWaves = 16 / kTeams, kStep = 64 * kWaves;
  __shared__ double sums[2][16];
  const int w = threadIdx.x >> 6, team = w / kWaves, lane = threadIdx.x % kStep;
  double total = 0.0;
  int turn = 0;
  for (int64_t p0 = 0; p0 < pairs; p0 += kTeams, turn ^= 1) {
    const int64_t p = p0 + team;
    double d = 0.0;
    if (p < pairs)
      for (int64_t i = lane; i < T; i += 4 * kStep) {
        double l[2][4];
        float r[2][4];
        bool counts[2][4];
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int64_t j = (side * pairs + p) * T + (i + u * kStep < T ? i + u * kStep : i);
            l[side][u] = lp[j];
            r[side][u] = ref[j];
            counts[side][u] = (mask == nullptr || mask[j] != 0) && i + u * kStep < T;
          }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (counts[0][u]) d += l[0][u] - r[0][u];
          if (counts[1][u]) d -= l[1][u] - r[1][u];
        }
      }
    d = wave_sum64(d);
    if ((threadIdx.x & 63) == 0) sums[turn][w] = d;
    __syncthreads();  // the other half is written before anyone is two rounds ahead
    if (lane == 0 && p < pairs) {
      d = 0.0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) d += sums[turn][team * kWaves + i];
      const float m = static_cast<float>(beta * d), e = expf(-fabsf(m));
      const float tail = log1pf(e), small = e / (1.0f + e), large = 1.0f / (1.0f + e);
      // -log sigmoid(m) = tail + max(-m, 0);  sigmoid(|m|) = large, sigmoid(-|m|) = small. A part of
      // weight 0 is left out: of an infinite margin (a banned word in an answer) it may be infinite
      if (smooth < 1.0f) total += (1.0f - smooth) * (tail + fmaxf(-m, 0.0f));
      if (smooth > 0.0f) total += smooth * (tail + fmaxf(m, 0.0f));
      if (m != m) total = m;
      // d term / d m = -(1 - smooth) sigmoid(-m) + smooth sigmoid(m)
      const float dm = smooth * (m > 0.0f ? large : small) - (1.0f - smooth) * (m > 0.0f ? small : large);
      const float c = (m != m ? m : dm) * beta / static_cast<float>(pairs);
      margin[p] = m;
      coef[p] = c;
      coef[pairs + p] = -c;
    }
  }
  __syncthreads();
  if (lane == 0) sums[0][team] = total;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < kTeams; ++i) total += sums[0][i];
  *loss = static_cast<float>(total / static_cast<double>(pairs));
}

// grad[row] = c k ([j = t] - e^(k (x_j - M)) / S), c = coef[row / per] * *scale0 * *scale1 (each
// NULL: 1). grad is contiguous [rows, V]. Rows of c = 0 are not read; others whose target lies outside
// [0, V) become NaN. A gradient that is stored past
// the Infinity Cache leaves it to the logits, whose last rows the forward has just read: they come
// first (8192 rows of 50,304 in bf16: 203 us, not 222).
// unit_done: the forward has written the gradient for *scale0 = 1, which is then left as it is.
template <typename T, int kThreads, bool kStream>
__global__ __launch_bounds__(kThreads) void logprob_grad_kernel(
    const T* logits, Rows rows, int64_t count, int64_t V, const int64_t* target, const uint8_t* mask, float k,
    Scale k2, const float2* stats, const float* coef, int64_t per, const float* scale0, const float* scale1,
    bool unit_done, T* grad) {
  constexpr int n = kPiece<T>;
  const int tid = threadIdx.x;
  const float s0 = scale0 != nullptr ? *scale0 : 1.0f;
  if (unit_done && s0 == 1.0f) return;
  for (int64_t turn = blockIdx.x; turn < count; turn += gridDim.x) {
    const int64_t row = kStream ? count - 1 - turn : turn;
    T* g = grad + row * V;
    float c = 0.0f;
    if (mask == nullptr || mask[row] != 0) {
      c = coef[row / per] * k * s0;
      if (scale1 != nullptr) c *= *scale1;
    }
    const int64_t head = head_of(g, V), pieces = (V - head) / n, tail = head + pieces * n;
    if (c == 0.0f) {
      write_zeros<T, kThreads, kStream>(g, head, tail, V - tail, pieces);
      continue;
    }
    const float2 st = stats[row];
    const int64_t t = target[row];
    if (t < 0 || t >= V) c = NAN;  // as the row's lp
    const float cs = c * st.y;
    const T* x = logits + rows.at(row);
    const auto one = [&](int64_t j, float v) {
      const float e = k2.exp(v - st.x);
      return from_f32<T>(j == t ? fmaf(-cs, e, c) : -cs * e);
    };
    if (tid < head) g[tid] = one(tid, to_f32(x[tid]));
    if (tid < V - tail) g[tail + tid] = one(tail + tid, to_f32(x[tail + tid]));
    for (int64_t p0 = tid; p0 < pieces; p0 += 4 * kThreads) {
      Piece<T> q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // 4 pieces in flight; past the row the first again
        const int64_t p = p0 + u * kThreads;
        q[u].raw = get16(x + head + (p < pieces ? p : p0) * n);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t p = p0 + u * kThreads;
        if (p >= pieces) break;
#pragma unroll
        for (int i = 0; i < n; ++i) q[u].e[i] = one(head + p * n + i, to_f32(q[u].e[i]));
        put16<kStream>(g + head + p * n, q[u].raw);
      }
    }
  }
}

// 1024 threads a row where it has two 16-byte pieces for each: the gradient of 8192 rows of 50,304 in
// bf16 took 228 us with 256 threads and 207 with 1024 (the log-probabilities 138 either way), 200 rows
// 13.9 and 11.3 (14.7 and 9.5).
bool wide_rows(int32_t dtype, int64_t V) { return V * dtype_size(dtype) >= 2048 * 16; }

int check_logits(const void* logits, int32_t dtype, int64_t rows, int64_t inner, int64_t V, int64_t so,
                 int64_t si, const int64_t* target, float temperature) {
  const int size = dtype_size(dtype);
  LEMA_REQUIRE(size != 0, "unknown dtype %d", dtype);
  LEMA_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && V >= 1 && V < (int64_t(1) << 31),
               "bad sizes: %lld rows of %lld logits", (long long)rows, (long long)V);
  LEMA_REQUIRE(inner >= 1 && so >= 0 && si >= 0, "bad strides");
  LEMA_REQUIRE(temperature > 0.0f && std::isfinite(temperature) &&
                   std::isfinite(static_cast<float>(kLog2e / temperature)) && 1.0f / temperature > 0.0f,
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
    const bool wide = wide_rows(dtype, V);
    const auto kernel = wide ? logprob_kernel<T, 1024> : logprob_kernel<T, 256>;
    kernel<<<blocks_of(rows), dim3(wide ? 1024 : 256), 0, st>>>(
        static_cast<const T*>(logits), Rows{inner, so, si}, rows, V, target, mask, temperature,
        Scale(temperature), lp, lp64, reinterpret_cast<float2*>(stats), pol);
  });
  return launch_status("logprob_kernel");
}

int grad_launch(const void* logits, int32_t dtype, int64_t rows, int64_t inner, int64_t V, int64_t so,
                int64_t si, const int64_t* target, const uint8_t* mask, float temperature, const float* stats,
                const float* coef, int64_t per, const float* scale0, const float* scale1, bool unit_done,
                void* grad, hipStream_t st) {
  for_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const bool wide = wide_rows(dtype, V);
    const bool past = rows * V * static_cast<int64_t>(sizeof(T)) > kStreamBytes;
    const auto kernel = wide ? (past ? logprob_grad_kernel<T, 1024, true> : logprob_grad_kernel<T, 1024, false>)
                             : (past ? logprob_grad_kernel<T, 256, true> : logprob_grad_kernel<T, 256, false>);
    // where nothing is likely to be left to do, few workgroups (16,384 that end at once take 17 us)
    const int64_t most = unit_done ? 512 : 1 << 21, grid = rows < most ? rows : most;
    kernel<<<dim3(grid), dim3(wide ? 1024 : 256), 0, st>>>(
        static_cast<const T*>(logits), Rows{inner, so, si}, rows, V, target, mask, 1.0f / temperature,
        Scale(temperature), reinterpret_cast<const float2*>(stats), coef, per, scale0, scale1, unit_done,
        static_cast<T*>(grad));
  });
  return launch_status("logprob_grad_kernel");
}

// Whether policy_grad_kernel holds a row.
bool one_pass(int32_t dtype, int64_t V) { return V * dtype_size(dtype) <= 16 * 1024 * 16; }

// Calls f with the threads of a row's workgroup and the pieces each holds, as compile-time constants.
// Up to 7 pieces leave a CU two workgroups of 1024, 10 and 16 one: 6144 rows of bf16 ran at 4.9 to 5.3 TB/s
// up to 57,344 logits, at 4.7 to 4.8 from 65,536 to 131,072, and read twice, at 3.8, beyond.
template <typename T, typename F>
inline void for_pieces(int64_t V, F f) {
  using std::integral_constant;
  const int64_t pieces = V / kPiece<T>;
  if (pieces <= 256)
    f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (pieces <= 512)
    f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (pieces <= 1024)
    f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else if (pieces <= 2048)
    f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  else if (pieces <= 4096)
    f(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
  else if (pieces <= 7168)
    f(integral_constant<int, 1024>{}, integral_constant<int, 7>{});
  else if (pieces <= 10240)
    f(integral_constant<int, 1024>{}, integral_constant<int, 10>{});
  else
    f(integral_constant<int, 1024>{}, integral_constant<int, 16>{});
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
                                float scale, float* lp, float* stats, float* term, float* coef, float* loss,
                                float* inv_n, void* grad, void* stream) {
  clear_error();
  if (int rc = check_logits(logits, dtype, rows, inner, V, so, si, target, temperature)) return rc;
  LEMA_REQUIRE(loss && inv_n, "null pointer");
  LEMA_REQUIRE(rows == 0 || (old_lp && advantage && lp && stats && aligned(stats, 8) && term && coef),
               "null pointer");
  LEMA_REQUIRE(clip_low >= 0.0f && clip_high >= 0.0f, "the clip distances must not be negative");
  LEMA_REQUIRE(aligned(grad, dtype_size(dtype)), "bad pointer");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const Policy pol{old_lp, advantage, kl != 0.0f ? ref_lp : nullptr, term, coef, clip_low, clip_high, kl};
  const bool fused = grad != nullptr && rows > 0 && one_pass(dtype, V);
  policy_count_kernel<<<dim3(1), dim3(1024), 0, st>>>(mask, rows, scale, inv_n);
  if (fused) {
    for_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      for_pieces<T>(V, [&](auto threads, auto count) {
        constexpr int kThreads = decltype(threads)::value, P = decltype(count)::value;
        const auto kernel = rows * V * static_cast<int64_t>(sizeof(T)) > kStreamBytes
                                ? policy_grad_kernel<T, kThreads, P, true>
                                : policy_grad_kernel<T, kThreads, P, false>;
        kernel<<<blocks_of(rows), dim3(kThreads), 0, st>>>(
            static_cast<const T*>(logits), Rows{inner, so, si}, rows, V, target, mask, 1.0f / temperature,
            Scale(temperature), lp, reinterpret_cast<float2*>(stats), pol, inv_n,
            static_cast<T*>(grad));
      });
    });
    if (int rc = launch_status("policy_grad_kernel")) return rc;
  } else if (rows > 0) {
    if (int rc = logprob_launch(logits, dtype, rows, inner, V, so, si, target, mask, temperature, lp,
                                nullptr, stats, pol, st))
      return rc;
  }
  policy_mean_kernel<<<dim3(1), dim3(1024), 0, st>>>(term, rows, inv_n, loss);
  if (int rc = launch_status("policy_mean_kernel")) return rc;
  if (grad == nullptr || fused || rows == 0) return LEMA_OK;
  return grad_launch(logits, dtype, rows, inner, V, so, si, target, mask, temperature, stats, coef, 1,
                     inv_n, nullptr, false, grad, st);
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
  const auto kernel = pairs >= 16 ? preference_kernel<16> : pairs >= 3 ? preference_kernel<4>
                                                                        : preference_kernel<1>;
  kernel<<<dim3(1), dim3(1024), 0, static_cast<hipStream_t>(stream)>>>(
      lp64, ref_lp, mask, pairs, T, beta, label_smoothing, loss, margin, coef);
  return launch_status("preference_kernel");
}

extern "C" int lema_token_logprobs_grad(const void* logits, int32_t dtype, int64_t rows, int64_t inner,
                                        int64_t V, int64_t so, int64_t si, const int64_t* target,
                                        const uint8_t* mask, float temperature, const float* stats,
                                        const float* coef, int64_t per, const float* scale0,
                                        const float* scale1, int32_t unit_done, void* grad, void* stream) {
  clear_error();
  if (int rc = check_logits(logits, dtype, rows, inner, V, so, si, target, temperature)) return rc;
  if (rows == 0) return LEMA_OK;
  LEMA_REQUIRE(stats && aligned(stats, 8) && coef && per >= 1 && grad && aligned(grad, dtype_size(dtype)) &&
                   (unit_done == 0 || scale0 != nullptr),
               "bad pointer");
  return grad_launch(logits, dtype, rows, inner, V, so, si, target, mask, temperature, stats, coef, per,
                     scale0, scale1, unit_done != 0, grad, static_cast<hipStream_t>(stream));
}
