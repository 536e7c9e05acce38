// Losses of preference and policy fine-tuning over logits [B, L, V], with their gradients.
//
//   logp[b, t] = x[target] - lse(x)                                  x = logits[b, t, :]
//
// preference (rows 2j and 2j + 1 of the batch answer one prompt, 2j the better way; r: log-likelihoods
// under a reference model):
//   s_b = sum_t w[b, t] logp[b, t]          d_j = beta ((s_2j - r_2j) - (s_2j+1 - r_2j+1))
//   loss = scale * sum_j (1 - e) log(1 + exp(-d_j)) + e log(1 + exp(d_j))
//   dloss/ds_2j = scale * beta * (sigmoid(d_j) - 1 + e) = -dloss/ds_2j+1
// policy (A: advantages, old: log-probabilities when the answer was drawn, ref: under the reference):
//   rho = exp(logp - old)                   k = exp(ref - logp) - 1 - (ref - logp)
//   loss = scale * sum w (kl_weight k - min(A rho, A clip(rho, 1 - low, 1 + high)))
//   dloss/dlogp = scale w (kl_weight (1 - exp(ref - logp)) - A rho [rho not held by the clip])
// both: dlogits = dloss/dlogp (onehot - softmax)
//
// A token of weight 0 does not count, whatever its logits hold: they are not read, and their gradient is
// zero. A target outside of the vocabulary gives NaN. Sums over tokens and pairs are held in 64 bits and
// taken in an order that depends on the sizes alone.
//
// What bounds it: memory; the logits that count read once, the gradient written once.
#include <atomic>
#include <cmath>
#include <cstddef>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "t5x_ops.h"

namespace t5x {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowThreads = 512;
constexpr int kCtasPerSm = 16;  // at most, of every grid here whose CTAs leave sums in the scratch

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 16 bytes of logits as floats and back.
template <typename T>
struct Pack;
template <>
struct Pack<float> {
  static constexpr int kN = 4;
  __device__ static void load(const float* p, float* x) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
  __device__ static void store(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  }
  __device__ static float one(float v) { return v; }
  __device__ static float back(float v) { return v; }
};
template <>
struct Pack<__nv_bfloat16> {
  static constexpr int kN = 8;
  __device__ static void load(const __nv_bfloat16* p, float* x) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  __device__ static void store(__nv_bfloat16* p, const float* x) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ static float one(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 back(float v) { return __float2bfloat16(v); }
};

// Calls many(p, index) for every whole 16 bytes of the row and one(index) for the values in front of the
// first 16-byte boundary and behind the last.
template <typename T, typename Many, typename One>
__device__ __forceinline__ void over_row(const T* row, int vocab, int tid, int threads, Many many, One one) {
  constexpr int kN = Pack<T>::kN;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T));
  int head = off ? kN - off : 0;
  if (head > vocab) head = vocab;
  const int packs = (vocab - head) / kN;
  for (int i = tid; i < head; i += threads) one(i);
#pragma unroll 4
  for (int i = tid; i < packs; i += threads) many(head + i * kN);
  for (int i = head + packs * kN + tid; i < vocab; i += threads) one(i);
}

// Largest logit and sum of exp(x - largest). (8 bytes that one instruction copies or stores.)
struct alignas(8) Softmax {
  float most, sum;
};
// (-inf where nothing has been seen: the difference of two such is not taken)
__device__ __forceinline__ Softmax join(Softmax a, Softmax b) {
  const float m = fmaxf(a.most, b.most);
  const float ref = m == -INFINITY ? 0.f : m;
  return {m, a.sum * exp2_approx((a.most - ref) * kLog2e) + b.sum * exp2_approx((b.most - ref) * kLog2e)};
}

template <typename T>
__device__ __forceinline__ Softmax row_softmax(const T* row, int vocab, int tid, int threads) {
  constexpr int kN = Pack<T>::kN;
  float most = -INFINITY, sum = 0.f;
  auto raise = [&](float m) {
    if (m > most) {
      sum *= exp2_approx((most - m) * kLog2e);  // (nothing seen yet: 0 * exp(-inf))
      most = m;
    }
  };
  over_row(
      row, vocab, tid, threads,
      [&](int at) {
        float x[kN];
        Pack<T>::load(row + at, x);
        float m = x[0];
#pragma unroll
        for (int i = 1; i < kN; ++i) m = fmaxf(m, x[i]);
        raise(m);
        const float ref = most == -INFINITY ? 0.f : most;
#pragma unroll
        for (int i = 0; i < kN; ++i) sum += exp2_approx((x[i] - ref) * kLog2e);
      },
      [&](int at) {
        const float x = Pack<T>::one(row[at]);
        raise(x);
        sum += exp2_approx((x - (most == -INFINITY ? 0.f : most)) * kLog2e);
      });
  return {most, sum};
}

// grad = by * (onehot - softmax)
template <typename T>
__device__ __forceinline__ void row_gradient(const T* row, T* grad, int vocab, Softmax s, int target, float by,
                                             int tid, int threads) {
  constexpr int kN = Pack<T>::kN;
  const float k = -by / s.sum;
  over_row(
      row, vocab, tid, threads,
      [&](int at) {
        float x[kN];
        Pack<T>::load(row + at, x);
#pragma unroll
        for (int i = 0; i < kN; ++i) x[i] = k * exp2_approx((x[i] - s.most) * kLog2e);
        if (target >= at && target < at + kN) {
#pragma unroll
          for (int i = 0; i < kN; ++i)
            if (target == at + i) x[i] += by;
        }
        Pack<T>::store(grad + at, x);
      },
      [&](int at) {
        const float g = k * exp2_approx((Pack<T>::one(row[at]) - s.most) * kLog2e);
        grad[at] = Pack<T>::back(at == target ? g + by : g);
      });
}

template <typename T>
__device__ __forceinline__ void row_zero(T* grad, int vocab, int tid, int threads) {
  over_row(
      grad, vocab, tid, threads, [&](int at) { *reinterpret_cast<uint4*>(grad + at) = make_uint4(0, 0, 0, 0); },
      [&](int at) { grad[at] = Pack<T>::back(0.f); });
}

// log softmax of the target. A row of -inf alone or with +inf or NaN gives NaN, as does a bad target.
template <typename T>
__device__ __forceinline__ float log_prob(const T* row, int vocab, long long target, Softmax s) {
  if (target < 0 || target >= vocab || s.most == -INFINITY) return NAN;
  return (Pack<T>::one(row[target]) - s.most) - log1pf(s.sum - 1.f);
}

// The softmax of what the 32 lanes have seen, in every lane.
__device__ __forceinline__ Softmax join_lanes(Softmax s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Softmax other = {__shfl_xor_sync(0xffffffffu, s.most, o), __shfl_xor_sync(0xffffffffu, s.sum, o)};
    s = join(s, other);
  }
  return s;
}

struct Rows {
  long long rows;  // B * L
  int length, vocab;
  long long stride_b, stride_t;  // in values, of the logits
  long long grad_b, grad_t;      // of their gradient
  const long long* targets;
  const float* weights;  // null: all 1
};
// Where a row of the logits and of their gradient begins.
struct RowAt {
  long long b, logits, grad;
};
__device__ __forceinline__ RowAt row_at(const Rows& r, long long row) {
  const long long b = row / r.length, t = row - b * r.length;
  return {b, b * r.stride_b + t * r.stride_t, b * r.grad_b + t * r.grad_t};
}

// Sums over the threads of the CTA, in every thread, in a fixed order.
template <int kThreads, int kSums>
__device__ __forceinline__ void cta_sums(double (&v)[kSums]) {
  constexpr int kWarps = kThreads / 32;
  __shared__ double part[kSums][kWarps];
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < kSums; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
  __syncthreads();
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kSums; ++i) part[i][threadIdx.x >> 5] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSums; ++i) v[i] = part[i][lane % kWarps];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) {
#pragma unroll
    for (int i = 0; i < kSums; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
}

// Whether this CTA is the last of the grid to come here; what the others wrote before is then visible.
__device__ __forceinline__ bool last_cta(unsigned* arrived) {
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(arrived, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  return last;
}

__device__ __forceinline__ float scale_of(const float* normalizer, float scale) {
  return normalizer != nullptr ? 1.f / *normalizer : scale;
}

// ---- policy ----
struct Policy {
  const float *old, *ref, *advantages;  // ref null: no KL term
  long long adv_b, adv_t;               // strides of the advantages
  float low, high, kl_weight, scale;    // the clip's borders, 1 - low and 1 + high
  const float* normalizer;              // device scalar in the place of 1 / scale, or null
};
struct PolicyToken {
  float loss, kl, clipped;  // before weight and scale
  float slope;              // dloss / dlogp
};
struct PolicyInputs {
  float old, ref, advantage;
};
__device__ __forceinline__ PolicyInputs policy_inputs(const Policy& p, long long row, long long b, long long t) {
  return {p.old[row], p.ref != nullptr ? p.ref[row] : 0.f, p.advantages[b * p.adv_b + t * p.adv_t]};
}
__device__ __forceinline__ PolicyToken policy_token(const Policy& p, PolicyInputs in, float logp) {
  const float a = in.advantage;
  const float ratio = expf(logp - in.old);
  const float gain = a * ratio, held = a * fminf(fmaxf(ratio, p.low), p.high);
  PolicyToken k;
  k.clipped = held < gain ? 1.f : 0.f;
  // (NaN on either side stays: fminf and the clip would drop it)
  k.loss = -(gain != gain ? gain : fminf(gain, held));
  k.slope = held < gain ? 0.f : -gain;
  k.kl = 0.f;
  if (p.ref != nullptr) {
    const float apart = in.ref - logp, e = expm1f(apart);
    k.kl = apart == INFINITY ? apart : e - apart;
    if (p.kl_weight != 0.f) {  // (of a term that only is reported an overflow stays out of the loss)
      k.loss += p.kl_weight * k.kl;
      k.slope -= p.kl_weight * e;
    }
  }
  return k;
}

// out: loss, kl, clipped, weight
__device__ __forceinline__ void policy_finish(double (&sums)[4], const Policy& p, double* partial, unsigned* arrived,
                                              float* out) {
  constexpr int kThreads = kRowThreads;
  cta_sums<kThreads>(sums);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (threadIdx.x == 0) partial[blockIdx.x * 4 + i] = sums[i];
  if (!last_cta(arrived)) return;
  const double scale = p.normalizer != nullptr ? 1.0 / static_cast<double>(*p.normalizer) : p.scale;
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (int k = threadIdx.x; k < static_cast<int>(gridDim.x); k += kThreads) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += __ldcg(partial + k * 4 + i);
  }
  cta_sums<kThreads>(v);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (threadIdx.x == 0) out[i] = static_cast<float>(i < 2 ? v[i] * scale : v[i]);
}

// Short rows, a warp each.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    policy_short_rows_kernel(const T* __restrict__ logits, T* __restrict__ grad, const Rows r, const Policy p,
                             double* partial, unsigned* arrived, float* out) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (kRowThreads / 32);
  const float scale = scale_of(p.normalizer, p.scale);
  double sums[4] = {0.0, 0.0, 0.0, 0.0};
  for (long long row = blockIdx.x * static_cast<long long>(kRowThreads / 32) + (threadIdx.x >> 5); row < r.rows;
       row += warps) {
    const float w = r.weights != nullptr ? r.weights[row] : 1.f;
    const RowAt at = row_at(r, row);
    if (w == 0.f) {
      if (grad != nullptr) row_zero(grad + at.grad, r.vocab, lane, 32);
      continue;
    }
    const long long target = r.targets[row];
    const PolicyInputs in = policy_inputs(p, row, at.b, row - at.b * r.length);
    const Softmax s = join_lanes(row_softmax(logits + at.logits, r.vocab, lane, 32));
    const float logp = log_prob(logits + at.logits, r.vocab, target, s);
    const PolicyToken k = policy_token(p, in, logp);
    if (lane == 0) {
      sums[0] += static_cast<double>(w) * k.loss;
      sums[1] += static_cast<double>(w) * k.kl;
      sums[2] += static_cast<double>(w) * k.clipped;
      sums[3] += w;
    }
    if (grad != nullptr)
      row_gradient(logits + at.logits, grad + at.grad, r.vocab, s,
                   target >= 0 && target < r.vocab ? static_cast<int>(target) : -1, w * k.slope * scale, lane, 32);
  }
  policy_finish(sums, p, partial, arrived, out);
}

// The loss from log-probabilities; slope: their gradient, or null.
__global__ void __launch_bounds__(kRowThreads)
    policy_tokens_kernel(const float* __restrict__ logp, float* __restrict__ slope, const Rows r, const Policy p,
                         double* partial, unsigned* arrived, float* out) {
  const float scale = scale_of(p.normalizer, p.scale);
  double sums[4] = {0.0, 0.0, 0.0, 0.0};
  for (long long row = blockIdx.x * static_cast<long long>(kRowThreads) + threadIdx.x; row < r.rows;
       row += static_cast<long long>(gridDim.x) * kRowThreads) {
    const float w = r.weights != nullptr ? r.weights[row] : 1.f;
    float by = 0.f;
    if (w != 0.f) {
      const long long b = row / r.length;
      const PolicyToken k = policy_token(p, policy_inputs(p, row, b, row - b * r.length), logp[row]);
      sums[0] += static_cast<double>(w) * k.loss;
      sums[1] += static_cast<double>(w) * k.kl;
      sums[2] += static_cast<double>(w) * k.clipped;
      sums[3] += w;
      by = w * k.slope * scale;
    }
    if (slope != nullptr) slope[row] = by;
  }
  policy_finish(sums, p, partial, arrived, out);
}

// ---- preference ----
struct Preference {
  const float* ref;  // [B]
  float beta, smoothing, scale;
  const float* normalizer;
};

// Short rows, a warp each: softmax and log-probability.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    preference_short_rows_kernel(const T* __restrict__ logits, const Rows r, Softmax* __restrict__ softmax,
                                 float* __restrict__ logp, unsigned* arrived) {
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;  // for the launch of the pairs
  const long long warps = static_cast<long long>(gridDim.x) * (kRowThreads / 32);
  for (long long row = blockIdx.x * static_cast<long long>(kRowThreads / 32) + (threadIdx.x >> 5); row < r.rows;
       row += warps) {
    if (r.weights != nullptr && r.weights[row] == 0.f) continue;
    const T* x = logits + row_at(r, row).logits;
    const Softmax s = join_lanes(row_softmax(x, r.vocab, lane, 32));
    if (lane == 0) {
      softmax[row] = s;
      logp[row] = log_prob(x, r.vocab, r.targets[row], s);
    }
  }
}

struct Margin {
  double margin;      // of sums of many tokens: in 64 bits; what follows of their difference in 32
  float loss, slope;  // slope: dloss / d(score of the preferred)
};
__device__ __forceinline__ Margin pair_margin(const Preference& p, bool real, double s0, double s1, float r0, float r1,
                                              float scale) {
  Margin m = {0.0, 0.f, 0.f};
  if (!real) return m;
  m.margin = p.beta * ((s0 - r0) - (s1 - r1));
  const float d = static_cast<float>(m.margin);
  // log(1 + exp(-d)) = log1p(exp(-|d|)) + max(-d, 0)
  const float e = expf(-fabsf(d)), tail = log1pf(e);
  const float sigmoid = (d >= 0.f ? 1.f : e) / (1.f + e);
  // (a side of weight 0 may be infinite: the answer that is not preferred cannot be)
  const float weight = 1.f - p.smoothing;
  m.loss = d != d ? d
                  : (weight > 0.f ? weight * (tail + fmaxf(-d, 0.f)) : 0.f) +
                        (p.smoothing > 0.f ? p.smoothing * (tail + fmaxf(d, 0.f)) : 0.f);
  // sigmoid - 1 + e, near 0 from the side that does not cancel
  const float under = (d >= 0.f ? e : 1.f) / (1.f + e);  // sigmoid(-d)
  m.slope = p.beta * (p.smoothing * sigmoid - weight * under) * scale;
  return m;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    preference_short_gradient_kernel(const T* __restrict__ logits, T* __restrict__ grad, const Rows r,
                                     const Softmax* __restrict__ softmax, const float* __restrict__ by) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (kRowThreads / 32);
  for (long long row = blockIdx.x * static_cast<long long>(kRowThreads / 32) + (threadIdx.x >> 5); row < r.rows;
       row += warps) {
    const float w = r.weights != nullptr ? r.weights[row] : 1.f;
    const RowAt at = row_at(r, row);
    if (w == 0.f) {
      row_zero(grad + at.grad, r.vocab, lane, 32);
      continue;
    }
    const long long target = r.targets[row];
    row_gradient(logits + at.logits, grad + at.grad, r.vocab, softmax[row],
                 target >= 0 && target < r.vocab ? static_cast<int>(target) : -1, w * by[at.b], lane, 32);
  }
}

// ---- long rows ----
// A CTA takes a row, or its part of a row that a cluster of CTAs shares, into registers: kPacks times 16 bytes
// a thread. The row's softmax and its gradient are both made from there, so that logits are read once, and the
// next row is on its way into shared memory meanwhile. Larger rows than eight CTAs hold go by in chunks, which
// are read a second time for the gradient.
//
// What bounds it: memory. Policy, 128 x 114 x 32128 bf16 of which 80% count: 313 us, 5.4 TB/s of what has to be read
// and written; 7 x 189 x 250112 fp32: 431 us, 5.5 TB/s; the gradients of a preference loss, 64 x 114 x 32128 bf16: 133
// us, 6.3 TB/s. Close behind come the instructions (60% of the issue slots, the exponentials' unit 54%), and a policy
// row has a chain from its last part to its slope that the SM's other CTA has to fill. So one thread finds out about
// the rows, a few of them ahead, and leaves that for all in shared memory (488 us where all of them did), a warp's
// share lies side by side, and what the loss itself needs is added behind the slope. Tried without effect: 256
// threads with twice the registers; the next row asked for in four groups; an eighth of the exponentials as
// polynomials (325); a row over two blocks of 256 threads (327); no second barrier, each warp joining the parts by
// itself (332); exponentials kept for the gradient, by which one block of 512 threads fills an SM (370).
constexpr int kPacks = 8;

// An exponential exp(x - most) is exp2(x log2 e - ref) here, a fused product and difference, with ref = most log2 e
// as rounded: the same factor, 2^(most log2 e - ref), for the sum, the target and the gradient. Up to 65536 that factor
// is within 2^(1/256) of 1. From there on it grows until it overflows (at 1e10, a usual value for masked
// places, 2^440), and the exponential is exp2((x - most) log2 e). So each part of a row is held against its own
// largest in one of two ways, and joining parts puts their sums on one reference (see shift_of).
constexpr float kFused = 65536.f;
__device__ __forceinline__ bool huge(float most) { return !(fabsf(most) <= kFused); }  // (NaN and the infinities too)
// What the reference of a largest is rounded by: ref = most log2 e - rounded_off(most).
__device__ __forceinline__ float rounded_off(float most) {
  return huge(most) ? 0.f : fmaf(most, kLog2e, -__fmul_rn(most, kLog2e));
}
// log2 of the factor that takes a sum held against a to one held against b; 0 for a = b = -inf
__device__ __forceinline__ float shift_of(float a, float b) {
  if (huge(a) || huge(b)) return a == b ? 0.f : fmaf(a - b, kLog2e, rounded_off(b) - rounded_off(a));
  return __fmul_rn(a, kLog2e) - __fmul_rn(b, kLog2e);
}
__device__ __forceinline__ float exp_from(float x, float most) {
  return exp2_approx(huge(most) ? (x - (most == -INFINITY ? 0.f : most)) * kLog2e
                                : fmaf(x, kLog2e, -__fmul_rn(most, kLog2e)));
}
// of a single value: NaN of +inf and NaN, a sum of zero of -inf
__device__ __forceinline__ Softmax row_of_one(float x) { return {x, exp_from(x, x)}; }
__device__ __forceinline__ Softmax join_rows(Softmax a, Softmax b) {
  const float m = fmaxf(a.most, b.most);
  return {m, a.sum * exp2_approx(shift_of(a.most, m)) + b.sum * exp2_approx(shift_of(b.most, m))};
}
// of a warp's lanes
__device__ __forceinline__ Softmax row_of_lanes(Softmax s) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(s.most));
  return {m, warp_sum(s.sum * exp2_approx(shift_of(s.most, m)))};
}
// (with the reference of the sum; the difference first, as a product with the lowest value overflows)
__device__ __forceinline__ float log_prob_of(float x, Softmax s) {
  if (s.most == -INFINITY) return NAN;
  return fmaf(rounded_off(s.most), 0.6931471805599453f, x - s.most) - log1pf(s.sum - 1.f);
}

// What the gradient of a row needs: by * onehot(target) + k * exp(x - most) with k = -by / sum.
struct Slope {
  float most, by, k;
  int target;  // -1: outside of the vocabulary
};

// 16 bytes of logits.
template <typename T>
struct Unpack;
template <>
struct Unpack<float> {
  __device__ static void floats(uint4 u, float* v) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  }
  __device__ static uint4 nothing() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  // The largest value so far, in a form of the type's own.
  using Most = float;
  __device__ static Most least() { return -INFINITY; }
  __device__ static void raise(Most& m, uint4 u) {
    m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)),
                       fmaxf(__uint_as_float(u.z), __uint_as_float(u.w))));
  }
  __device__ static float most(Most m) { return m; }
};
template <>
struct Unpack<__nv_bfloat16> {
  __device__ static void floats(uint4 x, float* v) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 nothing() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  __device__ static __nv_bfloat162 as2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
  using Most = __nv_bfloat162;
  __device__ static Most least() { return as2(0xff80ff80u); }
  __device__ static void raise(Most& m, uint4 x) {
    m = __hmax2(m, __hmax2(__hmax2(as2(x.x), as2(x.y)), __hmax2(as2(x.z), as2(x.w))));
  }
  __device__ static float most(Most m) { return fmaxf(__low2float(m), __high2float(m)); }
};

template <int kBytes>
__device__ __forceinline__ void fetch(uint32_t to, const void* from) {
  if (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void fetched() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A thread's share of a chunk of a row, of which `packs` times 16 bytes at p are there: a warp has kWarpPacks of
// them side by side, a thread every 32nd of those. So all warps but one have them all or none, and need not ask
// for each.
constexpr int kWarpPacks = 32 * kPacks;

template <typename T>
struct Share {
  static constexpr int kN = Pack<T>::kN;
  uint4 x[kPacks];

  // visit(i, offset) for those of the thread's that are there; `offset` counts 16 bytes from the chunk's first.
  template <typename Visit>
  __device__ __forceinline__ static void each(int packs, int tid, Visit visit) {
    const int first = (tid >> 5) * kWarpPacks, at = first + (tid & 31);
    if (first + kWarpPacks <= packs) {
#pragma unroll
      for (int i = 0; i < kPacks; ++i) visit(i, at + i * 32);
    } else if (first < packs) {
#pragma unroll
      for (int i = 0; i < kPacks; ++i)
        if (at + i * 32 < packs) visit(i, at + i * 32);
    }
  }
  // On its way to the thread's own places in shared memory, which no other thread reads or writes.
  __device__ __forceinline__ static void ask(uint4* slots, const T* p, int packs, int tid) {
    const uint32_t to = smem_u32(slots);
    each(packs, tid, [&](int, int k) { fetch<16>(to + k * 16, reinterpret_cast<const uint4*>(p) + k); });
  }
  __device__ __forceinline__ void get(const uint4* from, int packs, int tid) {
    if (((tid >> 5) + 1) * kWarpPacks > packs) {
#pragma unroll
      for (int i = 0; i < kPacks; ++i) x[i] = Unpack<T>::nothing();
    }
    each(packs, tid, [&](int i, int k) { x[i] = from[k]; });
  }
  // From where it lies.
  __device__ __forceinline__ void load(const T* p, int packs, int tid) {
    get(reinterpret_cast<const uint4*>(p), packs, tid);
  }
  // All that the thread has asked for is there.
  __device__ __forceinline__ void take(const uint4* slots, int packs, int tid) {
    fetched();
    get(slots, packs, tid);
  }
  // Value number `at` of the chunk, by its thread.
  __device__ __forceinline__ float value(int at) const {
    const uint4 u = pick(at / kN / 32 % kPacks);
    const uint32_t w = (at % kN) * sizeof(T) / 4 == 0   ? u.x
                       : (at % kN) * sizeof(T) / 4 == 1 ? u.y
                       : (at % kN) * sizeof(T) / 4 == 2 ? u.z
                                                        : u.w;
    if (sizeof(T) == 4) return __uint_as_float(w);
    return __uint_as_float(at & 1 ? w & 0xffff0000u : w << 16);
  }
  // Whether it is this thread's.
  __device__ __forceinline__ static bool holds(int at, int packs, int tid) {
    return at >= 0 && at < packs * kN && at / (kN * kWarpPacks) == tid >> 5 && at / kN % 32 == (tid & 31);
  }
  __device__ __forceinline__ void add_to(Softmax& s) const {
    typename Unpack<T>::Most most = Unpack<T>::least();
#pragma unroll
    for (int i = 0; i < kPacks; ++i) Unpack<T>::raise(most, x[i]);
    const float m = Unpack<T>::most(most);
    if (m > s.most) {
      s.sum *= exp2_approx(shift_of(s.most, m));
      s.most = m;
    }
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    if (!huge(s.most)) {
      const float off = -__fmul_rn(s.most, kLog2e);
#pragma unroll
      for (int i = 0; i < kPacks; ++i) {
        float v[kN];
        Unpack<T>::floats(x[i], v);
#pragma unroll
        for (int j = 0; j < kN; ++j) t[j % 4] += exp2_approx(fmaf(v[j], kLog2e, off));
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < kPacks; ++i) {
        float v[kN];
        Unpack<T>::floats(pick(i), v);
#pragma unroll
        for (int j = 0; j < kN; ++j) t[j % 4] += exp_from(v[j], s.most);
      }
    }
    s.sum += (t[0] + t[1]) + (t[2] + t[3]);
  }
  // x[i] for an i that the compiler does not know, without the array leaving the registers
  __device__ __forceinline__ uint4 pick(int i) const {
    uint4 v = x[0];
#pragma unroll
    for (int k = 1; k < kPacks; ++k)
      if (k == i) v = x[k];
    return v;
  }
  // Stores the gradient at g; `at`: where the target lies, counted from the chunk's first value.
  __device__ __forceinline__ void turn(T* g, int packs, int at, const Slope& now, int tid) const {
    if (!huge(now.most)) {
      const float off = -__fmul_rn(now.most, kLog2e);
      each(packs, tid, [&](int i, int k) {
        float y[kN];
        Unpack<T>::floats(x[i], y);
#pragma unroll
        for (int j = 0; j < kN; ++j) y[j] = now.k * exp2_approx(fmaf(y[j], kLog2e, off));
        Pack<T>::store(g + k * kN, y);
      });
    } else {
      const int first = (tid >> 5) * kWarpPacks + (tid & 31);
#pragma unroll 1
      for (int i = 0; i < kPacks; ++i)
        if (first + i * 32 < packs) {
          float y[kN];
          Unpack<T>::floats(pick(i), y);
#pragma unroll
          for (int j = 0; j < kN; ++j) y[j] = now.k * exp_from(y[j], now.most);
          Pack<T>::store(g + (first + i * 32) * kN, y);
        }
    }
    if (holds(at, packs, tid)) g[at] = Pack<T>::back(now.k * exp_from(value(at), now.most) + now.by);
  }
};

// Long rows in pieces of a row, a warp each: their softmaxes and the target's logit. Warps at different places
// of their pieces keep the reads going, and none waits for another: 80 us for 64 x 114 x 32128 bf16 logits of
// which 80% count, 4.7 TB/s, and 133 us for 14 x 509 x 32101 fp32, 5.5 TB/s; a CTA a row, as for the gradient
// below, took 109 and 184 us.
struct Pieces {
  Softmax* of_piece;  // of row and piece
  int shift;          // 1 << shift pieces a row
  float* of_target;   // NaN: outside of the vocabulary
  Softmax* of_row;

  // The row's softmax, kept, and its target's log-probability: in 64 bits, as the margin is a difference of two
  // differences of sums of hundreds of them.
  __device__ __forceinline__ double log_prob(long long row) const {
    const Softmax* of = of_piece + (row << shift);
    float most = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < 1 << shift; ++k) most = fmaxf(most, of[k].most);
    double sum = 0.0;
#pragma unroll 4
    for (int k = 0; k < 1 << shift; ++k)
      sum += static_cast<double>(of[k].sum) * exp2_approx(shift_of(of[k].most, most));
    of_row[row] = {most, static_cast<float>(sum)};
    const double x = of_target[row];
    if (most == -INFINITY) return NAN;
    // (with the same reference as the exponentials in the sum)
    const double d = huge(most) ? x - most : (x * kLog2e - __fmul_rn(most, kLog2e)) * 0.69314718055994531;
    return d - log1p(sum - 1.0);
  }
};

constexpr int kPieceThreads = 256, kPieceCtas = 4;  // CTAs of an SM

template <typename T>
__global__ void __launch_bounds__(kPieceThreads, kPieceCtas)
    preference_pieces_kernel(const T* __restrict__ logits, const Rows r, const Pieces p, unsigned* arrived) {
  constexpr int kN = Pack<T>::kN, kChunk = 32 * kPacks;
  const int lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x == 0) *arrived = 0;  // for the launch of the pairs
  const long long warps = static_cast<long long>(gridDim.x) * (kPieceThreads / 32);
  const long long pieces = r.rows << p.shift;
  auto weight_of = [&](long long i) {
    return i < pieces ? (r.weights != nullptr ? r.weights[i >> p.shift] : 1.f) : 0.f;
  };
  long long i = blockIdx.x * static_cast<long long>(kPieceThreads / 32) + (threadIdx.x >> 5);
  float next = weight_of(i);
  for (; i < pieces; i += warps) {
    const float w = next;
    next = weight_of(i + warps);
    if (w == 0.f) continue;
    const long long row = i >> p.shift;
    const int piece = static_cast<int>(i - (row << p.shift)), b = static_cast<int>(row) / r.length;
    const T* x = logits + b * r.stride_b + (static_cast<int>(row) - b * r.length) * r.stride_t;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15) / static_cast<int>(sizeof(T));
    const int head = off ? kN - off : 0, all = (r.vocab - head) / kN;
    const int size = (all + (1 << p.shift) - 1) >> p.shift, from = min(size * piece, all);
    const int packs = min(all - from, size);
    Softmax s = {-INFINITY, 0.f};
    if (piece == 0) {
      // the values in front of the first 16-byte boundary and behind the last
      const int outside = lane < head ? lane : all * kN + lane;
      if (outside < r.vocab) {
        s = row_of_one(Pack<T>::one(x[outside]));
      }
      if (lane == 0) {
        const long long target = r.targets[row];
        p.of_target[row] = target >= 0 && target < r.vocab ? Pack<T>::one(x[target]) : NAN;
      }
    }
    Share<T> mine;
    for (int at = 0; at < packs; at += kChunk) {
      mine.load(x + head + (from + at) * kN, packs - at, lane);
      mine.add_to(s);
    }
    __syncwarp();
    s = row_of_lanes(s);
    if (lane == 0) p.of_piece[i] = s;
  }
}

// A CTA per pair: scores, margin, the pair's loss, the slopes of its two sequences (and, from
// log-probabilities, of its tokens). The last CTA adds the losses. out: loss, pairs
__global__ void __launch_bounds__(kRowThreads)
    preference_pairs_kernel(const float* __restrict__ logp, const Pieces pieces, const Rows r, const Preference p,
                            float* scores, float* margins, float* __restrict__ by, float* __restrict__ token_slope,
                            double* pair_loss, unsigned* arrived, float* out) {
  const long long pair = blockIdx.x;
  const float scale = scale_of(p.normalizer, p.scale);
  double sum[3] = {0.0, 0.0, 0.0};  // of either answer, and whether any token counts
  const long long first = 2 * pair * r.length;
  const unsigned length = r.length;  // (at most 2^30)
  for (unsigned t = threadIdx.x; t < 2 * length; t += kRowThreads) {
    const float w = r.weights != nullptr ? r.weights[first + t] : 1.f;
    if (w == 0.f) continue;
    const double v = w * (logp != nullptr ? static_cast<double>(logp[first + t]) : pieces.log_prob(first + t));
    if (t < length)
      sum[0] += v;
    else
      sum[1] += v;
    sum[2] = 1.0;
  }
  cta_sums<kRowThreads>(sum);
  const bool real = sum[2] > 0.0;
  const Margin m = pair_margin(p, real, sum[0], sum[1], p.ref[2 * pair], p.ref[2 * pair + 1], scale);
  const float slope = m.slope;
  if (threadIdx.x == 0) {
    scores[2 * pair] = static_cast<float>(sum[0]);
    scores[2 * pair + 1] = static_cast<float>(sum[1]);
    margins[pair] = static_cast<float>(m.margin);
    if (by != nullptr) {
      by[2 * pair] = slope;
      by[2 * pair + 1] = -slope;
    }
    pair_loss[2 * pair] = m.loss;
    pair_loss[2 * pair + 1] = real ? 1.0 : 0.0;
  }
  if (token_slope != nullptr) {
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const long long first = (2 * pair + side) * r.length;
      for (int t = threadIdx.x; t < r.length; t += kRowThreads) {
        const float w = r.weights != nullptr ? r.weights[first + t] : 1.f;
        token_slope[first + t] = w == 0.f ? 0.f : (side ? -slope : slope) * w;
      }
    }
  }
  if (!last_cta(arrived)) return;
  const double whole = p.normalizer != nullptr ? 1.0 / static_cast<double>(*p.normalizer) : p.scale;
  double all[2] = {0.0, 0.0};
  for (int k = threadIdx.x; k < static_cast<int>(gridDim.x); k += kRowThreads) {
    all[0] += __ldcg(pair_loss + 2 * k);
    all[1] += __ldcg(pair_loss + 2 * k + 1);
  }
  cta_sums<kRowThreads>(all);
  if (threadIdx.x == 0) {
    out[0] = static_cast<float>(all[0] * whole);
    out[1] = static_cast<float>(all[1]);
  }
}

enum Mode : int { kPolicy, kTurn };  // all of the policy loss; the gradients of a preference loss

struct LongArgs {
  int shift, chunks;  // 1 << shift CTAs share a row; chunks of a CTA's part
  Policy policy;
  double* partial;
  unsigned* arrived;
  float* out;
  const Softmax* softmax;  // of the rows
  const float* by;         // of the sequences
};

// What there is to know of a row.
struct alignas(16) RowFacts {
  const void* x;     // its first value
  void* g;           // its gradient's
  int first, packs;  // the CTA's part: its first value, its number of 16 bytes
  long long target;
  float weight;
  // policy: old score, reference score, advantage; gradients: softmax, slope of the sequence
  alignas(16) float more[4];
};

template <typename T, int kThreads, int kMode>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
    long_rows_kernel(const T* __restrict__ logits, T* __restrict__ grad, const Rows r, const LongArgs a) {
  constexpr int kN = Pack<T>::kN, kWarps = kThreads / 32, kChunk = kThreads * kPacks;
  extern __shared__ uint4 slots[];  // a chunk
  __shared__ RowFacts facts[4];
  __shared__ Softmax part[kWarps], of_cta[2][8];
  __shared__ float of_target[2];
  __shared__ Slope said;
  using Chunk = Share<T>;
  static_assert(offsetof(RowFacts, target) % 8 == 0 && offsetof(RowFacts, more) % 16 == 0, "places of cp.async");
  static_assert(alignof(Softmax) == 8, "a store of both values");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = 1 << a.shift, rank = a.shift ? static_cast<int>(cluster_ctarank()) : 0;
  const int cluster = blockIdx.x >> a.shift, clusters = gridDim.x >> a.shift, rows = static_cast<int>(r.rows);
  const float scale = kMode == kPolicy ? scale_of(a.policy.normalizer, a.policy.scale) : 0.f;
  double sums[4] = {0.0, 0.0, 0.0, 0.0};

  // The cluster's rows are number cluster, cluster + clusters, ... The gradients begin with the rows read last,
  // which are still in L2. The facts of row k + 3 are asked for when row k has been taken, are there when row
  // k + 1 is, and are read, behind a barrier, when row k + 3 is asked for.
  const bool clerk = tid == kThreads - 32;
  const int mine_of_all = (rows - cluster + clusters - 1) / clusters;
  int ahead = cluster, described = 0;
  int b = (kMode == kTurn ? rows - 1 - ahead : ahead) / r.length;
  int t = (kMode == kTurn ? rows - 1 - ahead : ahead) - b * r.length;
  const int step_b = clusters / r.length, step_t = clusters - step_b * r.length;
  auto describe = [&] {  // (the clerk's)
    RowFacts& f = facts[described++ & 3];
    const int row = kMode == kTurn ? rows - 1 - ahead : ahead;
    if (ahead >= rows) {
      f.weight = 0.f;
      return;
    }
    const T* x = logits + (b * r.stride_b + t * r.stride_t);
    // the row's part between 16-byte boundaries, and of that this CTA's
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15) / static_cast<int>(sizeof(T));
    const int head = off ? kN - off : 0, all = (r.vocab - head) / kN;
    const int size = (all + ctas - 1) >> a.shift, from = min(size * rank, all);
    f.x = x;
    f.g = grad + (b * r.grad_b + t * r.grad_t);
    f.first = head + from * kN;
    f.packs = min(all - from, size);
    fetch<8>(smem_u32(&f.target), r.targets + row);
    if (r.weights != nullptr)
      fetch<4>(smem_u32(&f.weight), r.weights + row);
    else
      f.weight = 1.f;
    if (kMode == kTurn) {
      fetch<8>(smem_u32(f.more), a.softmax + row);
      fetch<4>(smem_u32(f.more + 2), a.by + b);
      b -= step_b, t -= step_t;
      if (t < 0) t += r.length, --b;
    } else {
      fetch<4>(smem_u32(f.more), a.policy.old + row);
      if (a.policy.ref != nullptr) fetch<4>(smem_u32(f.more + 1), a.policy.ref + row);
      fetch<4>(smem_u32(f.more + 2), a.policy.advantages + b * a.policy.adv_b + t * a.policy.adv_t);
      b += step_b, t += step_t;
      if (t >= r.length) t -= r.length, ++b;
    }
    ahead += clusters;
  };
  if (clerk) {
    describe(), describe(), describe();
    fetched();
  }
  __syncthreads();
  if (a.shift) cluster_sync_all();  // all CTAs have begun before any writes to another
  auto ask_row = [&](const RowFacts& f) {
    if (f.weight != 0.f) Chunk::ask(slots, static_cast<const T*>(f.x) + f.first, min(f.packs, kChunk), tid);
  };
  ask_row(facts[0]);
  int turn = 0;
  for (int k = 0; k < mine_of_all; ++k) {
    const RowFacts& f = facts[k & 3];
    const float w = f.weight;
    const int first = f.first, packs = f.packs;
    const T* x = static_cast<const T*>(f.x);
    T* g = static_cast<T*>(f.g);
    // The value in front of the first 16-byte boundary or behind the last that the thread sees to, or -1.
    int outside = -1;
    if (warp == 0 && rank == 0) {
      const int rest = first + (r.vocab - first) / kN * kN;
      outside = tid < first ? tid : (tid - first < r.vocab - rest ? rest + tid - first : -1);
    }
    if (w == 0.f) {
      fetched();  // (the clerk's)
      ask_row(facts[(k + 1) & 3]);
      if (clerk) describe();
      if (grad != nullptr) {
        for (int i = tid; i < packs; i += kThreads)
          *reinterpret_cast<uint4*>(g + first + i * kN) = make_uint4(0, 0, 0, 0);
        if (outside >= 0) g[outside] = Pack<T>::back(0.f);
      }
      __syncthreads();
      continue;
    }
    const int target = f.target >= 0 && f.target < r.vocab ? static_cast<int>(f.target) : -1;
    float x_outside = 0.f;
    if (outside >= 0) x_outside = Pack<T>::one(x[outside]);
    // The target's logit, by the thread that holds it, for all of the cluster. (Two places in turn here and with
    // the parts' softmaxes: a CTA may be at the next row that counts already, but not at the one behind that, as it
    // has to meet the others in between. At rows that do not count CTAs do not meet: those do not change places.)
    auto tell_target = [&](float v) {
      if (a.shift == 0) {
        of_target[turn] = v;
        return;
      }
      for (int c = 0; c < ctas; ++c)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(&of_target[turn]), c)), "f"(v)
                     : "memory");
    };
    auto ask = [&](int c) {
      Chunk::ask(slots, x + first + c * kChunk * kN, min(packs - c * kChunk, kChunk), tid);
    };
    Chunk mine;
    Slope now;
    if (kMode == kTurn) {
      const float by = w * f.more[2];
      now = {f.more[0], by, -by / f.more[1], target};
      for (int c = 0; c < a.chunks; ++c) {
        const int left = min(packs - c * kChunk, kChunk), at = first + c * kChunk * kN;
        mine.take(slots, left, tid);
        if (c + 1 < a.chunks) {
          ask(c + 1);
        } else {
          ask_row(facts[(k + 1) & 3]);
          if (clerk) describe();
          __syncthreads();
        }
        mine.turn(g + at, left, now.target - at, now, tid);
      }
    } else {
      Softmax s = {-INFINITY, 0.f};
      for (int c = 0; c < a.chunks; ++c) {
        const int left = min(packs - c * kChunk, kChunk);
        mine.take(slots, left, tid);
        const int at = target - (first + c * kChunk * kN);
        if (Chunk::holds(at, left, tid)) tell_target(mine.value(at));
        if (c + 1 < a.chunks)
          ask(c + 1);
        else if (grad != nullptr && c > 0)
          ask(c - 1);
        else
          ask_row(facts[(k + 1) & 3]);
        if (clerk && c == 0) describe();
        if (warp * kWarpPacks < left) mine.add_to(s);
      }
      if (outside >= 0) {
        s = join_rows(s, row_of_one(x_outside));
        if (outside == target) tell_target(x_outside);
      }
      __syncwarp();
      s = row_of_lanes(s);
      if (lane == 0) part[warp] = s;
      __syncthreads();
      if (warp == 0) {
        s = row_of_lanes(lane < kWarps ? part[lane] : Softmax{-INFINITY, 0.f});
        if (a.shift && lane < ctas)
          asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(
                           mapa_shared(smem_u32(&of_cta[turn][rank]), lane)),
                       "f"(s.most), "f"(s.sum)
                       : "memory");
        __syncwarp();
      }
      if (a.shift) {
        cluster_sync_all();
        if (warp == 0) s = row_of_lanes(lane < ctas ? of_cta[turn][lane] : Softmax{-INFINITY, 0.f});
      }
      PolicyToken token = {};
      if (tid == 0) {
        const float logp = log_prob_of(target >= 0 ? of_target[turn] : NAN, s);
        token = policy_token(a.policy, {f.more[0], f.more[1], f.more[2]}, logp);
        const float by = w * token.slope * scale;
        said = {s.most, by, -by / s.sum, target};
      }
      __syncthreads();  // (`part` is read, `said` is there; nobody writes it before all are past the next row's first)
      if (tid == 0) {
        sums[0] += static_cast<double>(w) * token.loss;
        sums[1] += static_cast<double>(w) * token.kl;
        sums[2] += static_cast<double>(w) * token.clipped;
        sums[3] += w;
      }
      turn ^= 1;
      if (grad == nullptr) continue;
      now = said;
#pragma unroll 1
      for (int c = a.chunks - 1; c >= 0; --c) {  // (the last is still held)
        const int left = min(packs - c * kChunk, kChunk), at = first + c * kChunk * kN;
        if (c + 1 < a.chunks) {
          mine.take(slots, left, tid);
          if (c > 0)
            ask(c - 1);
          else
            ask_row(facts[(k + 1) & 3]);
        }
        mine.turn(g + at, left, now.target - at, now, tid);
      }
    }
    if (outside >= 0) {
      const float v = now.k * exp_from(x_outside, now.most);
      g[outside] = Pack<T>::back(outside == now.target ? v + now.by : v);
    }
  }
  __syncwarp();
  if (a.shift) cluster_sync_all();  // no CTA ends while another may still write to it
  if (kMode != kPolicy) return;
  // Every cluster's sums, and behind the last cluster's those of all.
  if (warp != 0 || rank != 0) return;
  unsigned before = 0;
  if (lane == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) a.partial[cluster * 4 + k] = sums[k];
    __threadfence();
    before = atomicAdd(a.arrived, 1u) + 1;
  }
  if (__shfl_sync(0xffffffffu, before, 0) != clusters) return;
  __threadfence();
  const double whole =
      a.policy.normalizer != nullptr ? 1.0 / static_cast<double>(*a.policy.normalizer) : a.policy.scale;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    double v = 0.0;
    for (int c = lane; c < clusters; c += 32) v += __ldcg(a.partial + c * 4 + k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) a.out[k] = static_cast<float>(k < 2 ? v * whole : v);
  }
}

// grad *= *factor; nothing where the factor is 1, as it is behind `loss.backward()`. dst may be src.
template <typename T>
__global__ void __launch_bounds__(256)
    scale_kernel(const T* src, T* dst, long long n, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.f && src == dst) return;
  const long long stride = static_cast<long long>(gridDim.x) * 256;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += stride)
    dst[i] = Pack<T>::back(Pack<T>::one(src[i]) * f);
}

// ---- host ----
// Shorter rows are a warp's each. Policy, a warp and a CTA a row, us: 403 and 531 for 262144 rows of 4 KB fp32, 302
// and 300 for 131072 of 6 KB, 425 and 403 of 8 KB, 242 and 221 for 65536 of 8 KB bf16, 333 and 249 of 10 KB fp32.
// Preference, whose three launches do not wait for a row's slope: 542 and 541 for 4 KB, 409 and 398 for 6 KB, 314 and
// 231 for 65536 of 6 KB bf16, 541 and 532 for 131072 of 8 KB fp32; 604 and 1032 for 524288 of 2 KB.
constexpr long long kLongPolicyRow = 6144, kLongRow = 4096;

bool at_multiple(size_t of, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (reinterpret_cast<uintptr_t>(p) % of) return false;
  return true;
}

int check_rows(const char* what, const void* logits, int fp32, const void* grad, long long batch, int length,
               int vocab, long long stride_b, long long stride_t, const void* targets) {
  if (batch < 0 || length < 0 || vocab < 1 || vocab > (1 << 30)) return set_error("%s: bad sizes", what);
  if (batch > 0 && length > 0 && (logits == nullptr || targets == nullptr))
    return set_error("%s: null pointer", what);
  const uintptr_t size = fp32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size || reinterpret_cast<uintptr_t>(grad) % size)
    return set_error("%s: misaligned pointer", what);
  if (grad != nullptr && ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(grad)) & 15))
    return set_error("%s: logits and gradient must lie at the same place of 16 bytes", what);
  if ((length > 1 && stride_t < vocab) || (batch > 1 && stride_b < (length - 1) * stride_t + vocab))
    return set_error("%s: rows overlap", what);
  return 0;
}

// The gradient's strides: rows side by side, but for the few values that put each at its logits' place of 16 bytes.
void gradient_strides(int length, int vocab, int fp32, long long stride_b, long long stride_t, long long* grad_b,
                      long long* grad_t) {
  const long long pack = fp32 ? 4 : 8;
  auto fill = [&](long long like, long long least) { return least + ((like - least) % pack + pack) % pack; };
  *grad_t = fill(stride_t, vocab);
  *grad_b = fill(stride_b, (length - 1) * *grad_t + vocab);
}

unsigned row_grid(long long rows) {
  const long long ctas = (rows + kRowThreads / 32 - 1) / (kRowThreads / 32);
  const long long cap = static_cast<long long>(num_sms()) * 4;
  return static_cast<unsigned>(ctas < 1 ? 1 : (ctas < cap ? ctas : cap));
}

int launched(const char* what, int n) {
  count_launches(n);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error("%s: %s", what, cudaGetErrorString(e));
  return 0;
}

template <typename T, int kThreads, int kMode>
int launch_long(const char* what, const void* logits, void* grad, const Rows& r, LongArgs a, cudaStream_t st) {
  if (r.rows > (1 << 30)) return set_error("%s: too many rows", what);
  auto kernel = long_rows_kernel<T, kThreads, kMode>;
  const long long held = static_cast<long long>(kThreads) * kPacks * 16;  // bytes that a CTA holds
  const long long bytes = static_cast<long long>(r.vocab) * sizeof(T);
  a.shift = 0;
  while (a.shift < 3 && held << a.shift < bytes) ++a.shift;
  const long long packs = ((bytes / 16 - 1) >> a.shift) + 1;  // of a CTA, at most
  a.chunks = static_cast<int>((packs * 16 + held - 1) / held);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1u << a.shift);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = held;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 1u << a.shift;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = a.shift ? 1 : 0;
  // As many clusters as run at once: the rows are dealt out beforehand. (A cluster lies within a group of SMs,
  // whose size need not be a multiple of the cluster's.)
  static std::atomic<int> at_once[64][4];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return set_error("%s: %s", what, cudaGetErrorString(e));
  int cap = at_once[dev][a.shift].load(std::memory_order_relaxed);
  if (cap == 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(held));
    if (e == cudaSuccess && a.shift) e = cudaOccupancyMaxActiveClusters(&cap, kernel, &cfg);
    if (e == cudaSuccess && !a.shift) {
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&cap, kernel, kThreads, held);
      cap *= num_sms();
    }
    if (e != cudaSuccess) return set_error("%s: %s", what, cudaGetErrorString(e));
    if (cap < 1) return set_error("%s: the device has no room for the kernel", what);
    if (cap > kCtasPerSm * num_sms()) cap = kCtasPerSm * num_sms();
    at_once[dev][a.shift].store(cap, std::memory_order_relaxed);
  }
  cfg.gridDim = dim3(static_cast<unsigned>((r.rows < cap ? r.rows : cap) << a.shift));
  e = cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(logits), static_cast<T*>(grad), r, a);
  if (e != cudaSuccess) return set_error("%s: %s", what, cudaGetErrorString(e));
  return launched(what, 1);
}

// The smallest CTA that holds the row, so that short ones leave the SM room for many (512 threads for all of them:
// 1237 in the place of 383 us for 131072 policy rows of 8 KB, 636 and not 403 for 65536 of 16 KB). 64 threads for the
// policy alone: 221 and not 283 us for 65536 rows of 8 KB bf16; gradients alone lose by it, 353 and 360 us for 262144
// rows of 4 KB.
template <typename T, int kMode>
int launch_long(const char* what, const void* logits, void* grad, const Rows& r, const LongArgs& a, cudaStream_t st) {
  const long long bytes = static_cast<long long>(r.vocab) * sizeof(T);
  if constexpr (kMode == kPolicy)
    if (bytes <= 64 * kPacks * 16) return launch_long<T, 64, kMode>(what, logits, grad, r, a, st);
  if (bytes <= 128 * kPacks * 16) return launch_long<T, 128, kMode>(what, logits, grad, r, a, st);
  if (bytes <= 256 * kPacks * 16) return launch_long<T, 256, kMode>(what, logits, grad, r, a, st);
  return launch_long<T, 512, kMode>(what, logits, grad, r, a, st);
}

// Pieces of 24 to 48 KB. (Of 8 KB they are better balanced, but a pair's CTA has more of them to join: 80 and 10 us
// in the place of 82 and 8.5 at 64 KB a row, 145 and 29 in the place of 135 and 9 at 128 KB.)
int piece_shift(long long bytes) {
  int shift = 0;
  while (shift < 4 && bytes >> shift >= 49152) ++shift;
  return shift;
}

template <typename T>
int launch_pieces(const T* logits, const Rows& r, const Pieces& p, unsigned* arrived, cudaStream_t st) {
  if (r.rows > (1 << 30)) return set_error("preference_loss: too many rows");
  const long long ctas = ((r.rows << p.shift) * 32 + kPieceThreads - 1) / kPieceThreads;
  const long long cap = static_cast<long long>(num_sms()) * kPieceCtas;  // as many as run at once
  preference_pieces_kernel<T>
      <<<static_cast<unsigned>(ctas < cap ? ctas : cap), kPieceThreads, 0, st>>>(logits, r, p, arrived);
  return launched("preference_loss", 1);
}

constexpr size_t kHead = 16;  // bytes of scratch in front: the count of arrived CTAs

}  // namespace
}  // namespace t5x

using namespace t5x;

T5X_API void t5x_loss_gradient_strides(int length, int vocab, int fp32, long long stride_b, long long stride_t,
                                       long long* strides) {
  gradient_strides(length, vocab, fp32, stride_b, stride_t, strides, strides + 1);
}

T5X_API long long t5x_policy_loss_scratch_bytes() {
  return static_cast<long long>(kHead) + 4ll * 8 * num_sms() * kCtasPerSm;  // (four sums of each CTA)
}

T5X_API int t5x_policy_loss(const void* logits, int fp32, void* grad, long long batch, int length, int vocab,
                            long long stride_b, long long stride_t, const void* targets, const void* weights,
                            const void* old_scores, const void* ref_scores, const void* advantages,
                            long long adv_b, long long adv_t, float clip_low, float clip_high, float kl_weight,
                            float scale, const void* normalizer, void* scratch, void* out, void* stream) {
  if (check_rows("policy_loss", logits, fp32, grad, batch, length, vocab, stride_b, stride_t, targets)) return -1;
  if (scratch == nullptr || out == nullptr || (batch * length > 0 && (!old_scores || !advantages)))
    return set_error("policy_loss: null pointer");
  if (!at_multiple(16, {scratch}) || !at_multiple(8, {targets}) ||
      !at_multiple(4, {weights, old_scores, ref_scores, advantages, normalizer, out}))
    return set_error("policy_loss: misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead, st);
  if (e != cudaSuccess) return set_error("policy_loss: memset: %s", cudaGetErrorString(e));
  unsigned* arrived = static_cast<unsigned*>(scratch);
  double* partial = reinterpret_cast<double*>(static_cast<char*>(scratch) + kHead);
  Rows r = {batch * length, length, vocab, stride_b, stride_t, 0, 0, static_cast<const long long*>(targets),
            static_cast<const float*>(weights)};
  gradient_strides(length, vocab, fp32, stride_b, stride_t, &r.grad_b, &r.grad_t);
  const Policy p = {static_cast<const float*>(old_scores), static_cast<const float*>(ref_scores),
                    static_cast<const float*>(advantages), adv_b, adv_t, 1.f - clip_low, 1.f + clip_high,
                    kl_weight, scale, static_cast<const float*>(normalizer)};
  float* o = static_cast<float*>(out);
  if (static_cast<long long>(vocab) * (fp32 ? 4 : 2) >= kLongPolicyRow && r.rows > 0) {
    LongArgs a = {};
    a.policy = p;
    a.partial = partial;
    a.arrived = arrived;
    a.out = o;
    return fp32 ? launch_long<float, kPolicy>("policy_loss", logits, grad, r, a, st)
                : launch_long<__nv_bfloat16, kPolicy>("policy_loss", logits, grad, r, a, st);
  }
  const unsigned grid = row_grid(r.rows);
  if (fp32)
    policy_short_rows_kernel<<<grid, kRowThreads, 0, st>>>(static_cast<const float*>(logits),
                                                           static_cast<float*>(grad), r, p, partial, arrived, o);
  else
    policy_short_rows_kernel<<<grid, kRowThreads, 0, st>>>(static_cast<const __nv_bfloat16*>(logits),
                                                           static_cast<__nv_bfloat16*>(grad), r, p, partial, arrived,
                                                           o);
  return launched("policy_loss", 1);
}

T5X_API int t5x_policy_loss_tokens(const void* logp, void* slope, long long batch, int length, const void* weights,
                                   const void* old_scores, const void* ref_scores, const void* advantages,
                                   long long adv_b, long long adv_t, float clip_low, float clip_high,
                                   float kl_weight, float scale, const void* normalizer, void* scratch, void* out,
                                   void* stream) {
  if (batch < 0 || length < 0) return set_error("policy_loss_tokens: bad sizes");
  if (scratch == nullptr || out == nullptr || (batch * length > 0 && (!logp || !old_scores || !advantages)))
    return set_error("policy_loss_tokens: null pointer");
  if (!at_multiple(16, {scratch}) ||
      !at_multiple(4, {logp, slope, weights, old_scores, ref_scores, advantages, normalizer, out}))
    return set_error("policy_loss_tokens: misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead, st);
  if (e != cudaSuccess) return set_error("policy_loss_tokens: memset: %s", cudaGetErrorString(e));
  const Rows r = {batch * length, length, 1, 0, 0, 0, 0, nullptr, static_cast<const float*>(weights)};
  const Policy p = {static_cast<const float*>(old_scores), static_cast<const float*>(ref_scores),
                    static_cast<const float*>(advantages), adv_b, adv_t, 1.f - clip_low, 1.f + clip_high,
                    kl_weight, scale, static_cast<const float*>(normalizer)};
  policy_tokens_kernel<<<row_grid((r.rows + 31) / 32), kRowThreads, 0, st>>>(
      static_cast<const float*>(logp), static_cast<float*>(slope), r, p,
      reinterpret_cast<double*>(static_cast<char*>(scratch) + kHead), static_cast<unsigned*>(scratch),
      static_cast<float*>(out));
  return launched("policy_loss_tokens", 1);
}

T5X_API long long t5x_preference_loss_scratch_bytes(long long batch, int length, int vocab, int fp32) {
  // head | loss and count of each pair | softmax of each token | of its pieces | log-probability or logit of the
  // target | slope of each row
  const long long bytes = static_cast<long long>(vocab) * (fp32 ? 4 : 2);
  const long long pieces = bytes >= kLongRow ? 1 << piece_shift(bytes) : 0;
  return static_cast<long long>(kHead) + batch * 8 + batch * length * (12 + 8 * pieces) + batch * 4;
}

T5X_API int t5x_preference_loss(const void* logits, int fp32, void* grad, long long batch, int length, int vocab,
                                long long stride_b, long long stride_t, const void* targets, const void* weights,
                                const void* reference, float beta, float smoothing, float scale,
                                const void* normalizer, void* scratch, void* scores, void* margins, void* out,
                                void* stream) {
  if (check_rows("preference_loss", logits, fp32, grad, batch, length, vocab, stride_b, stride_t, targets)) return -1;
  if (batch < 2 || batch % 2) return set_error("preference_loss: the batch must hold pairs");
  if (length < 1 || length > (1 << 30)) return set_error("preference_loss: bad sizes");
  if (!scratch || !out || !reference || !scores || !margins) return set_error("preference_loss: null pointer");
  if (!at_multiple(16, {scratch}) || !at_multiple(8, {targets}) ||
      !at_multiple(4, {weights, reference, normalizer, scores, margins, out}))
    return set_error("preference_loss: misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long pairs = batch / 2;
  char* at = static_cast<char*>(scratch);
  Rows r = {batch * length, length, vocab, stride_b, stride_t, 0, 0, static_cast<const long long*>(targets),
            static_cast<const float*>(weights)};
  gradient_strides(length, vocab, fp32, stride_b, stride_t, &r.grad_b, &r.grad_t);
  const Preference p = {static_cast<const float*>(reference), beta, smoothing, scale,
                        static_cast<const float*>(normalizer)};
  unsigned* arrived = reinterpret_cast<unsigned*>(at);
  double* pair_loss = reinterpret_cast<double*>(at + kHead);
  Softmax* softmax = reinterpret_cast<Softmax*>(pair_loss + batch);
  const long long bytes = static_cast<long long>(vocab) * (fp32 ? 4 : 2);
  const bool in_long = bytes >= kLongRow;
  Pieces pieces = {softmax + r.rows, in_long ? piece_shift(bytes) : 0, nullptr, softmax};
  float* logp = reinterpret_cast<float*>(pieces.of_piece + (in_long ? r.rows << pieces.shift : 0));
  pieces.of_target = logp;
  float* by = logp + r.rows;
  auto go = [&](auto* x) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    LongArgs a = {};
    a.softmax = softmax;
    a.by = by;
    const unsigned grid = row_grid(r.rows);
    int rc = 0;
    if (in_long)
      rc = launch_pieces<T>(x, r, pieces, arrived, st);
    else
      preference_short_rows_kernel<T><<<grid, kRowThreads, 0, st>>>(x, r, softmax, logp, arrived);
    if (rc != 0) return rc;
    preference_pairs_kernel<<<static_cast<unsigned>(pairs), kRowThreads, 0, st>>>(
        in_long ? nullptr : logp, pieces, r, p, static_cast<float*>(scores), static_cast<float*>(margins), by, nullptr,
        pair_loss, arrived, static_cast<float*>(out));
    if (grad == nullptr) return launched("preference_loss", in_long ? 1 : 2);
    if (in_long)
      rc = launch_long<T, kTurn>("preference_loss", x, grad, r, a, st);
    else
      preference_short_gradient_kernel<T><<<grid, kRowThreads, 0, st>>>(x, static_cast<T*>(grad), r, softmax, by);
    return rc != 0 ? rc : launched("preference_loss", in_long ? 1 : 3);
  };
  return fp32 ? go(static_cast<const float*>(logits)) : go(static_cast<const __nv_bfloat16*>(logits));
}

T5X_API int t5x_preference_loss_tokens(const void* logp, void* slope, long long batch, int length,
                                       const void* weights, const void* reference, float beta, float smoothing,
                                       float scale, const void* normalizer, void* scratch, void* scores,
                                       void* margins, void* out, void* stream) {
  if (batch < 2 || batch % 2) return set_error("preference_loss_tokens: the batch must hold pairs");
  if (length < 0 || length > (1 << 30)) return set_error("preference_loss_tokens: bad sizes");
  if (!scratch || !out || !reference || !scores || !margins || (length > 0 && !logp))
    return set_error("preference_loss_tokens: null pointer");
  if (!at_multiple(16, {scratch}) ||
      !at_multiple(4, {logp, slope, weights, reference, normalizer, scores, margins, out}))
    return set_error("preference_loss_tokens: misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead, st);
  if (e != cudaSuccess) return set_error("preference_loss_tokens: memset: %s", cudaGetErrorString(e));
  const Rows r = {batch * length, length, 1, 0, 0, 0, 0, nullptr, static_cast<const float*>(weights)};
  const Preference p = {static_cast<const float*>(reference), beta, smoothing, scale,
                        static_cast<const float*>(normalizer)};
  preference_pairs_kernel<<<static_cast<unsigned>(batch / 2), kRowThreads, 0, st>>>(
      static_cast<const float*>(logp), Pieces(), r, p, static_cast<float*>(scores), static_cast<float*>(margins),
      nullptr, static_cast<float*>(slope), reinterpret_cast<double*>(static_cast<char*>(scratch) + kHead),
      static_cast<unsigned*>(scratch), static_cast<float*>(out));
  return launched("preference_loss_tokens", 1);
}

T5X_API int t5x_scale_gradient(const void* src, void* dst, long long n, int fp32, const void* factor, void* stream) {
  if (n <= 0) return 0;
  if (!src || !dst || !factor) return set_error("scale_gradient: null pointer");
  if (!at_multiple(fp32 ? 4 : 2, {src, dst}) || !at_multiple(4, {factor}))
    return set_error("scale_gradient: misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long need = (n + 1023) / 1024, cap = static_cast<long long>(num_sms()) * 8;
  const unsigned grid = static_cast<unsigned>(need < cap ? need : cap);
  if (fp32)
    scale_kernel<float><<<grid, 256, 0, st>>>(static_cast<const float*>(src), static_cast<float*>(dst), n,
                                              static_cast<const float*>(factor));
  else
    scale_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(src),
                                                      static_cast<__nv_bfloat16*>(dst), n,
                                                      static_cast<const float*>(factor));
  return launched("scale_gradient", 1);
}
