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
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "t5x_ops.h"

namespace t5x {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRowThreads = 512;

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

// Largest logit and sum of exp(x - largest).
struct Softmax {
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
  long long stride_b, stride_t;  // in values, of the logits and of their gradient
  const long long* targets;
  const float* weights;  // null: all 1
};
__device__ __forceinline__ long long row_at(const Rows& r, long long row) {
  const long long b = row / r.length;
  return b * r.stride_b + (row - b * r.length) * r.stride_t;
}

// Sum over the threads of the CTA, in every thread, in a fixed order.
template <int kThreads>
__device__ __forceinline__ double cta_sum(double v) {
  __shared__ double part[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) t += part[i];
  return t;
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
__device__ __forceinline__ PolicyToken policy_token(const Policy& p, long long row, long long b, long long t,
                                                    float logp) {
  const float a = p.advantages[b * p.adv_b + t * p.adv_t];
  const float ratio = expf(logp - p.old[row]);
  const float gain = a * ratio, held = a * fminf(fmaxf(ratio, p.low), p.high);
  PolicyToken k;
  k.clipped = held < gain ? 1.f : 0.f;
  // (NaN on either side stays: fminf and the clip would drop it)
  k.loss = -(gain != gain ? gain : fminf(gain, held));
  k.slope = held < gain ? 0.f : -gain;
  k.kl = 0.f;
  if (p.ref != nullptr) {
    const float apart = p.ref[row] - logp, e = expm1f(apart);
    k.kl = e - apart;
    k.loss += p.kl_weight * k.kl;
    k.slope -= p.kl_weight * e;
  }
  return k;
}

// out: loss, kl, clipped, weight
__device__ __forceinline__ void policy_finish(double* sums, const Policy& p, double* partial, unsigned* arrived,
                                              float* out) {
  constexpr int kThreads = kRowThreads;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double v = cta_sum<kThreads>(sums[i]);
    if (threadIdx.x == 0) partial[blockIdx.x * 4 + i] = v;
  }
  if (!last_cta(arrived)) return;
  const double scale = p.normalizer != nullptr ? 1.0 / static_cast<double>(*p.normalizer) : p.scale;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    double v = 0.0;
    for (int k = threadIdx.x; k < static_cast<int>(gridDim.x); k += kThreads) v += __ldcg(partial + k * 4 + i);
    v = cta_sum<kThreads>(v);
    if (threadIdx.x == 0) out[i] = static_cast<float>(i < 2 ? v * scale : v);
  }
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
    const long long at = row_at(r, row);
    if (w == 0.f) {
      if (grad != nullptr) row_zero(grad + at, r.vocab, lane, 32);
      continue;
    }
    const long long target = r.targets[row], b = row / r.length;
    const Softmax s = join_lanes(row_softmax(logits + at, r.vocab, lane, 32));
    const float logp = log_prob(logits + at, r.vocab, target, s);
    const PolicyToken k = policy_token(p, row, b, row - b * r.length, logp);
    if (lane == 0) {
      sums[0] += static_cast<double>(w) * k.loss;
      sums[1] += static_cast<double>(w) * k.kl;
      sums[2] += static_cast<double>(w) * k.clipped;
      sums[3] += w;
    }
    if (grad != nullptr)
      row_gradient(logits + at, grad + at, r.vocab, s,
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
      const PolicyToken k = policy_token(p, row, b, row - b * r.length, logp[row]);
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
                                 float* __restrict__ logp) {
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (kRowThreads / 32);
  for (long long row = blockIdx.x * static_cast<long long>(kRowThreads / 32) + (threadIdx.x >> 5); row < r.rows;
       row += warps) {
    if (r.weights != nullptr && r.weights[row] == 0.f) continue;
    const long long at = row_at(r, row);
    const Softmax s = join_lanes(row_softmax(logits + at, r.vocab, lane, 32));
    if (lane == 0) {
      softmax[row] = s;
      logp[row] = log_prob(logits + at, r.vocab, r.targets[row], s);
    }
  }
}

struct Margin {
  double margin, loss, slope;  // slope: dloss / d(score of the preferred)
};
__device__ __forceinline__ Margin pair_margin(const Preference& p, bool real, double s0, double s1, float r0, float r1,
                                              double scale) {
  Margin m = {0.0, 0.0, 0.0};
  if (!real) return m;
  m.margin = p.beta * ((s0 - r0) - (s1 - r1));
  // log(1 + exp(-d)) = log1p(exp(-|d|)) + max(-d, 0)
  const double e = exp(-fabs(m.margin)), tail = log1p(e);
  const double sigmoid = m.margin >= 0.0 ? 1.0 / (1.0 + e) : e / (1.0 + e);
  m.loss = m.margin != m.margin ? m.margin
                                : (1.0 - p.smoothing) * (tail + fmax(-m.margin, 0.0)) +
                                      p.smoothing * (tail + fmax(m.margin, 0.0));
  m.slope = p.beta * (sigmoid - (1.0 - p.smoothing)) * scale;
  return m;
}

// A CTA per pair: scores, margin, the pair's loss, the slopes of its two sequences (and, from
// log-probabilities, of its tokens). The last CTA adds the losses. out: loss, pairs
__global__ void __launch_bounds__(kRowThreads)
    preference_pairs_kernel(const float* __restrict__ logp, const Rows r, const Preference p, float* scores,
                            float* margins, float* __restrict__ by, float* __restrict__ token_slope,
                            double* pair_loss, unsigned* arrived, float* out) {
  const long long pair = blockIdx.x;
  const float scale = scale_of(p.normalizer, p.scale);
  double sum[2] = {0.0, 0.0}, seen = 0.0;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const long long first = (2 * pair + side) * r.length;
    for (int t = threadIdx.x; t < r.length; t += kRowThreads) {
      const float w = r.weights != nullptr ? r.weights[first + t] : 1.f;
      if (w != 0.f) {
        sum[side] += static_cast<double>(w) * logp[first + t];
        seen = 1.0;
      }
    }
    sum[side] = cta_sum<kRowThreads>(sum[side]);
  }
  const bool real = cta_sum<kRowThreads>(seen) > 0.0;
  const Margin m = pair_margin(p, real, sum[0], sum[1], p.ref[2 * pair], p.ref[2 * pair + 1], scale);
  const double slope = m.slope;
  if (threadIdx.x == 0) {
    scores[2 * pair] = static_cast<float>(sum[0]);
    scores[2 * pair + 1] = static_cast<float>(sum[1]);
    margins[pair] = static_cast<float>(m.margin);
    if (by != nullptr) {
      by[2 * pair] = static_cast<float>(slope);
      by[2 * pair + 1] = static_cast<float>(-slope);
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
        token_slope[first + t] = w == 0.f ? 0.f : static_cast<float>((side ? -slope : slope) * w);
      }
    }
  }
  if (!last_cta(arrived)) return;
  const double whole = p.normalizer != nullptr ? 1.0 / static_cast<double>(*p.normalizer) : p.scale;
  double loss = 0.0, pairs = 0.0;
  for (int k = threadIdx.x; k < static_cast<int>(gridDim.x); k += kRowThreads) {
    loss += __ldcg(pair_loss + 2 * k);
    pairs += __ldcg(pair_loss + 2 * k + 1);
  }
  loss = cta_sum<kRowThreads>(loss);
  pairs = cta_sum<kRowThreads>(pairs);
  if (threadIdx.x == 0) {
    out[0] = static_cast<float>(loss * whole);
    out[1] = static_cast<float>(pairs);
  }
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
    const long long at = row_at(r, row);
    if (w == 0.f) {
      row_zero(grad + at, r.vocab, lane, 32);
      continue;
    }
    const long long target = r.targets[row];
    row_gradient(logits + at, grad + at, r.vocab, softmax[row],
                 target >= 0 && target < r.vocab ? static_cast<int>(target) : -1, w * by[row / r.length], lane, 32);
  }
}

// ---- long rows ----
// A CTA's producer thread copies the rows in tiles of 16 KB into a ring in shared memory, in the order
// in which the worker warps take them, far ahead of them; so the loads go on while a row's sums meet.
// Each tile goes by twice, for the softmax and for the gradient, the second time out of L2. A keeper warp
// makes of the workers' sums what the gradient needs, so that no worker waits for a load of a single
// value, a logarithm or another CTA.
//
// policy: row after row, the gradient of one behind the softmax of the next.
// preference: the slope needs the sums of all rows of a pair. The tasks (a row's softmax, a row's gradient)
// stand in an order in which a group of pairs is followed by the next group's softmaxes and then its own
// gradients; a CTA takes the next task by a ticket. What a gradient waits for has smaller tickets, is
// therefore done or under way, and waits itself for smaller tickets at most.
constexpr int kWorkers = 256;
constexpr int kWorkerWarps = kWorkers / 32;
constexpr int kLongThreads = kWorkers + 64;
constexpr int kTileBytes = 16384;
constexpr int kStages = 6;
constexpr int kSlots = 16;  // rows between their sums and their gradient: at most the ring's tiles and two

enum Kind : int { kEnd, kStat, kGrad, kZero, kSkip };
struct Tile {
  long long row;
  int kind;
  int at, packs;  // first 16 bytes of the row's aligned part, how many
  int last;
};
// What the gradient of a row needs: by * onehot(target) + k * exp(x - most) with k = -by / sum.
struct Slope {
  float most, by, k;
  int target;
};
struct LongShared {
  alignas(128) unsigned char data[kStages][kTileBytes];
  uint64_t full[kStages], empty[kStages], sums[kSlots], said[kSlots];
  Tile tile[kStages];
  Softmax part[kSlots][kWorkerWarps];
  Slope slope[kSlots];
  int abort;
};

// The part of a row between 16-byte boundaries.
template <typename T>
__device__ __forceinline__ void aligned_part(const T* row, int vocab, int& head, int& packs) {
  constexpr int kN = Pack<T>::kN;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T));
  head = off ? kN - off : 0;
  packs = (vocab - head) / kN;
}

struct Order {
  long long rows, group;  // rows of the batch, of a group of pairs
  bool behind;            // a group's gradients follow the next group's softmaxes
  bool gradient;
};
// (row, is it the gradient's turn) of a ticket below rows * (1 + gradient)
__device__ __forceinline__ long long task_of(const Order& o, long long ticket, bool& gradient) {
  gradient = false;
  if (!o.gradient) return ticket;
  const long long last = (o.rows - 1) / o.group * o.group;  // first row of the last group
  if (!o.behind) {  // softmaxes of a group, then its gradients, those last read first
    const long long k = ticket / (2 * o.group), first = k * o.group, at = ticket - 2 * first;
    const long long n = o.rows - first < o.group ? o.rows - first : o.group;
    gradient = at >= n;
    return gradient ? first + 2 * n - 1 - at : first + at;
  }
  gradient = ticket >= o.rows + last;
  if (gradient) return ticket - o.rows;  // of the last group
  if (ticket < o.group) return ticket;
  const long long k = (ticket - o.group) / (2 * o.group) + 1;  // softmaxes of group k, gradients of k - 1
  const long long at = ticket - o.group - (k - 1) * 2 * o.group, first = k * o.group;
  const long long n = o.rows - first < o.group ? o.rows - first : o.group;
  gradient = at >= n;
  return gradient ? first - o.group + (at - n) : first + at;
}

struct Work {
  unsigned long long* ticket;
  unsigned *done, *pairs_done;  // done: rows of the pair whose softmax is there (or that do not count)
  Softmax* softmax;
  float* logp;
  double* pair_loss;
  float *scores, *margins;
  Order order;
};

// Two values at once where the arithmetic has pairs.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void split(uint64_t d, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// In the tiles an exponential exp(x - most) is exp2(x log2 e - ref), a fused product and difference, with
// ref = most log2 e as rounded: the same factor for the sum, the target and the gradient. Where a largest
// logit's product may overflow, it is exp2((x - most) log2 e).
constexpr float kHuge = 1.0e38f;
__device__ __forceinline__ bool huge(float most) { return !(fabsf(most) <= kHuge); }  // (NaN and -inf too)
// log2 of exp(a - b); 0 for a = b = -inf
__device__ __forceinline__ float shift(float a, float b) {
  if (huge(a) || huge(b)) return a == b ? 0.f : (a - b) * kLog2e;
  return __fmul_rn(a, kLog2e) - __fmul_rn(b, kLog2e);
}
__device__ __forceinline__ float exp_from(float x, float most) {
  return exp2_approx(huge(most) ? (x - (most == -INFINITY ? 0.f : most)) * kLog2e
                                : fmaf(x, kLog2e, -__fmul_rn(most, kLog2e)));
}
__device__ __forceinline__ Softmax join_rows(Softmax a, Softmax b) {
  const float m = fmaxf(a.most, b.most);
  return {m, a.sum * exp2_approx(shift(a.most, m)) + b.sum * exp2_approx(shift(b.most, m))};
}
__device__ __forceinline__ Softmax join_row_lanes(Softmax s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    s = join_rows(s, {__shfl_xor_sync(0xffffffffu, s.most, o), __shfl_xor_sync(0xffffffffu, s.sum, o)});
  return s;
}
__device__ __forceinline__ float log_prob_of(float x, Softmax s) {
  if (s.most == -INFINITY) return NAN;
  const float d = huge(s.most) ? x - s.most : fmaf(x, kLog2e, -__fmul_rn(s.most, kLog2e)) * 0.6931471805599453f;
  return d - log1pf(s.sum - 1.f);
}

// 16 bytes of the tile, as pairs
template <typename T>
struct Pairs;
template <>
struct Pairs<float> {
  uint64_t v[2];
  __device__ void load(const void* p) {
    const float4 x = *static_cast<const float4*>(p);
    v[0] = pair_of(x.x, x.y), v[1] = pair_of(x.z, x.w);
  }
  __device__ float most() const {
    float a, b, c, d;
    split(v[0], a, b), split(v[1], c, d);
    return fmaxf(fmaxf(a, b), fmaxf(c, d));
  }
};
template <>
struct Pairs<__nv_bfloat16> {
  uint64_t v[4];
  float top;
  __device__ void load(const void* p) {
    const uint4 x = *static_cast<const uint4*>(p);
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pair_of(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    const __nv_bfloat162 m = __hmax2(__hmax2(as2(u[0]), as2(u[1])), __hmax2(as2(u[2]), as2(u[3])));
    top = fmaxf(__low2float(m), __high2float(m));
  }
  __device__ static __nv_bfloat162 as2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
  __device__ float most() const { return top; }
};

// Adds a thread's 16 bytes each to the softmax of what it has seen.
template <typename T, int kPacks>
__device__ __forceinline__ void take(Softmax& s, const Pairs<T>* x) {
  constexpr int kPairsOf = sizeof(Pairs<T>::v) / 8;
  float m = x[0].most();
#pragma unroll
  for (int i = 1; i < kPacks; ++i) m = fmaxf(m, x[i].most());
  if (m > s.most) {
    s.sum *= exp2_approx(shift(s.most, m));
    s.most = m;
  }
  uint64_t t = pair_of(0.f, 0.f);
  if (!huge(s.most)) {
    const float ref = __fmul_rn(s.most, kLog2e);
    const uint64_t l2e = pair_of(kLog2e, kLog2e), off = pair_of(-ref, -ref);
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
#pragma unroll
      for (int j = 0; j < kPairsOf; ++j) {
        float a, b;
        split(fma2(x[i].v[j], l2e, off), a, b);
        t = add2(t, pair_of(exp2_approx(a), exp2_approx(b)));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPacks; ++i) {
#pragma unroll
      for (int j = 0; j < kPairsOf; ++j) {
        float a, b;
        split(x[i].v[j], a, b);
        t = add2(t, pair_of(exp_from(a, s.most), exp_from(b, s.most)));
      }
    }
  }
  float a, b;
  split(t, a, b);
  s.sum += a + b;
}

template <typename T, bool kPairs>
__global__ void __launch_bounds__(kLongThreads, 2)
    long_rows_kernel(const T* __restrict__ logits, T* __restrict__ grad, const Rows r, const Policy p,
                     const Preference q, const Work work, double* partial, unsigned* arrived, float* out,
                     int* status) {
  constexpr int kN = Pack<T>::kN;
  constexpr int kTilePacks = kTileBytes / 16;
  extern __shared__ __align__(128) unsigned char raw[];
  LongShared& sh = *reinterpret_cast<LongShared*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], kWorkerWarps + 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sh.sums[i], kWorkerWarps);
      mbar_init(&sh.said[i], 1);
    }
    sh.abort = 0;
    mbar_fence_init();
  }
  __syncthreads();
  volatile int* abort = &sh.abort;
  int stage = 0;
  uint32_t round = 0;
  bool ok = true;
  auto advance = [&] {
    if (++stage == kStages) stage = 0, ++round;
  };
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // the whole warp's
    ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
    return ok;
  };
  auto give_up = [&](int code) {
    if (lane == 0) {
      *abort = 1;
      report_status(status, code, 41, warp);
    }
  };

  if (warp == kWorkerWarps) {  // ---- producer ----
    int issued = 0;
    auto push = [&](const Tile& t, const void* src) {  // (one thread's)
      if (!ok || !mbar_wait(&sh.empty[stage], (round & 1) ^ 1, abort)) {
        ok = false;
        return;
      }
      sh.tile[stage] = t;
      if (src != nullptr) {
        mbar_expect_tx(&sh.full[stage], t.packs * 16);
        bulk_load(sh.data[stage], src, t.packs * 16, &sh.full[stage]);
      } else {
        mbar_arrive(&sh.full[stage]);
      }
      ++issued;
      advance();
    };
    auto stream = [&](int kind, long long row) {
      const T* x = logits + row_at(r, row);
      int head, packs;
      aligned_part(x, r.vocab, head, packs);
      for (int at = 0; at < packs && ok; at += kTilePacks) {
        const int n = packs - at < kTilePacks ? packs - at : kTilePacks;
        push({row, kind, at, n, at + n == packs}, x + head + static_cast<long long>(at) * kN);
      }
    };
    if (kPairs) {
      if (lane == 0) {
        const unsigned long long total = work.order.rows * (work.order.gradient ? 2 : 1);
        auto weight = [&](unsigned long long t) {
          bool g;
          return t < total && r.weights != nullptr ? r.weights[task_of(work.order, t, g)] : 1.f;
        };
        unsigned long long ticket = atomicAdd(work.ticket, 1ull);
        float w = weight(ticket);
        while (ok && ticket < total) {
          const unsigned long long next = atomicAdd(work.ticket, 1ull);  // (one ahead: the answer takes its time)
          bool gradient;
          const long long row = task_of(work.order, ticket, gradient);
          if (w == 0.f)
            push({row, gradient ? kZero : kSkip, 0, 0, 1}, nullptr);
          else
            stream(gradient ? kGrad : kStat, row);
          ticket = next;
          w = weight(ticket);
        }
      }
    } else {
      long long before = -1;  // the row whose gradient is still to come
      for (long long base = blockIdx.x; base < r.rows; base += 32ll * gridDim.x) {
        const long long mine = base + static_cast<long long>(lane) * gridDim.x;
        const float w = mine < r.rows && r.weights != nullptr ? r.weights[mine] : 1.f;
        const unsigned visible = __ballot_sync(0xffffffffu, w != 0.f);
        if (lane == 0) {
          for (int i = 0; i < 32; ++i) {
            const long long row = base + static_cast<long long>(i) * gridDim.x;
            if (row >= r.rows || !ok) break;
            if (visible >> i & 1) {
              stream(kStat, row);
              if (grad != nullptr && before >= 0) stream(kGrad, before);
              before = row;
            } else if (grad != nullptr) {
              push({row, kZero, 0, 0, 1}, nullptr);
            }
          }
        }
        __syncwarp();
      }
      if (lane == 0 && grad != nullptr && before >= 0) stream(kGrad, before);
    }
    if (lane == 0) {
      push({0, kEnd, 0, 0, 1}, nullptr);
      if (!ok) {  // no copy may be under way when the shared memory is given back
        give_up(kStatusTimeoutProducer);
        const int n = issued < kStages ? issued : kStages;
        for (int i = issued - n; i < issued; ++i)
          for (uint32_t it = 0; it < kWaitLimit && !mbar_try_wait(&sh.full[i % kStages], (i / kStages) & 1); ++it) {
          }
      }
    }
    return;
  }

  unsigned rows_summed = 0, rows_turned = 0;  // softmaxes and gradients so far
  if (warp > kWorkerWarps) {  // ---- keeper ----
    const float scale = kPairs ? 0.f : scale_of(p.normalizer, p.scale);
    double sums[4] = {0.0, 0.0, 0.0, 0.0};
    float w = 0.f, x = 0.f;  // weight and target's logit of the row under way
    long long target = -1, known = -1;
    float slope0 = 0.f;  // of the preferred row of the known pair
    while (wait(&sh.full[stage], round & 1)) {
      const Tile t = sh.tile[stage];
      if (t.kind == kEnd) break;
      const long long b = t.row / r.length;
      if (t.kind == kStat) {
        if (t.at == 0 && lane == 0) {  // (asked for while the row is summed)
          const T* row = logits + row_at(r, t.row);
          target = r.targets[t.row];
          w = r.weights != nullptr ? r.weights[t.row] : 1.f;
          x = target >= 0 && target < r.vocab ? Pack<T>::one(row[target]) : NAN;
        }
        if (t.last) {
          const int slot = rows_summed % kSlots;
          if (!wait(&sh.sums[slot], rows_summed / kSlots & 1)) break;
          const Softmax s = join_row_lanes(lane < kWorkerWarps ? sh.part[slot][lane] : Softmax{-INFINITY, 0.f});
          if (lane == 0) {
            const float logp = log_prob_of(x, s);
            if (kPairs) {
              work.softmax[t.row] = s;
              work.logp[t.row] = logp;
              red_release_gpu_add(work.done + b / 2, 1u);
            } else {
              const PolicyToken c = policy_token(p, t.row, b, t.row - b * r.length, logp);
              sums[0] += static_cast<double>(w) * c.loss;
              sums[1] += static_cast<double>(w) * c.kl;
              sums[2] += static_cast<double>(w) * c.clipped;
              sums[3] += w;
              const float by = w * c.slope * scale;
              sh.slope[slot] = {s.most, by, -by / s.sum,
                                target >= 0 && target < r.vocab ? static_cast<int>(target) : -1};
              mbar_arrive(&sh.said[slot]);
            }
          }
          ++rows_summed;
        }
      } else if (kPairs && t.at == 0) {
        const long long pair = b / 2;
        if (t.kind == kSkip) {
          if (lane == 0) red_release_gpu_add(work.done + pair, 1u);
        } else {
          const bool turned = t.kind == kGrad;
          const bool writes = t.row == pair * 2 * r.length;  // one row of a pair writes what the pair gives
          if (pair != known && (turned || writes)) {
            uint32_t it = 0;
            while (ld_acquire_gpu(work.done + pair) != 2u * r.length) {
              if (++it == kWaitLimit || *abort) {
                ok = false;
                break;
              }
              __nanosleep(20);
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            double sum[2] = {0.0, 0.0};
            bool seen = false;
#pragma unroll
            for (int side = 0; side < 2; ++side) {
              const long long first = (2 * pair + side) * r.length;
#pragma unroll 4
              for (int i = lane; i < r.length; i += 32) {
                const float wt = r.weights != nullptr ? r.weights[first + i] : 1.f;
                const float lp = __ldcg(work.logp + first + i);
                if (wt != 0.f) {
                  sum[side] += static_cast<double>(wt) * lp;
                  seen = true;
                }
              }
#pragma unroll
              for (int o = 16; o > 0; o >>= 1) sum[side] += __shfl_xor_sync(0xffffffffu, sum[side], o);
            }
            const bool real = __any_sync(0xffffffffu, seen);
            const Margin m = pair_margin(q, real, sum[0], sum[1], q.ref[2 * pair], q.ref[2 * pair + 1],
                                         scale_of(q.normalizer, q.scale));
            slope0 = static_cast<float>(m.slope);
            known = pair;
            if (writes) {
              unsigned before = 0;
              if (lane == 0) {
                work.scores[2 * pair] = static_cast<float>(sum[0]);
                work.scores[2 * pair + 1] = static_cast<float>(sum[1]);
                work.margins[pair] = static_cast<float>(m.margin);
                work.pair_loss[2 * pair] = m.loss;
                work.pair_loss[2 * pair + 1] = real ? 1.0 : 0.0;
                __threadfence();
                before = atomicAdd(work.pairs_done, 1u);
              }
              const long long pairs = r.rows / r.length / 2;
              if (__shfl_sync(0xffffffffu, before, 0) == pairs - 1) {
                __threadfence();
                double loss = 0.0, count = 0.0;
                for (long long i = lane; i < pairs; i += 32) {
                  loss += __ldcg(work.pair_loss + 2 * i);
                  count += __ldcg(work.pair_loss + 2 * i + 1);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                  loss += __shfl_xor_sync(0xffffffffu, loss, o);
                  count += __shfl_xor_sync(0xffffffffu, count, o);
                }
                if (lane == 0) {
                  const double whole = q.normalizer != nullptr ? 1.0 / static_cast<double>(*q.normalizer) : q.scale;
                  out[0] = static_cast<float>(loss * whole);
                  out[1] = static_cast<float>(count);
                }
              }
            }
          }
          if (turned) {
            if (lane == 0) {
              const long long at = r.targets[t.row];
              const float wt = r.weights != nullptr ? r.weights[t.row] : 1.f;
              const float most = __ldcg(&work.softmax[t.row].most), sum = __ldcg(&work.softmax[t.row].sum);
              const float by = wt * (b & 1 ? -slope0 : slope0);
              const int slot = rows_turned % kSlots;
              sh.slope[slot] = {most, by, -by / sum, at >= 0 && at < r.vocab ? static_cast<int>(at) : -1};
              mbar_arrive(&sh.said[slot]);
            }
            ++rows_turned;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[stage]);
      advance();
    }
    if (!ok) {
      give_up(kStatusTimeoutEpilogue);
      return;
    }
    if (kPairs) return;
    unsigned before = 0;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) partial[blockIdx.x * 4 + i] = sums[i];
      __threadfence();
      before = atomicAdd(arrived, 1u);
    }
    if (__shfl_sync(0xffffffffu, before, 0) != gridDim.x - 1) return;
    __threadfence();
    const double whole = p.normalizer != nullptr ? 1.0 / static_cast<double>(*p.normalizer) : p.scale;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      double v = 0.0;
      for (unsigned c = lane; c < gridDim.x; c += 32) v += __ldcg(partial + c * 4 + i);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) out[i] = static_cast<float>(i < 2 ? v * whole : v);
    }
    return;
  }

  // ---- workers ----
  Softmax seen = {-INFINITY, 0.f};       // of the row whose softmax is under way
  Slope now = {0.f, 0.f, 0.f, -1};       // of the row whose gradient is under way
  while (wait(&sh.full[stage], round & 1)) {
    const Tile t = sh.tile[stage];
    if (t.kind == kEnd) break;
    const unsigned char* data = sh.data[stage];
    const T* row = logits + row_at(r, t.row);
    int head = 0, outside = -1;  // the value outside of the aligned part that this thread sees to
    if (t.kind == kStat || t.kind == kGrad) {
      int packs;
      aligned_part(row, r.vocab, head, packs);
      if (t.at == 0) {
        const int i = tid < head ? tid : packs * kN + tid;  // (head + packs * kN + tid - head)
        if (i < r.vocab && (tid < head || tid < r.vocab - packs * kN)) outside = i;
      }
    }
    if (t.kind == kStat) {
      if (outside >= 0) {
        const float v = Pack<T>::one(row[outside]);
        seen = {v, v == -INFINITY ? 0.f : v * 0.f + 1.f};  // (NaN of +inf and NaN)
      }
      if (t.packs == kTilePacks) {
        constexpr int kMine = kTilePacks / kWorkers;
        Pairs<T> x[kMine];
#pragma unroll
        for (int i = 0; i < kMine; ++i) x[i].load(data + (tid + i * kWorkers) * 16);
        take<T, kMine>(seen, x);
      } else {
        for (int i = tid; i < t.packs; i += kWorkers) {
          Pairs<T> x[1];
          x[0].load(data + i * 16);
          take<T, 1>(seen, x);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[stage]);
      if (t.last) {
        const Softmax s = join_row_lanes(seen);
        if (lane == 0) {
          const int slot = rows_summed % kSlots;
          sh.part[slot][warp] = s;
          mbar_arrive(&sh.sums[slot]);
        }
        ++rows_summed;
        seen = {-INFINITY, 0.f};
      }
    } else if (t.kind == kGrad) {
      T* g = grad + row_at(r, t.row);
      if (t.at == 0) {
        const int slot = rows_turned % kSlots;
        if (!wait(&sh.said[slot], rows_turned / kSlots & 1)) break;
        now = sh.slope[slot];
        ++rows_turned;
        if (outside >= 0) {
          const float v = now.k * exp_from(Pack<T>::one(row[outside]), now.most);
          g[outside] = Pack<T>::back(outside == now.target ? v + now.by : v);
        }
      }
      const int first = head + t.at * kN;
      const float ref = __fmul_rn(now.most, kLog2e);
      const bool far = huge(now.most);
      const uint64_t l2e = pair_of(kLog2e, kLog2e), off = pair_of(-ref, -ref), k2 = pair_of(now.k, now.k);
      auto one = [&](int i) {
        Pairs<T> v;
        v.load(data + i * 16);
        float x[kN];
#pragma unroll
        for (int j = 0; j < kN / 2; ++j) {
          float a, b;
          if (far) {
            split(v.v[j], a, b);
            a = exp_from(a, now.most), b = exp_from(b, now.most);
          } else {
            split(fma2(v.v[j], l2e, off), a, b);
            a = exp2_approx(a), b = exp2_approx(b);
          }
          split(mul2(pair_of(a, b), k2), x[2 * j], x[2 * j + 1]);
        }
        const int at = first + i * kN;
        if (static_cast<unsigned>(now.target - at) < static_cast<unsigned>(kN)) {
#pragma unroll
          for (int j = 0; j < kN; ++j)
            if (now.target == at + j) x[j] += now.by;
        }
        Pack<T>::store(g + at, x);
      };
      if (t.packs == kTilePacks) {
#pragma unroll
        for (int i = 0; i < kTilePacks / kWorkers; ++i) one(tid + i * kWorkers);
      } else {
        for (int i = tid; i < t.packs; i += kWorkers) one(i);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[stage]);
    } else {
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[stage]);
      if (t.kind == kZero) row_zero(grad + row_at(r, t.row), r.vocab, tid, kWorkers);
    }
    advance();
  }
  if (!ok) give_up(kStatusTimeoutEpilogue);
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
constexpr long long kShortRow = 4096;  // bytes; shorter rows are a warp's

int check_rows(const char* what, const void* logits, int fp32, const void* grad, long long batch, int length,
               int vocab, long long stride_b, long long stride_t, const void* targets) {
  if (batch < 0 || length < 0 || vocab < 1) return set_error("%s: bad sizes", what);
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

unsigned long_grid(long long rows) {
  const long long cap = static_cast<long long>(num_sms()) * 2;
  return static_cast<unsigned>(rows < 1 ? 1 : (rows < cap ? rows : cap));
}

template <typename T, bool kPairs>
int launch_long(const char* what, const void* logits, void* grad, const Rows& r, const Policy& p, const Preference& q,
                const Work& work, double* partial, unsigned* arrived, float* out, cudaStream_t st) {
  auto kernel = long_rows_kernel<T, kPairs>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(LongShared));
  if (e != cudaSuccess) return set_error("%s: %s", what, cudaGetErrorString(e));
  kernel<<<long_grid(r.rows), kLongThreads, sizeof(LongShared), st>>>(
      static_cast<const T*>(logits), static_cast<T*>(grad), r, p, q, work, partial, arrived, out,
      device_status_buffer());
  return launched(what, 1);
}

// The order of the tasks of a preference loss: a pair of up to kBehindBytes of logits stands in a group of
// up to kGroupBytes, whose gradients follow the next group's softmaxes; a larger pair's gradients follow
// its own softmaxes, beginning with the rows read last.
constexpr long long kGroupBytes = 16 << 20, kBehindBytes = 24 << 20;

constexpr size_t kHead = 16;  // bytes of scratch in front: the ticket, the count of arrived CTAs or pairs done

}  // namespace
}  // namespace t5x

using namespace t5x;

T5X_API long long t5x_policy_loss_scratch_bytes() {
  return static_cast<long long>(kHead) + 4ll * 8 * num_sms() * 4;
}

T5X_API int t5x_policy_loss(const void* logits, int fp32, void* grad, long long batch, int length, int vocab,
                            long long stride_b, long long stride_t, const void* targets, const void* weights,
                            const void* old_scores, const void* ref_scores, const void* advantages,
                            long long adv_b, long long adv_t, float clip_low, float clip_high, float kl_weight,
                            float scale, const void* normalizer, void* scratch, void* out, void* stream) {
  if (check_rows("policy_loss", logits, fp32, grad, batch, length, vocab, stride_b, stride_t, targets)) return -1;
  if (scratch == nullptr || out == nullptr || (batch * length > 0 && (!old_scores || !advantages)))
    return set_error("policy_loss: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead, st);
  if (e != cudaSuccess) return set_error("policy_loss: memset: %s", cudaGetErrorString(e));
  unsigned* arrived = static_cast<unsigned*>(scratch);
  double* partial = reinterpret_cast<double*>(static_cast<char*>(scratch) + kHead);
  const Rows r = {batch * length, length, vocab, stride_b, stride_t, static_cast<const long long*>(targets),
                  static_cast<const float*>(weights)};
  const Policy p = {static_cast<const float*>(old_scores), static_cast<const float*>(ref_scores),
                    static_cast<const float*>(advantages), adv_b, adv_t, 1.f - clip_low, 1.f + clip_high,
                    kl_weight, scale, static_cast<const float*>(normalizer)};
  float* o = static_cast<float*>(out);
  if (static_cast<long long>(vocab) * (fp32 ? 4 : 2) >= kShortRow)
    return fp32 ? launch_long<float, false>("policy_loss", logits, grad, r, p, {}, {}, partial, arrived, o, st)
                : launch_long<__nv_bfloat16, false>("policy_loss", logits, grad, r, p, {}, {}, partial, arrived, o, st);
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead, st);
  if (e != cudaSuccess) return set_error("policy_loss_tokens: memset: %s", cudaGetErrorString(e));
  const Rows r = {batch * length, length, 1, 0, 0, nullptr, static_cast<const float*>(weights)};
  const Policy p = {static_cast<const float*>(old_scores), static_cast<const float*>(ref_scores),
                    static_cast<const float*>(advantages), adv_b, adv_t, 1.f - clip_low, 1.f + clip_high,
                    kl_weight, scale, static_cast<const float*>(normalizer)};
  policy_tokens_kernel<<<row_grid((r.rows + 31) / 32), kRowThreads, 0, st>>>(
      static_cast<const float*>(logp), static_cast<float*>(slope), r, p,
      reinterpret_cast<double*>(static_cast<char*>(scratch) + kHead), static_cast<unsigned*>(scratch),
      static_cast<float*>(out));
  return launched("policy_loss_tokens", 1);
}

T5X_API long long t5x_preference_loss_scratch_bytes(long long batch, int length) {
  // head | counts and flags of the pairs | loss and count of each pair | largest and sum of each token |
  // log-probability | slope of each row
  return static_cast<long long>(kHead) + batch / 2 * 8 + batch * 8 + batch * length * 12 + batch * 4;
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long pairs = batch / 2;
  char* at = static_cast<char*>(scratch);
  const Rows r = {batch * length, length, vocab, stride_b, stride_t, static_cast<const long long*>(targets),
                  static_cast<const float*>(weights)};
  const Preference p = {static_cast<const float*>(reference), beta, smoothing, scale,
                        static_cast<const float*>(normalizer)};
  Work w;
  w.ticket = reinterpret_cast<unsigned long long*>(at);
  w.pairs_done = reinterpret_cast<unsigned*>(at + 8);
  w.done = reinterpret_cast<unsigned*>(at + kHead);
  w.pair_loss = reinterpret_cast<double*>(at + kHead + pairs * 8);
  w.softmax = reinterpret_cast<Softmax*>(w.pair_loss + batch);
  w.logp = reinterpret_cast<float*>(w.softmax + r.rows);
  float* by = w.logp + r.rows;
  w.scores = static_cast<float*>(scores);
  w.margins = static_cast<float*>(margins);
  float* o = static_cast<float*>(out);
  const long long row_bytes = static_cast<long long>(vocab) * (fp32 ? 4 : 2);
  const bool in_long = row_bytes >= kShortRow;
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead + (in_long ? pairs * 8 : 0), st);
  if (e != cudaSuccess) return set_error("preference_loss: memset: %s", cudaGetErrorString(e));
  if (in_long) {
    const long long pair_bytes = 2 * length * row_bytes;
    const long long group = kGroupBytes / pair_bytes > 1 ? kGroupBytes / pair_bytes : 1;
    w.order = {r.rows, (group < pairs ? group : pairs) * 2 * length, pair_bytes <= kBehindBytes, grad != nullptr};
    if (fp32 ? launch_long<float, true>("preference_loss", logits, grad, r, {}, p, w, nullptr, nullptr, o, st)
             : launch_long<__nv_bfloat16, true>("preference_loss", logits, grad, r, {}, p, w, nullptr, nullptr, o, st))
      return -1;
    if (grad != nullptr) return 0;
    preference_pairs_kernel<<<static_cast<unsigned>(pairs), kRowThreads, 0, st>>>(
        w.logp, r, p, w.scores, w.margins, nullptr, nullptr, w.pair_loss, w.pairs_done, o);
    return launched("preference_loss", 1);
  }
  const unsigned grid = row_grid(r.rows);
  auto go = [&](auto* x) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    preference_short_rows_kernel<T><<<grid, kRowThreads, 0, st>>>(x, r, w.softmax, w.logp);
    preference_pairs_kernel<<<static_cast<unsigned>(pairs), kRowThreads, 0, st>>>(
        w.logp, r, p, w.scores, w.margins, by, nullptr, w.pair_loss, w.pairs_done, o);
    if (grad != nullptr)
      preference_short_gradient_kernel<T><<<grid, kRowThreads, 0, st>>>(x, static_cast<T*>(grad), r, w.softmax, by);
  };
  if (fp32)
    go(static_cast<const float*>(logits));
  else
    go(static_cast<const __nv_bfloat16*>(logits));
  return launched("preference_loss", 2 + (grad != nullptr));
}

T5X_API int t5x_preference_loss_tokens(const void* logp, void* slope, long long batch, int length,
                                       const void* weights, const void* reference, float beta, float smoothing,
                                       float scale, const void* normalizer, void* scratch, void* scores,
                                       void* margins, void* out, void* stream) {
  if (batch < 2 || batch % 2 || length < 0) return set_error("preference_loss_tokens: the batch must hold pairs");
  if (!scratch || !out || !reference || !scores || !margins || (length > 0 && !logp))
    return set_error("preference_loss_tokens: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead, st);
  if (e != cudaSuccess) return set_error("preference_loss_tokens: memset: %s", cudaGetErrorString(e));
  const Rows r = {batch * length, length, 1, 0, 0, nullptr, static_cast<const float*>(weights)};
  const Preference p = {static_cast<const float*>(reference), beta, smoothing, scale,
                        static_cast<const float*>(normalizer)};
  preference_pairs_kernel<<<static_cast<unsigned>(batch / 2), kRowThreads, 0, st>>>(
      static_cast<const float*>(logp), r, p, static_cast<float*>(scores), static_cast<float*>(margins), nullptr,
      static_cast<float*>(slope), reinterpret_cast<double*>(static_cast<char*>(scratch) + kHead),
      static_cast<unsigned*>(scratch), static_cast<float*>(out));
  return launched("preference_loss_tokens", 1);
}

T5X_API int t5x_scale_gradient(const void* src, void* dst, long long n, int fp32, const void* factor, void* stream) {
  if (n <= 0) return 0;
  if (!src || !dst || !factor) return set_error("scale_gradient: null pointer");
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
