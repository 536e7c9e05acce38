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
    const PolicyInputs in = policy_inputs(p, row, b, row - b * r.length);
    const Softmax s = join_lanes(row_softmax(logits + at, r.vocab, lane, 32));
    const float logp = log_prob(logits + at, r.vocab, target, s);
    const PolicyToken k = policy_token(p, in, logp);
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
  m.loss = d != d ? d : (1.f - p.smoothing) * (tail + fmaxf(-d, 0.f)) + p.smoothing * (tail + fmaxf(d, 0.f));
  // sigmoid - 1 + e, near 0 from the side that does not cancel
  const float under = (d >= 0.f ? e : 1.f) / (1.f + e);  // sigmoid(-d)
  m.slope = p.beta * (p.smoothing * sigmoid - (1.f - p.smoothing) * under) * scale;
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
// What both kernels share. A CTA's producer thread copies rows in tiles of up to 8 KB into a ring in
// shared memory, far ahead of the worker warps. A tile is one warp's, the next tile the next warp's: the
// warps of an SM are at different places of their work, so that some load or wait while others keep the
// units for the exponentials busy (with a tile for all warps they stood in step: 375M logits summed in
// 283 us instead of XXX). A keeper warp makes of the warps' sums what the gradient of the row needs, so that no
// worker waits for the load of a single value, a logarithm or another CTA; the producer hands it a row's few
// values, which it has asked for rows ahead.
constexpr int kTileBytes = 8192;
constexpr int kTilePacks = kTileBytes / 16;

enum Kind : int { kEnd, kStat, kGrad, kZero };
// What the gradient of a row needs: by * onehot(target) + k * exp(x - most) with k = -by / sum.
struct Slope {
  float most, by, k;
  int target;
};
struct Tile {
  long long offset;  // of the row in the logits and their gradient
  int kind;
  int last;          // the warp's last tile of the row
  int head;          // values in front of the row's first 16-byte boundary
  int at, packs;     // first 16 bytes behind it, how many
  int outside;       // 16 bytes of the whole row, on the tile whose warp sees to the values outside; else -1
  unsigned task;     // the how-many-th of the CTA's rows that are summed
  Slope now;         // of a kGrad tile
};
struct Task {
  long long row, b;
  int kind, target;  // target: -1 outside of the vocabulary
  float w, x;        // weight, the target's logit
  int warp;          // whose is the row's first tile
  PolicyInputs in;
};
// Slots for rows between their sums and their gradient: more than the ring has tiles, so that none is written
// again before the warps that read it have given their tiles back.
template <int kStages_, int kWarps_, int kSlots_>
struct LongShared {
  static constexpr int kStages = kStages_, kWarps = kWarps_, kSlots = kSlots_;
  alignas(128) unsigned char data[kStages][kTileBytes];
  uint64_t full[kStages], empty[kStages], told[kSlots], kept[kSlots], sums[kSlots], said[kSlots], met[kSlots];
  Tile tile[kStages];
  Task task[kSlots];
  Softmax part[kSlots][kWarps];
  Softmax of_cta[kSlots][8];  // of the CTAs that share the row
  Slope slope[kSlots];
  int abort;
  __device__ void init(int warps_of_row) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&told[i], 1);
      mbar_init(&kept[i], 1);
      mbar_init(&sums[i], warps_of_row);
      mbar_init(&said[i], 1);
      mbar_init(&met[i], 1);
    }
    abort = 0;
    mbar_fence_init();
  }
  // The sums of a row's warps, in every lane of the keeper.
  __device__ Softmax all_parts(int slot, int first, int warps_of_row) const;
};

// A wait with a limit of a second or two (a poll may be held back for some ten microseconds).
constexpr uint32_t kPolls = 1u << 17;
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  for (uint32_t it = 0; it < kPolls; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 0xf) == 0xf && *abort) return false;
  }
  return false;
}

// The part of a row between 16-byte boundaries.
template <typename T>
__device__ __forceinline__ void aligned_part(const T* row, int vocab, int& head, int& packs) {
  constexpr int kN = Pack<T>::kN;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T));
  head = off ? kN - off : 0;
  packs = (vocab - head) / kN;
}

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
__device__ __forceinline__ uint64_t same2(float a) { return pair_of(a, a); }

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

// 16 bytes of a tile, as pairs
template <typename T>
struct Pairs;
template <>
struct Pairs<float> {
  static constexpr int kPairs = 2;
  uint64_t v[2];
  __device__ void load(const void* p) {
    const float4 x = *static_cast<const float4*>(p);
    v[0] = pair_of(x.x, x.y), v[1] = pair_of(x.z, x.w);
  }
  __device__ void nothing() { v[0] = v[1] = same2(-INFINITY); }
  __device__ float most() const {
    float a, b, c, d;
    split(v[0], a, b), split(v[1], c, d);
    return fmaxf(fmaxf(a, b), fmaxf(c, d));
  }
};
template <>
struct Pairs<__nv_bfloat16> {
  static constexpr int kPairs = 4;
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
  __device__ void nothing() {
    v[0] = v[1] = v[2] = v[3] = same2(-INFINITY);
    top = -INFINITY;
  }
  __device__ static __nv_bfloat162 as2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
  __device__ float most() const { return top; }
};

// exp2 of the two values
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
  float a, b;
  split(x, a, b);
  return pair_of(exp2_approx(a), exp2_approx(b));
}

template <int kStages, int kWarps, int kSlots>
__device__ Softmax LongShared<kStages, kWarps, kSlots>::all_parts(int slot, int first, int warps_of_row) const {
  const int lane = threadIdx.x & 31;
  return join_row_lanes(lane < warps_of_row ? part[slot][(first + lane) % kWarps] : Softmax{-INFINITY, 0.f});
}

// Adds a lane's 16 bytes each to what it has seen.
template <typename T, int kMine>
__device__ __forceinline__ void take(Softmax& s, const Pairs<T>* x) {
  constexpr int kP = Pairs<T>::kPairs;
  float m = x[0].most();
#pragma unroll
  for (int i = 1; i < kMine; ++i) m = fmaxf(m, x[i].most());
  if (m > s.most) {
    s.sum *= exp2_approx(shift(s.most, m));
    s.most = m;
  }
  uint64_t t[2] = {same2(0.f), same2(0.f)};
  if (!huge(s.most)) {
    const float ref = __fmul_rn(s.most, kLog2e);
    const uint64_t l2e = same2(kLog2e), off = same2(-ref);
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
      for (int j = 0; j < kP; ++j) t[j & 1] = add2(t[j & 1], exp2_pair(fma2(x[i].v[j], l2e, off)));
  } else {
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
      for (int j = 0; j < kP; ++j) {
        float a, b;
        split(x[i].v[j], a, b);
        t[0] = add2(t[0], pair_of(exp_from(a, s.most), exp_from(b, s.most)));
      }
  }
  float a, b;
  split(add2(t[0], t[1]), a, b);
  s.sum += a + b;
}

// The tile's part of the row's softmax; a warp's.
template <typename T>
__device__ __forceinline__ void sum_tile(Softmax& s, const unsigned char* data, int packs, int lane) {
  constexpr int kMine = 4;
  Pairs<T> x[kMine];
  int at = 0;
#pragma unroll 1
  for (; at + kMine * 32 <= packs; at += kMine * 32) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) x[i].load(data + (at + i * 32 + lane) * 16);
    take<T, kMine>(s, x);
  }
  if (at < packs) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      if (at + i * 32 + lane < packs)
        x[i].load(data + (at + i * 32 + lane) * 16);
      else
        x[i].nothing();
    }
    take<T, kMine>(s, x);
  }
}

// The tile's part of the gradient; a warp's. g: the row's.
template <typename T>
__device__ __forceinline__ void turn_tile(T* g, const unsigned char* data, const Tile& t, const Slope& now, int lane) {
  constexpr int kN = Pack<T>::kN;
  const int first = t.head + t.at * kN;
  const bool far = huge(now.most);
  const float ref = __fmul_rn(now.most, kLog2e);
  const uint64_t l2e = same2(kLog2e), off = same2(-ref), k2 = same2(now.k);
  auto one = [&](int i, auto plain) {
    Pairs<T> v;
    v.load(data + i * 16);
    float x[kN];
#pragma unroll
    for (int j = 0; j < kN / 2; ++j) {
      uint64_t e;
      if (plain || !far) {
        e = exp2_pair(fma2(v.v[j], l2e, off));
      } else {
        float a, b;
        split(v.v[j], a, b);
        e = pair_of(exp_from(a, now.most), exp_from(b, now.most));
      }
      split(mul2(e, k2), x[2 * j], x[2 * j + 1]);
    }
    const int at = first + i * kN;
    if (!plain && static_cast<unsigned>(now.target - at) < static_cast<unsigned>(kN)) {
#pragma unroll
      for (int j = 0; j < kN; ++j)
        if (now.target == at + j) x[j] += now.by;
    }
    Pack<T>::store(g + at, x);
  };
  // a tile without the target, of a row whose exponentials take the short way
  if (!far && static_cast<unsigned>(now.target - first) >= static_cast<unsigned>(t.packs * kN)) {
#pragma unroll 4
    for (int i = lane; i < t.packs; i += 32) one(i, std::true_type());
  } else {
#pragma unroll 1
    for (int i = lane; i < t.packs; i += 32) one(i, std::false_type());
  }
}

// The value outside of the row's 16-byte boundaries that a thread sees to, or -1.
template <typename T>
__device__ __forceinline__ int outside_of(const Tile& t, int vocab, int tid) {
  if (t.outside < 0) return -1;
  const int behind = t.outside * Pack<T>::kN;  // head + ... - head
  return tid < t.head ? tid : (tid < vocab - behind ? behind + tid : -1);
}
template <typename T>
__device__ __forceinline__ Softmax one_value(T v) {
  const float x = Pack<T>::one(v);
  return {x, x == -INFINITY ? 0.f : x * 0.f + 1.f};  // (NaN of +inf and NaN)
}
template <typename T>
__device__ __forceinline__ void turn_one(T* g, const T* row, int i, const Slope& now) {
  const float v = now.k * exp_from(Pack<T>::one(row[i]), now.most);
  g[i] = Pack<T>::back(i == now.target ? v + now.by : v);
}

// The producer's side of a ring; one thread's.
template <typename Shared>
struct Ring {
  static constexpr int kStages = Shared::kStages, kSlots = Shared::kSlots;
  Shared& sh;
  volatile int* abort;
  int stage = 0, warp = 0, issued = 0;  // warp: whose the next tile is
  uint32_t round = 0;
  unsigned tasks = 0;
  bool ok = true;
  __device__ Ring(Shared& s) : sh(s), abort(&s.abort) {}
  __device__ void push(const Tile& t, const void* src) {
    if (!ok || !ring_wait(&sh.empty[stage], (round & 1) ^ 1, abort)) {
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
    if (++warp == Shared::kWarps) warp = 0;
    if (++stage == kStages) stage = 0, ++round;
  }
  // The keeper, of a row ahead of its tiles.
  __device__ void tell(Task t) {
    const int slot = tasks % kSlots;
    if (!ok || !ring_wait(&sh.kept[slot], (tasks / kSlots & 1) ^ 1, abort)) {
      ok = false;
      return;
    }
    t.warp = warp;
    sh.task[slot] = t;
    mbar_arrive(&sh.told[slot]);
    ++tasks;
  }
  // `packs` 16 bytes of a row from `from`, in `tiles` tiles of one size.
  template <typename T>
  __device__ void stream(Tile t, const T* logits, int from, int packs, int tiles) {
    const int size = (packs + tiles - 1) / tiles;
    for (int i = 0; i < tiles && ok; ++i) {
      t.at = from + i * size;
      t.packs = packs - i * size < size ? packs - i * size : size;
      t.last = i + Shared::kWarps >= tiles;
      push(t, logits + t.offset + t.head + static_cast<long long>(t.at) * Pack<T>::kN);
      t.outside = -1;
    }
  }
  __device__ void end() {
    Task t = {};
    t.kind = kEnd;
    tell(t);
    for (int i = 0; i < Shared::kWarps; ++i) push({0, kEnd, 1, 0, 0, 0, -1, 0, {}}, nullptr);
  }
  // No copy may be under way when the shared memory is given back.
  __device__ void drain() {
    const int n = issued < kStages ? issued : kStages;
    for (int i = issued - n; i < issued; ++i)
      for (uint32_t it = 0; it < kPolls && !mbar_try_wait(&sh.full[i % kStages], (i / kStages) & 1); ++it) {
      }
  }
};

// A worker warp's side: its tiles are every kWarps-th of the ring.
template <typename Shared>
struct Turn {
  int stage;
  uint32_t round;
  __device__ void advance() {
    stage += Shared::kWarps;
    while (stage >= Shared::kStages) stage -= Shared::kStages, ++round;
  }
};

// Policy. A row belongs to a cluster of CTAs, of which each takes a part that fits into its ring with room for
// the next ones: the part is read once, summed, and turned into the gradient where it lies. The parts' sums
// meet through distributed shared memory. A warp turns a tile behind the sums of its next one, so that it does
// not wait for the row's slope. (Tile t is turned behind the sums of its row, which end n - 1 tiles later at
// most, and of tile t + kWarps; tile u is loaded when tile u - kStages is turned: with n and kWarps no more than
// kStages the turning waits for smaller tiles only.)
using PolicyShared = LongShared<26, 16, 32>;
constexpr int kPolicyThreads = PolicyShared::kWarps * 32 + 64;

__device__ __forceinline__ void send_to_cta(Softmax* slot, uint64_t* bar, int cta, Softmax s) {
  uint64_t v;
  memcpy(&v, &s, 8);
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(
                   mapa_shared(smem_u32(slot), cta)),
               "l"(v), "r"(mapa_shared(smem_u32(bar), cta))
               : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kPolicyThreads, 1)
    policy_rows_kernel(const T* __restrict__ logits, T* __restrict__ grad, const Rows r, const Policy p, int ctas,
                       int tiles, double* partial, unsigned* arrived, float* out, int* status) {
  constexpr int kN = Pack<T>::kN, kWarps = PolicyShared::kWarps, kSlots = PolicyShared::kSlots;
  extern __shared__ __align__(128) unsigned char raw[];
  PolicyShared& sh = *reinterpret_cast<PolicyShared*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ctas > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const long long cluster = blockIdx.x / ctas, clusters = gridDim.x / ctas;
  const int warps_of_row = tiles < kWarps ? tiles : kWarps;
  if (tid == 0) sh.init(warps_of_row);
  __syncthreads();
  if (ctas > 1) cluster_sync_all();  // every CTA's barriers stand before another signals one
  volatile int* abort = &sh.abort;
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // the whole warp's
    ok = __all_sync(0xffffffffu, ring_wait(bar, parity, abort));
    return ok;
  };
  auto give_up = [&](int code) {
    if (lane == 0) {
      *abort = 1;
      report_status(status, code, 41, warp);
    }
  };

  if (warp == kWarps) {  // ---- producer: 32 rows' values at a time, asked for while the last 32 go by ----
    Ring<PolicyShared> ring(sh);
    Task next = {};
    long long next_offset = 0;
    auto ask = [&](long long base) {
      next.row = base + lane * clusters;
      next.kind = kEnd;
      if (next.row >= r.rows) return;
      next.b = next.row / r.length;
      const long long t = next.row - next.b * r.length;
      next_offset = next.b * r.stride_b + t * r.stride_t;
      next.w = r.weights != nullptr ? r.weights[next.row] : 1.f;
      next.kind = next.w != 0.f ? kStat : kZero;
      if (next.kind == kZero) return;
      const long long target = r.targets[next.row];
      next.target = target >= 0 && target < r.vocab ? static_cast<int>(target) : -1;
      next.in = policy_inputs(p, next.row, next.b, t);
      next.x = next.target >= 0 ? Pack<T>::one(logits[next_offset + next.target]) : NAN;
    };
    ask(cluster);
    for (long long base = cluster; base < r.rows; base += 32 * clusters) {
      const Task mine = next;
      const long long offset = next_offset;
      if (base + 32 * clusters < r.rows) ask(base + 32 * clusters);
      for (int i = 0; i < 32; ++i) {
        Task t;
        t.row = base + i * clusters;
        if (t.row >= r.rows) break;
        t.b = __shfl_sync(0xffffffffu, mine.b, i);
        t.kind = __shfl_sync(0xffffffffu, mine.kind, i);
        t.target = __shfl_sync(0xffffffffu, mine.target, i);
        t.w = __shfl_sync(0xffffffffu, mine.w, i);
        t.x = __shfl_sync(0xffffffffu, mine.x, i);
        t.in = {__shfl_sync(0xffffffffu, mine.in.old, i), __shfl_sync(0xffffffffu, mine.in.ref, i),
                __shfl_sync(0xffffffffu, mine.in.advantage, i)};
        Tile tile = {__shfl_sync(0xffffffffu, offset, i), t.kind, 1, 0, 0, 0, -1, 0, {}};
        int all;
        aligned_part(logits + tile.offset, r.vocab, tile.head, all);
        const int part = (all + ctas - 1) / ctas, from = part * rank < all ? part * rank : all;
        const int packs = all - from < part ? all - from : part;
        if (t.kind == kZero) {  // (all lanes': nothing of it is in the way of the tiles)
          if (grad == nullptr) continue;
          T* g = grad + tile.offset;
          for (int k = lane; k < packs; k += 32)
            *reinterpret_cast<uint4*>(g + tile.head + static_cast<long long>(from + k) * kN) = make_uint4(0, 0, 0, 0);
          tile.outside = rank == 0 ? all : -1;
          const int k = outside_of<T>(tile, r.vocab, lane);
          if (k >= 0) g[k] = Pack<T>::back(0.f);
          continue;
        }
        if (lane != 0) continue;
        tile.outside = rank == 0 ? all : -1;
        tile.task = ring.tasks;
        ring.tell(t);
        ring.stream(tile, logits, from, packs, tiles);
      }
    }
    if (lane == 0) {
      ring.end();
      if (!ring.ok) {
        give_up(kStatusTimeoutProducer);
        ring.drain();
      }
    }
  } else if (warp > kWarps) {  // ---- keeper ----
    const float scale = scale_of(p.normalizer, p.scale);
    double sums[4] = {0.0, 0.0, 0.0, 0.0};
    for (unsigned n = 0;; ++n) {
      const int slot = n % kSlots;
      const uint32_t parity = n / kSlots & 1;
      if (!wait(&sh.told[slot], parity)) break;
      const Task t = sh.task[slot];
      if (t.kind == kEnd) break;
      if (!wait(&sh.sums[slot], parity)) break;
      Softmax s = sh.all_parts(slot, t.warp, warps_of_row);
      if (ctas > 1) {
        if (lane == 0) mbar_expect_tx(&sh.met[slot], 8 * ctas);
        __syncwarp();
        if (lane < ctas) send_to_cta(&sh.of_cta[slot][rank], &sh.met[slot], lane, s);
        if (!wait(&sh.met[slot], parity)) break;
        s = join_row_lanes(lane < ctas ? sh.of_cta[slot][lane] : Softmax{-INFINITY, 0.f});
      }
      if (lane == 0) {
        const PolicyToken c = policy_token(p, t.in, log_prob_of(t.x, s));
        const float by = t.w * c.slope * scale;
        sh.slope[slot] = {s.most, by, -by / s.sum, t.target};
        mbar_arrive(&sh.said[slot]);
        mbar_arrive(&sh.kept[slot]);
        sums[0] += static_cast<double>(t.w) * c.loss;
        sums[1] += static_cast<double>(t.w) * c.kl;
        sums[2] += static_cast<double>(t.w) * c.clipped;
        sums[3] += t.w;
      }
      __syncwarp();
    }
    if (!ok) give_up(kStatusTimeoutEpilogue);
    unsigned before = 0;
    if (lane == 0 && rank == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) partial[cluster * 4 + i] = ok ? sums[i] : NAN;
      __threadfence();
      before = atomicAdd(arrived, 1u) + 1;
    }
    if (__shfl_sync(0xffffffffu, before, 0) == clusters) {
      __threadfence();
      const double whole = p.normalizer != nullptr ? 1.0 / static_cast<double>(*p.normalizer) : p.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        double v = 0.0;
        for (long long c = lane; c < clusters; c += 32) v += __ldcg(partial + c * 4 + i);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) out[i] = static_cast<float>(i < 2 ? v * whole : v);
      }
    }
  } else {  // ---- workers ----
    Turn<PolicyShared> at = {warp, 0}, old = at;  // old: of the tile whose gradient is still to come
    bool pending = false;
    Softmax seen = {-INFINITY, 0.f};
    auto turn = [&](int stage) {
      const Tile t = sh.tile[stage];
      if (!wait(&sh.said[t.task % kSlots], t.task / kSlots & 1)) return;
      const Slope now = sh.slope[t.task % kSlots];
      const int i = outside_of<T>(t, r.vocab, lane);
      if (i >= 0) turn_one(grad + t.offset, logits + t.offset, i, now);
      turn_tile<T>(grad + t.offset, sh.data[stage], t, now, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[stage]);
    };
    while (wait(&sh.full[at.stage], at.round & 1)) {
      const Tile t = sh.tile[at.stage];
      if (t.kind == kStat) {
        const int i = outside_of<T>(t, r.vocab, lane);
        if (i >= 0) seen = one_value(logits[t.offset + i]);
        sum_tile<T>(seen, sh.data[at.stage], t.packs, lane);
        if (t.last) {
          const Softmax s = join_row_lanes(seen);
          if (lane == 0) {
            sh.part[t.task % kSlots][warp] = s;
            mbar_arrive(&sh.sums[t.task % kSlots]);
          }
          seen = {-INFINITY, 0.f};
        }
        if (grad == nullptr) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.empty[at.stage]);
          at.advance();
          continue;
        }
      }
      if (pending) turn(old.stage);
      pending = t.kind == kStat;
      old = at;
      if (!ok || t.kind == kEnd) break;
      at.advance();
    }
    if (!ok) give_up(kStatusTimeoutEpilogue);
  }
  if (ctas > 1) {
    __syncwarp();
    cluster_sync_all();  // no CTA ends while another may still write to it
  }
}

// Preference. The slope of a row needs the sums of all rows of its pair: one kernel makes the rows' softmaxes
// and log-probabilities, another (above) the pairs' slopes, a third, beginning with the rows read last, which
// are still in L2, the gradients. (One kernel for all of it, whose gradients waited for the rows of their pair,
// would read most logits from L2 the second time, but its CTAs wait for one another.) Two CTAs an SM.
using PairShared = LongShared<12, 8, 16>;
constexpr int kPairThreads = PairShared::kWarps * 32 + 64;

// kTurn: the gradients, from `softmax` and the slopes `by` of the sequences; else the softmaxes.
template <typename T, bool kTurn>
__global__ void __launch_bounds__(kPairThreads, 2)
    preference_rows_kernel(const T* __restrict__ logits, T* __restrict__ grad, const Rows r, int tiles,
                           Softmax* __restrict__ softmax, float* __restrict__ logp, const float* __restrict__ by,
                           int* status) {
  constexpr int kWarps = PairShared::kWarps, kSlots = PairShared::kSlots;
  const int warps_of_row = tiles < kWarps ? tiles : kWarps;
  extern __shared__ __align__(128) unsigned char raw[];
  PairShared& sh = *reinterpret_cast<PairShared*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sh.init(warps_of_row);
  __syncthreads();
  volatile int* abort = &sh.abort;
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {  // the whole warp's
    ok = __all_sync(0xffffffffu, ring_wait(bar, parity, abort));
    return ok;
  };
  auto give_up = [&](int code) {
    if (lane == 0) {
      *abort = 1;
      report_status(status, code, 42, warp);
    }
  };

  if (warp == kWarps) {  // ---- producer: 32 rows' values at a time, asked for while the last 32 go by ----
    Ring<PairShared> ring(sh);
    Task next = {};
    Slope next_slope = {};
    long long next_offset = 0;
    auto ask = [&](long long base) {
      const long long at = base + static_cast<long long>(lane) * gridDim.x;
      next.kind = kEnd;
      if (at >= r.rows) return;
      next.row = kTurn ? r.rows - 1 - at : at;
      next.b = next.row / r.length;
      next_offset = next.b * r.stride_b + (next.row - next.b * r.length) * r.stride_t;
      next.w = r.weights != nullptr ? r.weights[next.row] : 1.f;
      next.kind = next.w != 0.f ? (kTurn ? kGrad : kStat) : kZero;
      if (next.kind == kZero) return;
      const long long target = r.targets[next.row];
      next.target = target >= 0 && target < r.vocab ? static_cast<int>(target) : -1;
      if (kTurn) {
        const Softmax s = softmax[next.row];
        const float slope = next.w * by[next.b];
        next_slope = {s.most, slope, -slope / s.sum, next.target};
      } else {
        next.x = next.target >= 0 ? Pack<T>::one(logits[next_offset + next.target]) : NAN;
      }
    };
    ask(blockIdx.x);
    for (long long base = blockIdx.x; base < r.rows; base += 32ll * gridDim.x) {
      const Task mine = next;
      const Slope slope = next_slope;
      const long long offset = next_offset;
      if (base + 32ll * gridDim.x < r.rows) ask(base + 32ll * gridDim.x);
      for (int i = 0; i < 32; ++i) {
        if (base + static_cast<long long>(i) * gridDim.x >= r.rows) break;
        Task t;
        t.row = __shfl_sync(0xffffffffu, mine.row, i);
        t.b = 0;
        t.kind = __shfl_sync(0xffffffffu, mine.kind, i);
        t.target = 0;
        t.w = 0.f;
        t.x = __shfl_sync(0xffffffffu, mine.x, i);
        t.in = {};
        Tile tile = {__shfl_sync(0xffffffffu, offset, i), t.kind, 1, 0, 0, 0, -1, 0, {}};
        tile.now = {__shfl_sync(0xffffffffu, slope.most, i), __shfl_sync(0xffffffffu, slope.by, i),
                    __shfl_sync(0xffffffffu, slope.k, i), __shfl_sync(0xffffffffu, slope.target, i)};
        int all;
        aligned_part(logits + tile.offset, r.vocab, tile.head, all);
        if (t.kind == kZero) {  // (all lanes')
          if (kTurn) row_zero(grad + tile.offset, r.vocab, lane, 32);
          continue;
        }
        if (lane != 0) continue;
        tile.outside = all;
        tile.task = ring.tasks;
        if (!kTurn) ring.tell(t);
        ring.stream(tile, logits, 0, all, tiles);
      }
    }
    if (lane == 0) {
      ring.end();
      if (!ring.ok) {
        give_up(kStatusTimeoutProducer);
        ring.drain();
      }
    }
  } else if (warp > kWarps) {  // ---- keeper ----
    for (unsigned n = 0;; ++n) {
      const int slot = n % kSlots;
      const uint32_t parity = n / kSlots & 1;
      if (!wait(&sh.told[slot], parity)) break;
      const Task t = sh.task[slot];
      if (t.kind == kEnd) break;
      if (!wait(&sh.sums[slot], parity)) break;
      const Softmax s = sh.all_parts(slot, t.warp, warps_of_row);
      if (lane == 0) {
        softmax[t.row] = s;
        logp[t.row] = log_prob_of(t.x, s);
        mbar_arrive(&sh.kept[slot]);
      }
      __syncwarp();
    }
    if (!ok) give_up(kStatusTimeoutEpilogue);
  } else {  // ---- workers ----
    Turn<PairShared> at = {warp, 0};
    Softmax seen = {-INFINITY, 0.f};
    while (wait(&sh.full[at.stage], at.round & 1)) {
      const Tile t = sh.tile[at.stage];
      if (t.kind == kEnd) break;
      const int outside = outside_of<T>(t, r.vocab, lane);
      if (kTurn) {
        if (outside >= 0) turn_one(grad + t.offset, logits + t.offset, outside, t.now);
        turn_tile<T>(grad + t.offset, sh.data[at.stage], t, t.now, lane);
      } else {
        if (outside >= 0) seen = one_value(logits[t.offset + outside]);
        sum_tile<T>(seen, sh.data[at.stage], t.packs, lane);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[at.stage]);
      at.advance();
      if (!kTurn && t.last) {
        const Softmax s = join_row_lanes(seen);
        if (lane == 0) {
          sh.part[t.task % kSlots][warp] = s;
          mbar_arrive(&sh.sums[t.task % kSlots]);
        }
        seen = {-INFINITY, 0.f};
      }
    }
    if (!ok) give_up(kStatusTimeoutEpilogue);
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
// Rows of these bytes go through the ring; shorter ones are a warp's each, and so are longer ones (a vocabulary
// of 400,000 in 32 bits: more than eight CTAs hold), which no model here has.
constexpr long long kRingRow = 4096, kRingRowMost = 1600 << 10;
bool by_ring(long long vocab, int fp32) {
  const long long bytes = vocab * (fp32 ? 4 : 2);
  return bytes >= kRingRow && bytes <= kRingRowMost;
}

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

// Tiles of a CTA's part of a row, the same for all rows wherever their 16-byte boundaries lie (none is empty:
// a part of n tiles has more than 512 (n - 1) times 16 bytes, or, for n = 1, 250).
int tiles_of(long long vocab, int size, int ctas) {
  const long long packs = (vocab * size / 16 + ctas - 1) / ctas;
  return static_cast<int>((packs + kTilePacks - 1) / kTilePacks);
}

template <typename T>
int launch_policy(const void* logits, void* grad, const Rows& r, const Policy& p, double* partial, unsigned* arrived,
                  float* out, cudaStream_t st) {
  // The smallest cluster whose CTAs' parts leave room for two more in the ring (the largest cluster's parts
  // may be larger).
  const long long bytes = static_cast<long long>(r.vocab) * sizeof(T);
  int ctas = 1;
  while (ctas < 8 && (bytes + ctas - 1) / ctas > 8 * kTileBytes) ctas *= 2;
  if (grad == nullptr) ctas = 1;  // (nothing has to stay)
  const int tiles = tiles_of(r.vocab, sizeof(T), ctas);
  auto kernel = policy_rows_kernel<T>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(PolicyShared));
  if (e != cudaSuccess) return set_error("policy_loss: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kPolicyThreads);
  cfg.dynamicSmemBytes = sizeof(PolicyShared);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  // As many clusters as run at once: the rows are dealt out beforehand. (A cluster lies within a group of SMs,
  // whose size need not be a multiple of the cluster's.)
  static std::atomic<int> at_once[64][4];
  int dev = 0, size = ctas == 1 ? 0 : ctas == 2 ? 1 : ctas == 4 ? 2 : 3;
  cudaGetDevice(&dev);
  int cap = at_once[dev][size].load(std::memory_order_relaxed);
  if (cap == 0) {
    cap = num_sms();
    if (ctas > 1) {
      e = cudaOccupancyMaxActiveClusters(&cap, kernel, &cfg);
      if (e != cudaSuccess) return set_error("policy_loss: %s", cudaGetErrorString(e));
    }
    if (cap < 1) cap = 1;
    at_once[dev][size].store(cap, std::memory_order_relaxed);
  }
  cfg.gridDim = dim3(static_cast<unsigned>((r.rows < cap ? r.rows : cap) * ctas));
  e = cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(logits), static_cast<T*>(grad), r, p, ctas, tiles, partial,
                         arrived, out, device_status_buffer());
  if (e != cudaSuccess) return set_error("policy_loss: %s", cudaGetErrorString(e));
  return launched("policy_loss", 1);
}

template <typename T, bool kTurn>
int launch_preference(const void* logits, void* grad, const Rows& r, Softmax* softmax, float* logp, const float* by,
                      cudaStream_t st) {
  auto kernel = preference_rows_kernel<T, kTurn>;
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(PairShared));
  if (e != cudaSuccess) return set_error("preference_loss: %s", cudaGetErrorString(e));
  const long long cap = static_cast<long long>(num_sms()) * 2;
  kernel<<<static_cast<unsigned>(r.rows < cap ? r.rows : cap), kPairThreads, sizeof(PairShared), st>>>(
      static_cast<const T*>(logits), static_cast<T*>(grad), r, tiles_of(r.vocab, sizeof(T), 1), softmax, logp, by,
      device_status_buffer());
  return launched("preference_loss", 1);
}

constexpr size_t kHead = 16;  // bytes of scratch in front: the count of arrived CTAs

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
  if (by_ring(vocab, fp32))
    return r.rows == 0 ? set_error("policy_loss: no rows")
           : fp32      ? launch_policy<float>(logits, grad, r, p, partial, arrived, o, st)
                       : launch_policy<__nv_bfloat16>(logits, grad, r, p, partial, arrived, o, st);
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
  // head | loss and count of each pair | softmax of each token | log-probability | slope of each row
  return static_cast<long long>(kHead) + batch * 8 + batch * length * 12 + batch * 4;
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
  unsigned* arrived = reinterpret_cast<unsigned*>(at);
  double* pair_loss = reinterpret_cast<double*>(at + kHead);
  Softmax* softmax = reinterpret_cast<Softmax*>(pair_loss + batch);
  float* logp = reinterpret_cast<float*>(softmax + r.rows);
  float* by = logp + r.rows;
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead, st);
  if (e != cudaSuccess) return set_error("preference_loss: memset: %s", cudaGetErrorString(e));
  auto go = [&](auto* x) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    const bool ring = by_ring(vocab, fp32);
    const unsigned grid = row_grid(r.rows);
    int rc = 0;
    if (ring)
      rc = launch_preference<T, false>(x, nullptr, r, softmax, logp, nullptr, st);
    else
      preference_short_rows_kernel<T><<<grid, kRowThreads, 0, st>>>(x, r, softmax, logp);
    if (rc != 0) return rc;
    preference_pairs_kernel<<<static_cast<unsigned>(pairs), kRowThreads, 0, st>>>(
        logp, r, p, static_cast<float*>(scores), static_cast<float*>(margins), by, nullptr, pair_loss, arrived,
        static_cast<float*>(out));
    if (grad == nullptr) return launched("preference_loss", 2 - ring);
    if (ring)
      rc = launch_preference<T, true>(x, grad, r, softmax, logp, by, st);
    else
      preference_short_gradient_kernel<T><<<grid, kRowThreads, 0, st>>>(x, static_cast<T*>(grad), r, softmax, by);
    return rc != 0 ? rc : launched("preference_loss", ring ? 1 : 3);
  };
  return fp32 ? go(static_cast<const float*>(logits)) : go(static_cast<const __nv_bfloat16*>(logits));
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
