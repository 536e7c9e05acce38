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

// The rows are walked by teams: warps for short rows, whole CTAs for long ones.
template <int kTeam>
struct Team {
  int tid, id, count;
  __device__ Team()
      : tid(kTeam == 32 ? threadIdx.x & 31 : threadIdx.x),
        id(kTeam == 32 ? (blockIdx.x * blockDim.x + threadIdx.x) >> 5 : blockIdx.x),
        count(kTeam == 32 ? (gridDim.x * blockDim.x) >> 5 : gridDim.x) {}
  // The whole row's softmax; valid in the first warp of the team.
  __device__ Softmax reduce(Softmax s) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Softmax other = {__shfl_xor_sync(0xffffffffu, s.most, o), __shfl_xor_sync(0xffffffffu, s.sum, o)};
      s = join(s, other);
    }
    if (kTeam > 32) {
      __shared__ Softmax part[kTeam / 32];
      if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
      __syncthreads();
      if (threadIdx.x < 32) {
        s = threadIdx.x < kTeam / 32 ? part[threadIdx.x] : Softmax{-INFINITY, 0.f};
#pragma unroll
        for (int o = kTeam / 64; o > 0; o >>= 1) {
          const Softmax other = {__shfl_xor_sync(0xffffffffu, s.most, o), __shfl_xor_sync(0xffffffffu, s.sum, o)};
          s = join(s, other);
        }
      }
    }
    return s;
  }
  // v of the team's first thread.
  template <typename V>
  __device__ V broadcast(V v) const {
    if (kTeam == 32) {
      int w[sizeof(V) / 4];
      memcpy(w, &v, sizeof(V));
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(V) / 4); ++i) w[i] = __shfl_sync(0xffffffffu, w[i], 0);
      memcpy(&v, w, sizeof(V));
      return v;
    }
    __shared__ V s;
    __syncthreads();  // (the last row's is read)
    if (threadIdx.x == 0) s = v;
    __syncthreads();
    return s;
  }
};

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

template <typename T, int kTeam>
__global__ void __launch_bounds__(kRowThreads)
    policy_rows_kernel(const T* __restrict__ logits, T* __restrict__ grad, const Rows r, const Policy p,
                       double* partial, unsigned* arrived, float* out) {
  const Team<kTeam> team;
  const float scale = scale_of(p.normalizer, p.scale);
  double sums[4] = {0.0, 0.0, 0.0, 0.0};
  for (long long row = team.id; row < r.rows; row += team.count) {
    const float w = r.weights != nullptr ? r.weights[row] : 1.f;
    const long long at = row_at(r, row);
    if (w == 0.f) {
      if (grad != nullptr) row_zero(grad + at, r.vocab, team.tid, kTeam);
      continue;
    }
    struct Said {
      Softmax s;
      float by;
      int target;
    } said = {team.reduce(row_softmax(logits + at, r.vocab, team.tid, kTeam)), 0.f, 0};
    if (team.tid == 0) {
      const long long target = r.targets[row], b = row / r.length;
      const float logp = log_prob(logits + at, r.vocab, target, said.s);
      const PolicyToken k = policy_token(p, row, b, row - b * r.length, logp);
      sums[0] += static_cast<double>(w) * k.loss;
      sums[1] += static_cast<double>(w) * k.kl;
      sums[2] += static_cast<double>(w) * k.clipped;
      sums[3] += w;
      said.by = w * k.slope * scale;
      said.target = target >= 0 && target < r.vocab ? static_cast<int>(target) : -1;
    }
    if (grad == nullptr) {
      if (kTeam > 32) __syncthreads();  // (the partial sums are read)
      continue;
    }
    said = team.broadcast(said);
    if (said.by == 0.f)
      row_zero(grad + at, r.vocab, team.tid, kTeam);
    else
      row_gradient(logits + at, grad + at, r.vocab, said.s, said.target, said.by, team.tid, kTeam);
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

template <typename T, int kTeam>
__global__ void __launch_bounds__(kRowThreads)
    preference_rows_kernel(const T* __restrict__ logits, const Rows r, Softmax* __restrict__ softmax,
                           float* __restrict__ logp) {
  const Team<kTeam> team;
  for (long long row = team.id; row < r.rows; row += team.count) {
    if (r.weights != nullptr && r.weights[row] == 0.f) continue;
    const long long at = row_at(r, row);
    const Softmax s = team.reduce(row_softmax(logits + at, r.vocab, team.tid, kTeam));
    if (team.tid == 0) {
      softmax[row] = s;
      logp[row] = log_prob(logits + at, r.vocab, r.targets[row], s);
    }
    if (kTeam > 32) __syncthreads();  // (the partial sums are read)
  }
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
  const double margin =
      real ? p.beta * ((sum[0] - p.ref[2 * pair]) - (sum[1] - p.ref[2 * pair + 1])) : 0.0;
  // log(1 + exp(-d)) = log1p(exp(-|d|)) + max(-d, 0)
  const double e = exp(-fabs(margin)), tail = log1p(e);
  const double sigmoid = margin >= 0.0 ? 1.0 / (1.0 + e) : e / (1.0 + e);
  const double slope = real ? p.beta * (sigmoid - (1.0 - p.smoothing)) * scale : 0.0;
  if (threadIdx.x == 0) {
    double loss = 0.0;
    if (real)
      loss = margin != margin ? margin
                              : (1.0 - p.smoothing) * (tail + fmax(-margin, 0.0)) +
                                    p.smoothing * (tail + fmax(margin, 0.0));
    scores[2 * pair] = static_cast<float>(sum[0]);
    scores[2 * pair + 1] = static_cast<float>(sum[1]);
    margins[pair] = static_cast<float>(margin);
    if (by != nullptr) {
      by[2 * pair] = static_cast<float>(slope);
      by[2 * pair + 1] = static_cast<float>(-slope);
    }
    pair_loss[2 * pair] = loss;
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

template <typename T, int kTeam>
__global__ void __launch_bounds__(kRowThreads)
    preference_gradient_kernel(const T* __restrict__ logits, T* __restrict__ grad, const Rows r,
                               const Softmax* __restrict__ softmax, const float* __restrict__ by) {
  const Team<kTeam> team;
  for (long long row = team.id; row < r.rows; row += team.count) {
    const float w = r.weights != nullptr ? r.weights[row] : 1.f;
    const long long at = row_at(r, row);
    const float slope = w == 0.f ? 0.f : w * by[row / r.length];
    if (slope == 0.f) {
      row_zero(grad + at, r.vocab, team.tid, kTeam);
      continue;
    }
    const long long target = r.targets[row];
    row_gradient(logits + at, grad + at, r.vocab, softmax[row],
                 target >= 0 && target < r.vocab ? static_cast<int>(target) : -1, slope, team.tid, kTeam);
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
constexpr int kShortRow = 2048;  // values; shorter rows are a warp's

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

unsigned row_grid(long long rows, bool by_warp) {
  const long long ctas = by_warp ? (rows + kRowThreads / 32 - 1) / (kRowThreads / 32) : rows;
  const long long cap = static_cast<long long>(num_sms()) * 4;
  return static_cast<unsigned>(ctas < 1 ? 1 : (ctas < cap ? ctas : cap));
}

int launched(const char* what, int n) {
  count_launches(n);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error("%s: %s", what, cudaGetErrorString(e));
  return 0;
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
  const bool by_warp = vocab < kShortRow;
  const unsigned grid = row_grid(r.rows, by_warp);
  auto go = [&](auto kernel, auto* x) {
    kernel<<<grid, kRowThreads, 0, st>>>(x, static_cast<std::remove_const_t<std::remove_pointer_t<decltype(x)>>*>(grad),
                                         r, p, partial, arrived, static_cast<float*>(out));
  };
  if (fp32) {
    const float* x = static_cast<const float*>(logits);
    by_warp ? go(policy_rows_kernel<float, 32>, x) : go(policy_rows_kernel<float, kRowThreads>, x);
  } else {
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(logits);
    by_warp ? go(policy_rows_kernel<__nv_bfloat16, 32>, x) : go(policy_rows_kernel<__nv_bfloat16, kRowThreads>, x);
  }
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
  policy_tokens_kernel<<<row_grid((r.rows + kRowThreads - 1) / kRowThreads, false), kRowThreads, 0, st>>>(
      static_cast<const float*>(logp), static_cast<float*>(slope), r, p,
      reinterpret_cast<double*>(static_cast<char*>(scratch) + kHead), static_cast<unsigned*>(scratch),
      static_cast<float*>(out));
  return launched("policy_loss_tokens", 1);
}

T5X_API long long t5x_preference_loss_scratch_bytes(long long batch, int length) {
  // head | loss and count of each pair | largest and sum of each token | log-probability | slope of each row
  return static_cast<long long>(kHead) + batch * 8 + batch * length * 12 + batch * 4;
}

T5X_API int t5x_preference_loss(const void* logits, int fp32, void* grad, long long batch, int length, int vocab,
                                long long stride_b, long long stride_t, const void* targets, const void* weights,
                                const void* reference, float beta, float smoothing, float scale,
                                const void* normalizer, void* scratch, void* scores, void* margins, void* out,
                                void* stream) {
  if (check_rows("preference_loss", logits, fp32, grad, batch, length, vocab, stride_b, stride_t, targets)) return -1;
  if (batch < 2 || batch % 2) return set_error("preference_loss: the batch must hold pairs");
  if (!scratch || !out || !reference || !scores || !margins) return set_error("preference_loss: null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(scratch, 0, kHead, st);
  if (e != cudaSuccess) return set_error("preference_loss: memset: %s", cudaGetErrorString(e));
  const Rows r = {batch * length, length, vocab, stride_b, stride_t, static_cast<const long long*>(targets),
                  static_cast<const float*>(weights)};
  const Preference p = {static_cast<const float*>(reference), beta, smoothing, scale,
                        static_cast<const float*>(normalizer)};
  char* at = static_cast<char*>(scratch);
  unsigned* arrived = reinterpret_cast<unsigned*>(at);
  double* pair_loss = reinterpret_cast<double*>(at + kHead);
  Softmax* softmax = reinterpret_cast<Softmax*>(at + kHead + batch * 8);
  float* logp = reinterpret_cast<float*>(softmax + r.rows);
  float* by = logp + r.rows;
  const bool by_warp = vocab < kShortRow;
  const unsigned grid = row_grid(r.rows, by_warp);
  auto go = [&](auto rows, auto gradient, auto* x) {
    if (r.rows > 0) rows<<<grid, kRowThreads, 0, st>>>(x, r, softmax, logp);
    preference_pairs_kernel<<<static_cast<unsigned>(batch / 2), kRowThreads, 0, st>>>(
        logp, r, p, static_cast<float*>(scores), static_cast<float*>(margins), by, nullptr, pair_loss, arrived,
        static_cast<float*>(out));
    if (grad != nullptr && r.rows > 0)
      gradient<<<grid, kRowThreads, 0, st>>>(
          x, static_cast<std::remove_const_t<std::remove_pointer_t<decltype(x)>>*>(grad), r, softmax, by);
  };
  if (fp32) {
    const float* x = static_cast<const float*>(logits);
    by_warp ? go(preference_rows_kernel<float, 32>, preference_gradient_kernel<float, 32>, x)
            : go(preference_rows_kernel<float, kRowThreads>, preference_gradient_kernel<float, kRowThreads>, x);
  } else {
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(logits);
    by_warp ? go(preference_rows_kernel<__nv_bfloat16, 32>, preference_gradient_kernel<__nv_bfloat16, 32>, x)
            : go(preference_rows_kernel<__nv_bfloat16, kRowThreads>,
                 preference_gradient_kernel<__nv_bfloat16, kRowThreads>, x);
  }
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
