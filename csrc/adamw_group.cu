// One AdamW step of many parameters in one launch, moments in 32 bits or in 8, and the global-norm
// clip factor of their gradients.
//
//   g'  = g * clip_scale                          (clip_scale: device scalar, or 1)
//   mu  = b1 mu + (1 - b1) g'        nu = b2 nu + (1 - b2) g'^2
//   u   = (mu / bc1) / (sqrt(nu / bc2 + eps_root) + eps) + weight_decay * p
//   p  -= lr * u                                  and the bf16 working copy is written
//
// What bounds it: memory. 30 bytes an element with moments in 32 bits (p, mu and nu read and
// written, g read, the bf16 copy written), 18.06 with moments in 8. Launched once per parameter, a
// model of 190 tensors spent 190 launches on it, most of them with less work than a launch costs.
//
// The items travel in the kernel's parameters (no table in device memory that a captured graph would
// have to keep alive). Each CTA takes one chunk of kChunk elements of one item; it finds the item by
// a binary search over the items' first chunks.
//
// Moments in 8 bits: blocks of 256 consecutive values of a tensor share a scale, the largest
// magnitude of the block, held in 32 bits; a value is stored as the e4m3 number next to
// x / largest * 448. The step itself is computed in 32 bits from the moments before they are
// rounded. Of the two neighbours the rounding takes either with the probability that keeps the mean:
// with b2 = 0.999 a second moment moves by 0.1 % of itself per step, half a step of e4m3 is up to
// 6 %, and rounding to nearest would never move it (it stops below a hundredth of the true value).
// The draw is a hash of (seed, step, place in the tensor): a step repeated gives the same bits. A
// second moment that is not zero is never stored as zero, which would divide by eps.
#include <cuda_fp8.h>

#include <cmath>

#include "common.cuh"
#include "t5x_ops.h"

namespace t5x {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 2048;      // elements per CTA
constexpr int kQuantBlock = 256;  // values that share a scale
constexpr int kMaxItems = 448;    // (28 KB of the 32 KB that a launch's parameters may have)
constexpr int kFewItems = 48;

struct Hyper {
  float lr, b1, b2, c1, c2, eps, eps_root, weight_decay, bc1, bc2;  // c = 1 - b
  uint32_t noise_key;
};

template <int kItems>
struct Group {
  Hyper h;
  const float* clip_scale;
  int count;
  unsigned first[kItems];  // first chunk of each item
  t5x_adamw_item item[kItems];
};

template <int kItems>
__device__ __forceinline__ int find_item(const Group<kItems>& grp, unsigned chunk) {
  int lo = 0, hi = grp.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (grp.first[mid] <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Every pointer of the item takes the wide accesses.
__device__ __forceinline__ bool wide(const t5x_adamw_item& it) {
  return ((reinterpret_cast<uintptr_t>(it.p) | reinterpret_cast<uintptr_t>(it.g) |
           reinterpret_cast<uintptr_t>(it.mu) | reinterpret_cast<uintptr_t>(it.nu)) & 15) == 0 &&
         (reinterpret_cast<uintptr_t>(it.out) & 7) == 0;
}

// (The same roundings as in the kernel of one parameter in adamw.cu, so that both give the same bits:
// left to itself the compiler fuses the other product of the second moment here.)
__device__ __forceinline__ void update(const Hyper& h, float gg, float& pp, float& mm, float& nn) {
  mm = __fmaf_rn(h.b1, mm, __fmul_rn(h.c1, gg));
  nn = __fmaf_rn(h.b2, nn, __fmul_rn(__fmul_rn(h.c2, gg), gg));
  const float u = (mm / h.bc1) / (sqrtf(nn / h.bc2 + h.eps_root) + h.eps) + h.weight_decay * pp;
  pp -= h.lr * u;
}

__device__ __forceinline__ uint2 pack_bf16(float4 v) {
  __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y);
  __nv_bfloat162 hi = __floats2bfloat162_rn(v.z, v.w);
  return make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
}

template <int kItems>
__global__ void __launch_bounds__(kThreads)
    adamw_group_kernel(const __grid_constant__ Group<kItems> grp) {
  const unsigned chunk = blockIdx.x;
  const int which = find_item(grp, chunk);
  const t5x_adamw_item it = grp.item[which];
  const Hyper h = grp.h;
  const float cs = grp.clip_scale != nullptr ? *grp.clip_scale : 1.f;
  const long long begin = static_cast<long long>(chunk - grp.first[which]) * kChunk;
  const int n = static_cast<int>(it.n - begin < kChunk ? it.n - begin : kChunk);
  float* p = static_cast<float*>(it.p) + begin;
  const float* g = static_cast<const float*>(it.g) + begin;
  float* mu = static_cast<float*>(it.mu) + begin;
  float* nu = static_cast<float*>(it.nu) + begin;
  __nv_bfloat16* out = it.out != nullptr ? static_cast<__nv_bfloat16*>(it.out) + begin : nullptr;
  if (n == kChunk && wide(it)) {
    constexpr int kVec = kChunk / (4 * kThreads);
    float4 gv[kVec], pv[kVec], mv[kVec], nv[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const int i = k * kThreads + threadIdx.x;
      gv[k] = reinterpret_cast<const float4*>(g)[i];
      pv[k] = reinterpret_cast<const float4*>(p)[i];
      mv[k] = reinterpret_cast<const float4*>(mu)[i];
      nv[k] = reinterpret_cast<const float4*>(nu)[i];
    }
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      const int i = k * kThreads + threadIdx.x;
      update(h, gv[k].x * cs, pv[k].x, mv[k].x, nv[k].x);
      update(h, gv[k].y * cs, pv[k].y, mv[k].y, nv[k].y);
      update(h, gv[k].z * cs, pv[k].z, mv[k].z, nv[k].z);
      update(h, gv[k].w * cs, pv[k].w, mv[k].w, nv[k].w);
      reinterpret_cast<float4*>(mu)[i] = mv[k];
      reinterpret_cast<float4*>(nu)[i] = nv[k];
      reinterpret_cast<float4*>(p)[i] = pv[k];
      if (out != nullptr) reinterpret_cast<uint2*>(out)[i] = pack_bf16(pv[k]);
    }
    return;
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float pp = p[i], mm = mu[i], nn = nu[i];
    update(h, g[i] * cs, pp, mm, nn);
    mu[i] = mm;
    nu[i] = nn;
    p[i] = pp;
    if (out != nullptr) out[i] = __float2bfloat16(pp);
  }
}

// ---- moments in 8 bits ----

// 32 bits for the value at `place` of a tensor: 16 for each moment. The factors are the leading
// bits of the golden ratio and of the square roots of 2 and 3 (all odd).
__device__ __forceinline__ uint32_t noise(uint32_t place, uint32_t key) {
  uint32_t h = (place + key) * 0x9E3779B1u;
  h ^= h >> 15;
  h *= 0x6A09E667u;
  h ^= h >> 13;
  h *= 0xBB67AE85u;
  return h ^ (h >> 16);
}

// The e4m3 code of y in [0, 448], rounded to a neighbour by the 16 random bits r: e4m3 keeps three
// of the 23 bits of the mantissa, so the bits that fall away are topped up by a random number below
// one step before they are cut off. Below 2^-6 the steps are 2^-9 wide; adding 2^-6 puts y among
// numbers whose steps are the same.
__device__ __forceinline__ uint32_t to_e4m3(float y, uint32_t r) {
  const bool low = y < 0.015625f;
  const uint32_t bits = __float_as_uint(low ? y + 0.015625f : y) + (r << 4) + 8u;
  const int code = static_cast<int>(bits >> 20) - (low ? 968 : 960);
  return static_cast<uint32_t>(code < 126 ? code : 126);
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
  const __half2_raw h =
      __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// 1 / largest; 0 where all are zero. (A largest that is not finite makes the whole block NaN when it
// is read back, as the largest itself is kept.)
__device__ __forceinline__ float inverse(float most) { return most > 0.f ? 1.f / most : 0.f; }

__device__ __forceinline__ uint32_t code_mu(float m, float inv, uint32_t r) {
  return to_e4m3(fabsf(m) * inv * 448.f, r & 0xffffu) | ((__float_as_uint(m) >> 24) & 0x80u);
}
__device__ __forceinline__ uint32_t code_nu(float v, float inv, uint32_t r) {
  const uint32_t c = to_e4m3(v * inv * 448.f, r >> 16);
  return c == 0u && v > 0.f ? 1u : c;
}

// A warp per block of 256 values: lane l holds values 4l .. 4l + 3 and 128 + 4l .. 128 + 4l + 3, so
// that every access of the warp is contiguous.
template <int kItems>
__global__ void __launch_bounds__(kThreads)
    adamw8_group_kernel(const __grid_constant__ Group<kItems> grp) {
  const unsigned chunk = blockIdx.x;
  const int which = find_item(grp, chunk);
  const t5x_adamw_item it = grp.item[which];
  const Hyper h = grp.h;
  const int lane = threadIdx.x & 31;
  const long long block = static_cast<long long>(chunk - grp.first[which]) * (kChunk / kQuantBlock) +
                          (threadIdx.x >> 5);
  const long long begin = block * kQuantBlock;
  if (begin >= it.n) return;
  const float cs = grp.clip_scale != nullptr ? *grp.clip_scale : 1.f;
  const int n = static_cast<int>(it.n - begin < kQuantBlock ? it.n - begin : kQuantBlock);
  float* p = static_cast<float*>(it.p) + begin;
  const float* g = static_cast<const float*>(it.g) + begin;
  uint8_t* mu = static_cast<uint8_t*>(it.mu) + begin;
  uint8_t* nu = static_cast<uint8_t*>(it.nu) + begin;
  __nv_bfloat16* out = it.out != nullptr ? static_cast<__nv_bfloat16*>(it.out) + begin : nullptr;
  float* mu_most = static_cast<float*>(it.mu_absmax) + block;
  float* nu_most = static_cast<float*>(it.nu_absmax) + block;
  const uint32_t place = static_cast<uint32_t>(begin);

  float gg[8], pp[8], mm[8], vv[8];
  const bool fast = n == kQuantBlock && wide(it);
  if (fast) {
    float4 gv[2], pv[2];
    uint32_t mc[2], nc[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = k * 32 + lane;
      gv[k] = reinterpret_cast<const float4*>(g)[i];
      pv[k] = reinterpret_cast<const float4*>(p)[i];
      mc[k] = reinterpret_cast<const uint32_t*>(mu)[i];
      nc[k] = reinterpret_cast<const uint32_t*>(nu)[i];
    }
    const float ms = *mu_most, ns = *nu_most;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float2 m0 = from_e4m3x2(mc[k]), m1 = from_e4m3x2(mc[k] >> 16);
      const float2 n0 = from_e4m3x2(nc[k]), n1 = from_e4m3x2(nc[k] >> 16);
      mm[4 * k] = m0.x, mm[4 * k + 1] = m0.y, mm[4 * k + 2] = m1.x, mm[4 * k + 3] = m1.y;
      vv[4 * k] = n0.x, vv[4 * k + 1] = n0.y, vv[4 * k + 2] = n1.x, vv[4 * k + 3] = n1.y;
      gg[4 * k] = gv[k].x, gg[4 * k + 1] = gv[k].y, gg[4 * k + 2] = gv[k].z, gg[4 * k + 3] = gv[k].w;
      pp[4 * k] = pv[k].x, pp[4 * k + 1] = pv[k].y, pp[4 * k + 2] = pv[k].z, pp[4 * k + 3] = pv[k].w;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mm[j] = mm[j] * (1.f / 448.f) * ms;
      vv[j] = vv[j] * (1.f / 448.f) * ns;
    }
  } else {
    const float ms = *mu_most, ns = *nu_most;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = (j >> 2) * 128 + lane * 4 + (j & 3);
      const bool in = i < n;
      gg[j] = in ? g[i] : 0.f;
      pp[j] = in ? p[i] : 0.f;
      mm[j] = in ? from_e4m3x2(mu[i]).x * (1.f / 448.f) * ms : 0.f;
      vv[j] = in ? from_e4m3x2(nu[i]).x * (1.f / 448.f) * ns : 0.f;
    }
  }
  uint32_t mb = 0, nb = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    update(h, gg[j] * cs, pp[j], mm[j], vv[j]);
    const int i = (j >> 2) * 128 + lane * 4 + (j & 3);
    if (fast || i < n) {  // as integers NaN is above every number, so that a NaN stays the largest
      mb = max(mb, abs_bits(mm[j]));
      nb = max(nb, abs_bits(vv[j]));
    }
  }
  mb = __reduce_max_sync(0xffffffffu, mb);
  nb = __reduce_max_sync(0xffffffffu, nb);
  const float mi = inverse(__uint_as_float(mb)), ni = inverse(__uint_as_float(nb));
  if (lane == 0) {  // (every lane has read the old scales: the reduction is behind the reads)
    *mu_most = __uint_as_float(mb);
    *nu_most = __uint_as_float(nb);
  }
  if (fast) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = k * 32 + lane;
      uint32_t mc = 0, nc = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t r = noise(place + 4 * i + j, h.noise_key);
        mc |= code_mu(mm[4 * k + j], mi, r) << (8 * j);
        nc |= code_nu(vv[4 * k + j], ni, r) << (8 * j);
      }
      const float4 pv = make_float4(pp[4 * k], pp[4 * k + 1], pp[4 * k + 2], pp[4 * k + 3]);
      reinterpret_cast<float4*>(p)[i] = pv;
      reinterpret_cast<uint32_t*>(mu)[i] = mc;
      reinterpret_cast<uint32_t*>(nu)[i] = nc;
      if (out != nullptr) reinterpret_cast<uint2*>(out)[i] = pack_bf16(pv);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = (j >> 2) * 128 + lane * 4 + (j & 3);
    if (i >= n) continue;
    const uint32_t r = noise(place + i, h.noise_key);
    p[i] = pp[j];
    mu[i] = static_cast<uint8_t>(code_mu(mm[j], mi, r));
    nu[i] = static_cast<uint8_t>(code_nu(vv[j], ni, r));
    if (out != nullptr) out[i] = __float2bfloat16(pp[j]);
  }
}

// ---- global norm ----

// Sum of squares of the chunks blockIdx.x, blockIdx.x + gridDim.x, ... in 64 bits across chunks
// (eight values of a thread in 32). A CTA's chunks and the order of all sums depend on the grid
// alone. `finish`: the CTA that arrives last adds the partial sums of this and the earlier launches of
// the call and stores the clip factor min(1, max_norm / (norm + 1e-16)).
template <int kItems>
__global__ void __launch_bounds__(kThreads)
    sumsq_group_kernel(const __grid_constant__ Group<kItems> grp, unsigned chunks, double* partial,
                       int partial_first, unsigned* arrived, float max_norm, float* clip_out) {
  __shared__ double s_sum[kThreads / 32];
  __shared__ bool s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum = 0.0;
  for (unsigned chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int which = find_item(grp, chunk);
    const t5x_adamw_item& it = grp.item[which];
    const long long begin = static_cast<long long>(chunk - grp.first[which]) * kChunk;
    const int n = static_cast<int>(it.n - begin < kChunk ? it.n - begin : kChunk);
    const float* g = static_cast<const float*>(it.g) + begin;
    float s = 0.f;
    if (n == kChunk && (reinterpret_cast<uintptr_t>(it.g) & 15) == 0) {
#pragma unroll
      for (int k = 0; k < kChunk / (4 * kThreads); ++k) {
        const float4 v = reinterpret_cast<const float4*>(g)[k * kThreads + threadIdx.x];
        s += v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w;
      }
    } else {
      for (int i = threadIdx.x; i < n; i += kThreads) s += g[i] * g[i];
    }
    sum += static_cast<double>(s);
  }
  auto block_sum = [&](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) s_sum[warp] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) t += s_sum[w];
    return t;
  };
  sum = block_sum(sum);
  if (threadIdx.x == 0) {
    partial[partial_first + blockIdx.x] = sum;
    s_last = false;
    if (clip_out != nullptr) {
      __threadfence();
      s_last = atomicAdd(arrived, 1u) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double total = 0.0;
  for (int i = threadIdx.x; i < partial_first + static_cast<int>(gridDim.x); i += kThreads)
    total += __ldcg(partial + i);
  total = block_sum(total);
  if (threadIdx.x == 0) {
    const float f = max_norm / (static_cast<float>(sqrt(total)) + 1e-16f);
    *clip_out = f > 1.f ? 1.f : f;  // (NaN stays)
  }
}

// Fills `grp` with items [from, ...) up to its capacity; returns how many it took and the chunks.
template <int kItems>
int fill(Group<kItems>& grp, const t5x_adamw_item* items, int from, int count, unsigned* chunks) {
  grp.count = 0;
  unsigned long long c = 0;
  int i = from;
  for (; i < count && grp.count < kItems; ++i) {
    const unsigned long long need = (static_cast<unsigned long long>(items[i].n) + kChunk - 1) / kChunk;
    if (need == 0) continue;
    if (c + need > 0x7fffffffull) break;
    grp.first[grp.count] = static_cast<unsigned>(c);
    grp.item[grp.count++] = items[i];
    c += need;
  }
  *chunks = static_cast<unsigned>(c);
  return i - from;
}

int validate(const char* what, const t5x_adamw_item* items, int count, int bits) {
  if (count < 0 || (count > 0 && items == nullptr)) return set_error("%s: bad item list", what);
  for (int i = 0; i < count; ++i) {
    const t5x_adamw_item& it = items[i];
    if (it.n < 0) return set_error("%s: item %d has a negative size", what, i);
    if (it.n > (1ll << 41)) return set_error("%s: item %d is too large", what, i);
    if (it.n == 0) continue;
    if (it.g == nullptr) return set_error("%s: null pointer", what);
    if (reinterpret_cast<uintptr_t>(it.g) & 3) return set_error("%s: misaligned pointer", what);
    if (bits == 0) continue;
    if (it.p == nullptr || it.mu == nullptr || it.nu == nullptr ||
        (bits == 8 && (it.mu_absmax == nullptr || it.nu_absmax == nullptr)))
      return set_error("%s: null pointer", what);
    uintptr_t fours = reinterpret_cast<uintptr_t>(it.p);
    if (bits == 8)
      fours |= reinterpret_cast<uintptr_t>(it.mu_absmax) | reinterpret_cast<uintptr_t>(it.nu_absmax);
    else
      fours |= reinterpret_cast<uintptr_t>(it.mu) | reinterpret_cast<uintptr_t>(it.nu);
    if ((fours & 3) || (reinterpret_cast<uintptr_t>(it.out) & 1))
      return set_error("%s: misaligned pointer", what);
  }
  return 0;
}

template <int kItems>
int step_in_groups(const t5x_adamw_item* items, int count, const Hyper& h, const float* clip_scale, int bits,
                   cudaStream_t st) {
  Group<kItems> grp;
  grp.h = h;
  grp.clip_scale = clip_scale;
  for (int from = 0; from < count;) {
    unsigned chunks;
    from += fill(grp, items, from, count, &chunks);
    if (chunks == 0) continue;
    if (bits == 8)
      adamw8_group_kernel<kItems><<<chunks, kThreads, 0, st>>>(grp);
    else
      adamw_group_kernel<kItems><<<chunks, kThreads, 0, st>>>(grp);
    count_launches(1);
  }
  return 0;
}

template <int kItems>
int sumsq_in_groups(const t5x_adamw_item* items, int count, void* scratch, float max_norm, float* clip,
                    cudaStream_t st) {
  Group<kItems> grp;
  grp.clip_scale = nullptr;
  unsigned* arrived = static_cast<unsigned*>(scratch);
  double* partial = reinterpret_cast<double*>(static_cast<char*>(scratch) + 16);
  const unsigned cap = static_cast<unsigned>(num_sms()) * 8;
  int first = 0, from = 0;
  do {
    unsigned chunks = 0;
    from += fill(grp, items, from, count, &chunks);
    const bool last = from >= count;
    if (chunks == 0 && !last) continue;
    const unsigned grid = chunks == 0 ? 1 : (chunks < cap ? chunks : cap);
    sumsq_group_kernel<kItems><<<grid, kThreads, 0, st>>>(grp, chunks, partial, first, arrived, max_norm,
                                                          last ? clip : nullptr);
    count_launches(1);
    first += static_cast<int>(grid);
  } while (from < count);
  return 0;
}

int launches_for(int count) { return count <= kMaxItems ? 1 : (count + kMaxItems - 1) / kMaxItems; }

}  // namespace
}  // namespace t5x

T5X_API long long t5x_grad_clip_scratch_bytes(const t5x_adamw_item* items, int count) {
  // (a launch ends early only where its chunks would pass 2^31: such lists get a launch an item)
  using namespace t5x;
  long long total = 0;
  for (int i = 0; i < count; ++i) total += items[i].n > 0 ? items[i].n : 0;
  const long long launches = total / (1ll << 40) > 0 ? count : launches_for(count);
  return 16 + 8ll * num_sms() * 8 * (launches + 1);
}

T5X_API int t5x_grad_clip_scale(const t5x_adamw_item* items, int count, void* scratch, float max_norm,
                                void* clip_scale, void* stream) {
  using namespace t5x;
  if (validate("grad_clip_scale", items, count, 0)) return -1;
  if (scratch == nullptr || clip_scale == nullptr) return set_error("grad_clip_scale: null pointer");
  if ((reinterpret_cast<uintptr_t>(scratch) & 7) || (reinterpret_cast<uintptr_t>(clip_scale) & 3))
    return set_error("grad_clip_scale: misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(scratch, 0, 16, st);
  if (e != cudaSuccess) return set_error("grad_clip_scale: memset: %s", cudaGetErrorString(e));
  float* clip = static_cast<float*>(clip_scale);
  if (count <= kFewItems)
    sumsq_in_groups<kFewItems>(items, count, scratch, max_norm, clip, st);
  else
    sumsq_in_groups<kMaxItems>(items, count, scratch, max_norm, clip, st);
  e = cudaGetLastError();
  if (e != cudaSuccess) return set_error("grad_clip_scale: %s", cudaGetErrorString(e));
  return 0;
}

T5X_API int t5x_adamw_group(const t5x_adamw_item* items, int count, int state_bits, float lr, double b1,
                            double b2, float eps, float eps_root, float weight_decay, int step,
                            unsigned int seed, const void* clip_scale, void* stream) {
  using namespace t5x;
  if (state_bits != 8 && state_bits != 32) return set_error("adamw_group: moments have 8 or 32 bits");
  if (step < 1) return set_error("adamw_group: step counts from 1");
  if (validate("adamw_group", items, count, state_bits)) return -1;
  Hyper h;
  h.lr = lr;
  h.b1 = static_cast<float>(b1);
  h.b2 = static_cast<float>(b2);
  h.eps = eps;
  h.eps_root = eps_root;
  h.weight_decay = weight_decay;
  if (state_bits == 32) {  // as in the kernel of one parameter, for the same bits
    h.c1 = 1.f - h.b1;
    h.c2 = 1.f - h.b2;
    h.bc1 = 1.f - powf(h.b1, static_cast<float>(step));
    h.bc2 = 1.f - powf(h.b2, static_cast<float>(step));
  } else {  // (1 - 0.999f is 1.3e-5 off 0.001)
    h.c1 = static_cast<float>(1.0 - b1);
    h.c2 = static_cast<float>(1.0 - b2);
    h.bc1 = static_cast<float>(1.0 - pow(b1, step));
    h.bc2 = static_cast<float>(1.0 - pow(b2, step));
  }
  h.noise_key = seed * 0x9E3779B1u + static_cast<unsigned>(step) * 0xBB67AE85u;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const float* cs = static_cast<const float*>(clip_scale);
  if (count <= kFewItems)
    step_in_groups<kFewItems>(items, count, h, cs, state_bits, st);
  else
    step_in_groups<kMaxItems>(items, count, h, cs, state_bits, st);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error("adamw_group: %s", cudaGetErrorString(e));
  return 0;
}
