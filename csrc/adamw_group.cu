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
// have to keep alive). Each CTA takes one chunk of one item, which it finds by a binary search over the
// items' first chunks between two of 256 hints (over all of 300 items the search took 5 % of the time).
//
// Moments in 8 bits: blocks of 256 consecutive values of a tensor share a scale, the largest
// magnitude of the block, held in 32 bits; a value is stored as the e4m3 number next to
// x / largest * 448. The step itself is computed in 32 bits from the moments before they are
// rounded. Of the two neighbours the rounding takes either with the probability that keeps the mean:
// with b2 = 0.999 a second moment moves by 0.1 % of itself per step, half a step of e4m3 is up to
// 6 %, and rounding to nearest would never move it (it stops below a hundredth of the true value).
// The draw is a hash of (seed, step, place in the tensor): a step repeated gives the same bits. A
// second moment that is not zero is never stored as zero, which would divide by eps. For that the scale of a
// block with anything in it is 2^-100 at least: the smallest number of such a block is 2^-118, and arithmetic
// here takes what lies below 2^-126 for zero.
#include <cuda_fp8.h>

#include <cmath>

#include "common.cuh"
#include "t5x_ops.h"

namespace t5x {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 2048;      // elements per CTA
constexpr int kQuantBlock = 256;  // values that share a scale
// The bits of 2^-100, of infinity and of NaN.
constexpr uint32_t kLeastScale = (127u - 100) << 23, kInfinity = 0x7f800000u, kNan = 0x7fffffffu;
constexpr int kSpan = 4;          // chunks that a CTA of the norm takes in a row
// Of a launch: what fits in 31 KB of the 32 KB that its parameters may have. (All with the items of 8 bits: 558 small
// tensors took two launches where one is enough.)
constexpr int kMaxItems = 576, kMaxItems8 = 448, kMaxNorms = 1408;
constexpr int kHints = 256;
constexpr int kFewItems = 48;

struct Hyper {
  float lr, b1, b2, c1, c2, eps, eps_root, weight_decay, bc1, bc2;  // c = 1 - b
  float one, ibc2, lr_bc1, lr_decay;  // for moments in 8 bits: 1, 1 / bc2, -lr / bc1, -lr * weight_decay
  uint32_t noise_key;
};

// Of an item, what the kernel of moments in 32 bits, in 8, and the norm need.
struct Item32 {
  void* p;
  const void* g;
  void *mu, *nu, *out;
  long long n;
  static Item32 of(const t5x_adamw_item& i) { return {i.p, i.g, i.mu, i.nu, i.out, i.n}; }
};
struct Item8 : t5x_adamw_item {
  static Item8 of(const t5x_adamw_item& i) { return {i}; }
};
struct ItemNorm {
  const void* g;
  long long n;
  static ItemNorm of(const t5x_adamw_item& i) { return {i.g, i.n}; }
};

template <typename Item, int kItems>
struct Group {
  Hyper h;
  const float* clip_scale;
  int count, shift;
  unsigned ahead;                   // chunks from a CTA's own to the one that it has fetched into L2
  unsigned first[kItems];           // first chunk of each item
  bool wide[kItems];                // every pointer of the item takes the wide accesses
  unsigned short near[kHints + 1];  // item of chunk (i << shift); behind the last chunk the last item
  Item item[kItems];
};
template <int kItems>
using Group32 = Group<Item32, kItems>;
template <int kItems>
using Group8 = Group<Item8, kItems>;
template <int kItems>
using GroupNorm = Group<ItemNorm, kItems>;
static_assert(sizeof(Group32<kMaxItems>) < 32700 && sizeof(Group8<kMaxItems8>) < 32700 &&
                  sizeof(GroupNorm<kMaxNorms>) < 32700 - 64,
              "parameters of a launch");

template <typename Items>
__device__ __forceinline__ int find_item(const Items& grp, unsigned chunk) {
  const unsigned hint = chunk >> grp.shift;
  int lo = grp.near[hint], hi = grp.near[hint + 1] + 1;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (grp.first[mid] <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

bool takes_wide(const t5x_adamw_item& it) {
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
    adamw_group_kernel(const __grid_constant__ Group32<kItems> grp) {
  const unsigned chunk = blockIdx.x;
  const int which = find_item(grp, chunk);
  const auto it = grp.item[which];
  const Hyper h = grp.h;
  const float cs = grp.clip_scale != nullptr ? *grp.clip_scale : 1.f;
  const long long begin = static_cast<long long>(chunk - grp.first[which]) * kChunk;
  const int n = static_cast<int>(it.n - begin < kChunk ? it.n - begin : kChunk);
  float* p = static_cast<float*>(it.p) + begin;
  const float* g = static_cast<const float*>(it.g) + begin;
  float* mu = static_cast<float*>(it.mu) + begin;
  float* nu = static_cast<float*>(it.nu) + begin;
  __nv_bfloat16* out = it.out != nullptr ? static_cast<__nv_bfloat16*>(it.out) + begin : nullptr;
  if (n == kChunk && grp.wide[which]) {
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

// 32 random bits for the value at a place of its tensor, 16 for each moment: a hash of (place + key),
// with the key from seed and step, begun with the product (place + key) * kNoise1. The factors are the
// leading bits of the golden ratio and of the square roots of 2 and 3 (all odd).
constexpr uint32_t kNoise1 = 0x9E3779B1u;
struct Noise {
  uint32_t mu, nu;  // the 16 bits at bits 4 to 19
};
__device__ __forceinline__ Noise noise(uint32_t h) {
  h ^= h >> 15;
  h *= 0x6A09E667u;
  h ^= h >> 13;
  h *= 0xBB67AE85u;
  // the halves of h ^ (h >> 16)
  const uint32_t high = h >> 12;
  return {((h << 4) ^ high) & 0xffff0u, high & 0xffff0u};
}

// ---- pairs of values: sm_100 does two 32-bit products or sums in one instruction ----
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
        "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.ftz.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2_down(float2 a, float2 b) {  // (rounded toward zero)
  uint64_t d;
  asm("add.rz.ftz.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// a / b to the nearest from inv = 1 / b to the nearest: Markstein's correction (IBM J. Res. Dev. 34, 1990).
__device__ __forceinline__ float2 divide2(float2 a, float2 b, float2 inv) {
  const float2 q = mul2(a, inv);
  return fma2(fma2(make_float2(-q.x, -q.y), b, a), inv, q);
}
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The step of two values; m and v: the old moments, then the new ones. Their products and sums are
// rounded one by one, so that a moment before it is stored is, bit for bit, what tensor operations make
// of it: a draw that lies next to its border would else fall on the other side of it, and a second
// moment that is a step of e4m3 apart shows in the weights of the next step. (The assembler makes one
// fused instruction of a paired product and the paired sum behind it; it cannot where the sum is a
// product with a `one` that it does not know.)
__device__ __forceinline__ void update2(const Hyper& h, float2 g, float2& p, float2& m, float2& v) {
  m = fma2(mul2(m, both(h.b1)), both(h.one), mul2(g, both(h.c1)));
  v = fma2(mul2(v, both(h.b2)), both(h.one), mul2(mul2(g, g), both(h.c2)));
  float2 d = fma2(v, both(h.ibc2), both(h.eps_root));
  d = add2(make_float2(sqrtf(d.x), sqrtf(d.y)), both(h.eps));
  const float2 r = make_float2(reciprocal(d.x), reciprocal(d.y));
  p = add2(p, fma2(mul2(m, r), both(h.lr_bc1), mul2(p, both(h.lr_decay))));
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
  const __half2_raw h =
      __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffffu), __NV_E4M3);
  return __half22float2(__half2(h));
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The two e4m3 codes of x / largest * 448, each rounded to a neighbour by 16 random bits (at bits 4 to 19
// of `noise`): e4m3 keeps three of the 23 bits of the mantissa, so the bits that fall away are topped
// up by a random number below one step before they are cut off. Below 2^-6 the steps are 2^-9 wide;
// with 2^-6 added the value lies among numbers whose steps are the same, and what is left when it is
// taken off again is exact. (That sum drops bits below those of the draw, which cannot carry: rounded to the
// nearest it moved one in 60 million values across a border.) kSecond: no sign, and nothing is stored as
// zero (the caller sees to zeros).
// `quarter`: a quarter of the largest, inv: its reciprocal, which is a normal number for any largest (that of a largest
// above 2^126 itself is not, and was zero).
// (A largest that is not finite makes the whole block NaN when it is read back: infinity is kept as NaN, as codes other
// than zero times infinity would be infinite second moments, steps of 0 for good.)
template <bool kSecond>
__device__ __forceinline__ uint32_t codes2(float2 x, float quarter, float inv, uint32_t noise0, uint32_t noise1) {
  const float2 y = mul2(divide2(x, both(quarter), both(inv)), both(112.f));
  auto shift = [](float v) {
    const float by = kSecond ? 0.015625f
                             : __uint_as_float((__float_as_uint(v) & 0x80000000u) | 0x3c800000u);
    return fabsf(v) < 0.015625f ? by : 0.f;
  };
  const float2 c = make_float2(shift(y.x), shift(y.y));
  float2 z = add2_down(y, c);
  z.x = __uint_as_float((__float_as_uint(z.x) + noise0 + 8u) & 0xfff00000u);
  z.y = __uint_as_float((__float_as_uint(z.y) + noise1 + 8u) & 0xfff00000u);
  z = fma2(c, both(-1.f), z);
  if (kSecond) {
    z.x = fmaxf(z.x, 0.001953125f);
    z.y = fmaxf(z.y, 0.001953125f);
  }
  return __nv_cvt_float2_to_fp8x2(z, __NV_SATFINITE, __NV_E4M3);
}

// (16-byte aligned address, size a multiple of 16 bytes)
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// What a lane reads of a block: values 4l .. 4l + 3 and 128 + 4l .. 128 + 4l + 3, so that every access of
// the warp is contiguous.
struct Block8 {
  float4 g[2], p[2];
  uint32_t mu[2], nu[2];
  float mu_most, nu_most;
};

// The step of one block by a warp, from the block's values to its new ones in their places.
struct Result8 {
  float2 p[4];  // pair j: values (j / 2) * 128 + 4 * lane + 2 * (j % 2) and the next
  uint32_t mu[4], nu[4];
  uint32_t mu_most, nu_most;
};
__device__ __forceinline__ Result8 step8(const Hyper& h, float clip, const Block8& in, uint32_t key, int lane) {
  // codes stand for code * (largest / 448)
  const float2 mu_unit = both(__fmul_rn(in.mu_most, 1.f / 448.f));
  const float2 nu_unit = both(__fmul_rn(in.nu_most, 1.f / 448.f));
  Result8 r;
  float2 m[4], v[4];
  r.mu_most = r.nu_most = 0;
  float nu_least = 1.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = j >> 1, s = (j & 1) * 16;
    const float2 g = j & 1 ? make_float2(in.g[k].z, in.g[k].w) : make_float2(in.g[k].x, in.g[k].y);
    r.p[j] = j & 1 ? make_float2(in.p[k].z, in.p[k].w) : make_float2(in.p[k].x, in.p[k].y);
    m[j] = mul2(from_e4m3x2(in.mu[k] >> s), mu_unit);
    v[j] = mul2(from_e4m3x2(in.nu[k] >> s), nu_unit);
    update2(h, mul2(g, both(clip)), r.p[j], m[j], v[j]);
    // as integers NaN is above every number, so that a NaN stays the largest
    r.mu_most = max(r.mu_most, max(abs_bits(m[j].x), abs_bits(m[j].y)));
    r.nu_most = max(r.nu_most, max(__float_as_uint(v[j].x), __float_as_uint(v[j].y)));
    nu_least = fminf(nu_least, fminf(v[j].x, v[j].y));
  }
  r.mu_most = __reduce_max_sync(0xffffffffu, r.mu_most);
  r.nu_most = __reduce_max_sync(0xffffffffu, r.nu_most);
  r.mu_most = r.mu_most != 0 ? max(r.mu_most, kLeastScale) : 0;
  r.nu_most = r.nu_most != 0 ? max(r.nu_most, kLeastScale) : 0;
  if (r.mu_most == kInfinity) r.mu_most = kNan;
  if (r.nu_most == kInfinity) r.nu_most = kNan;
  const float mu_quarter = 0.25f * __uint_as_float(r.mu_most), nu_quarter = 0.25f * __uint_as_float(r.nu_most);
  const float mu_inv = mu_quarter > 0.f ? __frcp_rn(mu_quarter) : 0.f;  // (all zeros: codes of zero)
  const float nu_inv = nu_quarter > 0.f ? __frcp_rn(nu_quarter) : 0.f;
  const uint32_t seed = (key + lane * 4) * kNoise1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t i = (j >> 1) * 128 + (j & 1) * 2;
    const Noise a = noise(seed + i * kNoise1), b = noise(seed + (i + 1) * kNoise1);
    r.mu[j] = codes2<false>(m[j], mu_quarter, mu_inv, a.mu, b.mu);
    r.nu[j] = codes2<true>(v[j], nu_quarter, nu_inv, a.nu, b.nu);
  }
  if (nu_least <= 0.f) {  // rare: weights that have had no gradient yet
#pragma unroll
    for (int j = 0; j < 4; ++j)
      r.nu[j] &= (v[j].x > 0.f ? 0xffu : 0u) | (v[j].y > 0.f ? 0xff00u : 0u);
  }
  return r;
}

// A warp per block of 256 values. What bounds it: some 65 instructions an element beside its 18 bytes (80
// before products and sums went in pairs), so that a warp spends half of its time with no load in
// flight, and under a load of seconds the clock (the power cap takes 10 %). A CTA therefore has the chunk
// of a later CTA fetched into L2, one wave of CTAs ahead: 77M elements in 190 tensors 246 -> 211 us,
// sustained 253 -> 230; half a wave 218, two 228, four 298. Four CTAs an SM 230, five (spills) 242; a warp
// that works on several blocks in a row 276 to 316. With the moments rounded as tensor operations round
// them 247 us sustained (5.6 TB/s).
template <int kItems>
__global__ void __launch_bounds__(kThreads, 4)
    adamw8_group_kernel(const __grid_constant__ Group8<kItems> grp) {
  const unsigned chunk = blockIdx.x;
  const int which = find_item(grp, chunk);
  const auto it = grp.item[which];
  const int lane = threadIdx.x & 31;
  const long long block = static_cast<long long>(chunk - grp.first[which]) * (kChunk / kQuantBlock) +
                          (threadIdx.x >> 5);
  const long long begin = block * kQuantBlock;
  if (begin >= it.n) return;
  const int n = static_cast<int>(it.n - begin < kQuantBlock ? it.n - begin : kQuantBlock);
  float* p = static_cast<float*>(it.p) + begin;
  const float* g = static_cast<const float*>(it.g) + begin;
  uint8_t* mu = static_cast<uint8_t*>(it.mu) + begin;
  uint8_t* nu = static_cast<uint8_t*>(it.nu) + begin;
  __nv_bfloat16* out = it.out != nullptr ? static_cast<__nv_bfloat16*>(it.out) + begin : nullptr;
  float* mu_most = static_cast<float*>(it.mu_absmax) + block;
  float* nu_most = static_cast<float*>(it.nu_absmax) + block;
  const bool fast = n == kQuantBlock && grp.wide[which];

  if (threadIdx.x == 0 && chunk + grp.ahead < gridDim.x) {
    const unsigned later = chunk + grp.ahead;
    const int w = find_item(grp, later);
    const Item8& item = grp.item[w];
    const long long at = static_cast<long long>(later - grp.first[w]) * kChunk;
    if (at + kChunk <= item.n && grp.wide[w]) {
      prefetch_l2(static_cast<const float*>(item.g) + at, kChunk * 4);
      prefetch_l2(static_cast<const float*>(item.p) + at, kChunk * 4);
      prefetch_l2(static_cast<const uint8_t*>(item.mu) + at, kChunk);
      prefetch_l2(static_cast<const uint8_t*>(item.nu) + at, kChunk);
    }
  }
  Block8 in;
  in.mu_most = *mu_most;
  in.nu_most = *nu_most;
  if (fast) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = j * 32 + lane;
      in.g[j] = reinterpret_cast<const float4*>(g)[i];
      in.p[j] = reinterpret_cast<const float4*>(p)[i];
      in.mu[j] = reinterpret_cast<const uint32_t*>(mu)[i];
      in.nu[j] = reinterpret_cast<const uint32_t*>(nu)[i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // (what lies behind the end counts as zero: it stays out of the largest)
      in.mu[j] = in.nu[j] = 0;
      float gs[4], ps[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = j * 128 + lane * 4 + q;
        gs[q] = i < n ? g[i] : 0.f;
        ps[q] = i < n ? p[i] : 0.f;
        in.mu[j] |= (i < n ? mu[i] : 0u) << (8 * q);
        in.nu[j] |= (i < n ? nu[i] : 0u) << (8 * q);
      }
      in.g[j] = make_float4(gs[0], gs[1], gs[2], gs[3]);
      in.p[j] = make_float4(ps[0], ps[1], ps[2], ps[3]);
    }
  }
  const float clip = grp.clip_scale != nullptr ? *grp.clip_scale : 1.f;
  const Result8 r = step8(grp.h, clip, in, grp.h.noise_key + static_cast<uint32_t>(begin), lane);
  if (lane == 0) {  // (every lane has read the old scales: the reduction is behind the reads)
    *mu_most = __uint_as_float(r.mu_most);
    *nu_most = __uint_as_float(r.nu_most);
  }
  if (fast) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int i = j * 32 + lane;
      const float4 pv = make_float4(r.p[2 * j].x, r.p[2 * j].y, r.p[2 * j + 1].x, r.p[2 * j + 1].y);
      reinterpret_cast<float4*>(p)[i] = pv;
      reinterpret_cast<uint32_t*>(mu)[i] = r.mu[2 * j] | (r.mu[2 * j + 1] << 16);
      reinterpret_cast<uint32_t*>(nu)[i] = r.nu[2 * j] | (r.nu[2 * j + 1] << 16);
      if (out != nullptr) reinterpret_cast<uint2*>(out)[i] = pack_bf16(pv);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int i = (j >> 1) * 128 + lane * 4 + (j & 1) * 2 + q;
      if (i >= n) continue;
      const float v = q ? r.p[j].y : r.p[j].x;
      p[i] = v;
      mu[i] = static_cast<uint8_t>(r.mu[j] >> (8 * q));
      nu[i] = static_cast<uint8_t>(r.nu[j] >> (8 * q));
      if (out != nullptr) out[i] = __float2bfloat16(v);
    }
  }
}

// ---- global norm ----

// Sum of squares of every gridDim.x-th span of chunks, in 64 bits (the factor scales every gradient: it
// is the one that exact arithmetic gives, rounded once), from the last span to the first: the step that
// follows begins with those that were read last and are still in L2. A CTA's spans and the order of
// all sums depend on the grid alone. With `clip_out` the CTA that arrives last adds the partial sums of
// this and the earlier launches of the call and stores min(1, max_norm / (norm + 1e-16)).
template <int kItems>
__global__ void __launch_bounds__(kThreads)
    sumsq_group_kernel(const __grid_constant__ GroupNorm<kItems> grp, unsigned chunks, double* partial,
                       int partial_first, unsigned* arrived, float max_norm, float* clip_out) {
  __shared__ double s_sum[kThreads / 32];
  __shared__ bool s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum = 0.0, more = 0.0;
  const unsigned spans = (chunks + kSpan - 1) / kSpan;
  for (unsigned at = blockIdx.x; at < spans; at += gridDim.x) {
    unsigned chunk = (spans - 1 - at) * kSpan;
    const unsigned end = chunk + kSpan < chunks ? chunk + kSpan : chunks;
    int which = find_item(grp, chunk);
    while (chunk < end) {
      while (which + 1 < grp.count && grp.first[which + 1] <= chunk) ++which;
      const unsigned behind = which + 1 < grp.count && grp.first[which + 1] < end ? grp.first[which + 1] : end;
      const long long begin = static_cast<long long>(chunk - grp.first[which]) * kChunk;
      const long long left = grp.item[which].n - begin;
      const int n = static_cast<int>(left < (behind - chunk) * kChunk ? left : (behind - chunk) * kChunk);
      const float* g = static_cast<const float*>(grp.item[which].g) + begin;
      if (n == kSpan * kChunk && grp.wide[which]) {
#pragma unroll
        for (int k = 0; k < kSpan * kChunk / (4 * kThreads); ++k) {
          const float4 v = reinterpret_cast<const float4*>(g)[k * kThreads + threadIdx.x];
          const double x = v.x, y = v.y, z = v.z, w = v.w;
          sum = fma(x, x, sum);
          more = fma(y, y, more);
          sum = fma(z, z, sum);
          more = fma(w, w, more);
        }
      } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const double x = g[i];
          sum = fma(x, x, sum);
        }
      }
      chunk = behind;
    }
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
  sum = block_sum(sum + more);
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
    const double f = static_cast<double>(max_norm) / (sqrt(total) + 1e-16);
    *clip_out = static_cast<float>(f > 1.0 ? 1.0 : f);  // (NaN stays)
  }
}

// Fills `grp` with items [from, ...) up to its capacity; returns how many it took and the chunks.
template <typename Item, int kItems>
int fill(Group<Item, kItems>& grp, const t5x_adamw_item* items, int from, int count, unsigned* chunks) {
  grp.count = 0;
  unsigned long long c = 0;
  int i = from;
  for (; i < count && grp.count < kItems; ++i) {
    const unsigned long long need = (static_cast<unsigned long long>(items[i].n) + kChunk - 1) / kChunk;
    if (need == 0) continue;
    if (c + need > 0x7fffffffull) break;
    grp.first[grp.count] = static_cast<unsigned>(c);
    grp.wide[grp.count] = takes_wide(items[i]);
    grp.item[grp.count++] = Item::of(items[i]);
    c += need;
  }
  grp.shift = 0;
  while ((c >> grp.shift) >= kHints) ++grp.shift;
  for (int k = 0, at = 0; k <= kHints; ++k) {
    const unsigned long long chunk_k = static_cast<unsigned long long>(k) << grp.shift;
    while (at + 1 < grp.count && grp.first[at + 1] <= chunk_k) ++at;
    grp.near[k] = static_cast<unsigned short>(at);
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
void launch(const Group32<kItems>& grp, unsigned chunks, cudaStream_t st) {
  adamw_group_kernel<kItems><<<chunks, kThreads, 0, st>>>(grp);
}
template <int kItems>
void launch(const Group8<kItems>& grp, unsigned chunks, cudaStream_t st) {
  adamw8_group_kernel<kItems><<<chunks, kThreads, 0, st>>>(grp);
}

template <typename Items>
void step_in_groups(const t5x_adamw_item* items, int count, const Hyper& h, const float* clip_scale,
                    cudaStream_t st) {
  Items grp;
  grp.h = h;
  grp.clip_scale = clip_scale;
  grp.ahead = static_cast<unsigned>(num_sms()) * 4;
  for (int from = 0; from < count;) {
    unsigned chunks;
    from += fill(grp, items, from, count, &chunks);
    if (chunks == 0) continue;
    launch(grp, chunks, st);
    count_launches(1);
  }
}

template <int kItems>
int sumsq_in_groups(const t5x_adamw_item* items, int count, void* scratch, float max_norm, float* clip,
                    cudaStream_t st) {
  GroupNorm<kItems> grp;
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
    const unsigned spans = (chunks + kSpan - 1) / kSpan;
    const unsigned grid = spans == 0 ? 1 : (spans < cap ? spans : cap);
    sumsq_group_kernel<kItems><<<grid, kThreads, 0, st>>>(grp, chunks, partial, first, arrived, max_norm,
                                                          last ? clip : nullptr);
    count_launches(1);
    first += static_cast<int>(grid);
  } while (from < count);
  return 0;
}

int launches_for(int count) { return count <= kMaxNorms ? 1 : (count + kMaxNorms - 1) / kMaxNorms; }

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
    sumsq_in_groups<kMaxNorms>(items, count, scratch, max_norm, clip, st);
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
  h.one = 1.f;
  h.ibc2 = 1.f / h.bc2;
  h.lr_bc1 = -lr / h.bc1;
  h.lr_decay = -lr * weight_decay;
  h.noise_key = seed * kNoise1 + static_cast<unsigned>(step) * 0xBB67AE85u;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const float* cs = static_cast<const float*>(clip_scale);
  if (state_bits == 32 && count <= kFewItems)
    step_in_groups<Group32<kFewItems>>(items, count, h, cs, st);
  else if (state_bits == 32)
    step_in_groups<Group32<kMaxItems>>(items, count, h, cs, st);
  else if (count <= kFewItems)
    step_in_groups<Group8<kFewItems>>(items, count, h, cs, st);
  else
    step_in_groups<Group8<kMaxItems8>>(items, count, h, cs, st);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error("adamw_group: %s", cudaGetErrorString(e));
  return 0;
}
