// A key/value cache held in 8 bits: the pieces that its kernels share.
//
// Codes are int8 [batch, head, slot, dim]; a block of tokens of one head shares the largest absolute value `a` of what
// it holds (fp32 [batch, head, slot / block]), and a code c stands for c * a / 127. Quotients are rounded once, from
// IEEE products and divisions that the build's fast-math flags do not reach, so a code does not depend on which
// kernel, or which statement in tensor operations, made it. A largest value that is not finite makes every value of
// its block NaN (0 * inf), and the codes 0.
#pragma once
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "t5x_ops.h"

namespace t5x {

struct Cache8 {
  int8_t* codes[2];      // keys, values
  float* absmax[2];
  const int* index;      // tokens held, by row (or one for all)
  int index_stride;      // 1, or 0
  float* weight;         // attention weight by slot [batch, head, slot], or null
  int* position;         // positions of the slots, or null (the slot is the position)
  const int* dropped;    // tokens evicted, by row; with `position`
  int batch, heads, slots, dim;
  int block_log2;
};

// Whether a number has at most 11 bits, as the values of 16-bit types have (and the largest of them).
__device__ __forceinline__ bool is_short(float x) { return (__float_as_uint(x) & 0x1fffu) == 0; }

// The code of u * num / a, rounded to the nearest whole number (ties to even), in a block of largest value a: of the value
// u with num = 127, of an older code u with num = the largest value it was relative to. u * (num / a) is at most 4e-5 off.
//
// Where u, num and a are short (a code is), a quotient that is not itself on a border between two codes is more than 2^-20 of
// itself away from it: with whole numbers U, N, A below 2^11 it is U N 2^-s / A, a border is (2 k + 1) / 2, and
// they differ by 2^-s / 2 A at least, 1 / (2 U N) of the quotient, where 127 or a code is the other factor. The product, two
// steps of 24 bits off at most, is brought to 21 bits first, which puts those on a border there and leaves the others on
// their side. Elsewhere a quotient near a border is taken in 64 bits, where it cannot round to the other side (u * num has
// 31 bits, a has 24: they differ by 2^-25 at least).
__device__ __forceinline__ float in_21_bits(float q) {
  const float high = __fmul_rn(q, 9.f);
  return __fsub_rn(high, __fsub_rn(high, q));
}

struct Coder {
  float num, a, factor;
  bool plain;  // a lies where neither the factor nor a product leaves the normal numbers
  bool brief;  // num and a are short; for u the caller knows

  __device__ __forceinline__ Coder(float num_, float a_) : num(num_), a(a_) {
    plain = a >= 0x1p-60f && a <= 0x1p100f;
    brief = plain && is_short(num) && is_short(a);
    factor = plain ? __fdiv_rn(num, a) : 0.f;
  }
  __device__ __noinline__ static int exactly(float u, float num, float a) {
    double x, y, z;  // (conversions that the build's flags do not let lose numbers below the normal ones)
    asm("cvt.f64.f32 %0, %1;" : "=d"(x) : "f"(u));
    asm("cvt.f64.f32 %0, %1;" : "=d"(y) : "f"(num));
    asm("cvt.f64.f32 %0, %1;" : "=d"(z) : "f"(a));
    const double q = x * y / z;
    return q == q ? __double2int_rn(fmin(fmax(q, -127.0), 127.0)) : 0;
  }
  // kShort: u is short
  template <bool kShort>
  __device__ __forceinline__ int of(float u) const {
    if (kShort && brief) return __float_as_int(in_21_bits(u * factor) + 12582912.f) - 0x4b400000;  // (3 * 2^22: steps of one)
    const float q = u * factor, r = rintf(q);
    if (!plain || fabsf(fabsf(q - r) - 0.5f) < 1e-4f) return exactly(u, num, a);
    return static_cast<int>(r);
  }
};

// Two numbers an instruction.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Codes of two short values (Coder), in the low byte of each half: quotients in 21 bits, then under the exponent of 3 * 2^22.
__device__ __forceinline__ uint64_t codes_of_two(uint64_t x, uint64_t factor) {
  const uint64_t minus = pair_of(-1.f, -1.f);
  const uint64_t q = mul2(x, factor), high = mul2(q, pair_of(9.f, 9.f)), rest = fma2(q, minus, high);
  return add2(fma2(rest, minus, high), pair_of(12582912.f, 12582912.f));
}
__device__ __forceinline__ uint32_t low_bytes(const uint32_t (&r)[4]) {
  return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}
__device__ __forceinline__ uint32_t low_bytes(uint64_t a, uint64_t b) {
  uint32_t r[4];
  asm("mov.b64 {%0, %1}, %2;" : "=r"(r[0]), "=r"(r[1]) : "l"(a));
  asm("mov.b64 {%0, %1}, %2;" : "=r"(r[2]), "=r"(r[3]) : "l"(b));
  return low_bytes(r);
}
// the two values of a word
template <typename T>
__device__ __forceinline__ uint64_t values_of(uint32_t w);
template <>
__device__ __forceinline__ uint64_t values_of<__nv_bfloat16>(uint32_t w) {
  return pair_of(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ uint64_t values_of<__half>(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return pair_of(f.x, f.y);
}

// NaN counts as larger than any number: the bits of |x| are ordered so
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }

// tokens that row b holds
__device__ __forceinline__ int held_of(const Cache8& c, int b) {
  return min(max(c.index[static_cast<long long>(b) * c.index_stride], 0), c.slots);
}

// New keys and values [batch, token, head, dim].
template <typename T>
struct NewTokens {
  const T* x[2];
  long long sb[2], st[2], sh[2];
  const int* lengths;  // tokens by row, or null: `count` each
  int count;
  int vec;             // four adjacent values may be loaded at a time
};

template <typename T>
__device__ __forceinline__ void load_four(const T* src, bool vec, float (&v)[4]) {
  alignas(4 * sizeof(T)) T in[4];
  if (vec) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(in) = *reinterpret_cast<const uint4*>(src);
    else *reinterpret_cast<uint2*>(in) = *reinterpret_cast<const uint2*>(src);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) in[i] = src[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_float(in[i]);
}

// Slots lo .. hi of one block of a (row, head), its keys (what = 0) or values, get the tokens from lo - start on. By THREADS
// threads, number `tid`, all of which call it, with s_most[THREADS / 32] of their own; all threads of the CTA meet in it.
template <typename T, int D, int THREADS>
__device__ __forceinline__ void append_block(const Cache8& c, const NewTokens<T>& n, int what, int b, int h, int start, int lo,
                                             int hi, int tid, uint32_t* s_most) {
  const long long bh = static_cast<long long>(b) * c.heads + h;
  const int blk = lo >> c.block_log2, first = blk << c.block_log2;
  const T* x = n.x[what] + b * n.sb[what] + h * n.sh[what];
  const long long st = n.st[what];
  int8_t* codes = c.codes[what] + bh * c.slots * D;
  float* absmax = c.absmax[what] + bh * (c.slots >> c.block_log2) + blk;
  constexpr int lanes = D / 4, step = THREADS / lanes;
  const int d = tid % lanes * 4, from = tid / lanes;
  const bool vec = n.vec != 0;

  const float before = lo > first ? __ldcg(absmax) : 0.f;
  uint32_t most = 0;
#pragma unroll 4
  for (int s = lo + from; s < hi; s += step) {
    float v[4];
    load_four(x + (s - start) * st + d, vec, v);
    most = max(max(most, max(abs_bits(v[0]), abs_bits(v[1]))), max(abs_bits(v[2]), abs_bits(v[3])));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if ((tid & 31) == 0) s_most[tid >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) most = max(most, s_most[w]);
  most = max(most, abs_bits(before));
  const float a = __uint_as_float(most);
  if (most != abs_bits(before) && lo > first) {
    const Coder again(before, a);
#pragma unroll 2
    for (int s = first + from; s < lo; s += step) {
      char4* at = reinterpret_cast<char4*>(codes + static_cast<long long>(s) * D + d);
      const char4 v = *at;
      *at = make_char4(again.of<true>(v.x), again.of<true>(v.y), again.of<true>(v.z), again.of<true>(v.w));
    }
  }
  constexpr bool kShort = sizeof(T) == 2;
  const Coder code(127.f, a);
#pragma unroll 2
  for (int s = lo + from; s < hi; s += step) {
    float v[4];
    load_four(x + (s - start) * st + d, vec, v);
    *reinterpret_cast<char4*>(codes + static_cast<long long>(s) * D + d) = make_char4(code.of<kShort>(v[0]), code.of<kShort>(v[1]), code.of<kShort>(v[2]),
                                                                                                 code.of<kShort>(v[3]));
  }
  if (what == 0)
    for (int s = lo + tid; s < hi; s += THREADS) {
      if (c.weight != nullptr) c.weight[bh * c.slots + s] = 0.f;
      if (c.position != nullptr) c.position[bh * c.slots + s] = s + c.dropped[b];
    }
  __syncthreads();  // everyone has read *absmax and s_most
  if (tid == 0) *absmax = a;
}

template <typename T>
NewTokens<T> make_tokens(const T5xNewTokens* in) {
  NewTokens<T> n = {};
  if (in == nullptr) return n;
  n.vec = 1;
  for (int i = 0; i < 2; ++i) {
    n.x[i] = static_cast<const T*>(in->x[i]);
    n.sb[i] = in->stride_batch[i];
    n.st[i] = in->stride_token[i];
    n.sh[i] = in->stride_head[i];
    if (!aligned_to(4 * sizeof(T), {in->x[i]}) || (n.sb[i] | n.st[i] | n.sh[i]) % 4 != 0) n.vec = 0;
  }
  n.lengths = static_cast<const int*>(in->lengths);
  n.count = in->count;
  return n;
}

Cache8 make_cache8(const T5xCache8* in);
int check_cache8(const char* what, const Cache8& c);  // 0, or set_error's
int check_new_tokens(const char* what, const T5xNewTokens* n);
int cache8_append(const Cache8& c, const T5xNewTokens* n, cudaStream_t stream);

}  // namespace t5x
