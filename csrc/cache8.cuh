// A key/value cache held in 8 bits: the pieces that its kernels share.
//
// Codes are int8 [batch, head, slot, dim]; a block of tokens of one head shares the largest absolute value `a` of what
// it holds (fp32 [batch, head, slot / block]), and a code c stands for c * a / 127. Quotients are rounded once, from
// IEEE products and divisions that the build's fast-math flags do not reach, so a code does not depend on which
// kernel, or which statement in tensor operations, made it. A largest value that is not finite makes every value of
// its block NaN (0 * inf), and the codes 0.
#pragma once
#include <cuda_fp16.h>

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

// The code of u * num / a, rounded to the nearest whole number (ties to even), in a block of largest value a: of the value
// u with num = 127, of an older code u with num = the largest value it was relative to. One multiplication by num / a is
// at most 4e-5 off; where that may decide, the quotient is taken in 64 bits, where it cannot round to the other side of
// a border (u * num has 31 bits, a has 24, so they differ by 2^-25 at least).
struct Coder {
  float num, a, factor;
  bool plain;  // a lies where neither the factor nor a product leaves the normal numbers

  __device__ __forceinline__ Coder(float num_, float a_) : num(num_), a(a_) {
    plain = a >= 0x1p-60f && a <= 0x1p100f;
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
  __device__ __forceinline__ int operator()(float u) const {
    const float q = u * factor, r = rintf(q);
    if (!plain || fabsf(fabsf(q - r) - 0.5f) < 1e-4f) return exactly(u, num, a);
    return static_cast<int>(r);
  }
};

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

Cache8 make_cache8(const T5xCache8* in);
int check_cache8(const char* what, const Cache8& c);  // 0, or set_error's
int check_new_tokens(const char* what, const T5xNewTokens* n);
int cache8_append(const Cache8& c, const T5xNewTokens* n, cudaStream_t stream);

}  // namespace t5x
