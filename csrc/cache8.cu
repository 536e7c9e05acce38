// Writing to a cache held in 8 bits: tokens appended, and the tokens that got most attention moved into a smaller one.
#include <algorithm>

#include "cache8.cuh"
#include "t5x_ops.h"

namespace t5x {
namespace {

// ---------------------------------------------------------------------------
// Append. A CTA takes one block of one head, its keys or its values. The block's largest absolute value grows to that
// of the new tokens; the codes that are there are rounded again, relative to it, so that each block keeps one scale.
// ---------------------------------------------------------------------------
constexpr int kAppendThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads)
    cache8_append_kernel(const __grid_constant__ Cache8 c, const __grid_constant__ NewTokens<T> n) {
  __shared__ uint32_t s_most[kAppendThreads / 32];
  const int what = blockIdx.x & 1, b = blockIdx.z, h = blockIdx.y;
  chain_release();  // (an attention behind this waits for what it reads of it)
  const int start = held_of(c, b);
  const int fresh = n.lengths == nullptr ? n.count : min(max(n.lengths[b], 0), n.count);
  const int blk = (start >> c.block_log2) + static_cast<int>(blockIdx.x >> 1);
  if (blk >= c.slots >> c.block_log2) return;
  const int first = blk << c.block_log2;
  const int lo = max(start, first);
  const int hi = static_cast<int>(min(min(static_cast<long long>(start) + fresh, static_cast<long long>(first) + (1 << c.block_log2)),
                                      static_cast<long long>(c.slots)));
  if (lo < hi) append_block<T, D, kAppendThreads>(c, n, what, b, h, start, lo, hi, threadIdx.x, s_most);
}

// ---------------------------------------------------------------------------
// Eviction: which slots stay.
// ---------------------------------------------------------------------------
constexpr int kSelectThreads = 1024;

// Order of weights as unsigned numbers: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (!(w == w)) return 0xffffffffu;
  uint32_t u = __float_as_uint(w);
  if (u == 0x80000000u) u = 0;
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int block_scan(int v, int* s_sums) {  // sum over the threads before; leaves the total in s_sums[32]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += u;
  }
  __syncthreads();
  if (lane == 31) s_sums[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    const int w = s_sums[lane];
    int run = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    s_sums[lane] = run - w;
    if (lane == 31) s_sums[32] = run;
  }
  __syncthreads();
  return sum - v + s_sums[warp];
}

// A CTA takes the slots of one head of one row: the border weight digit by digit from counts, then a walk in order.
__global__ void __launch_bounds__(kSelectThreads)
    cache8_select_kernel(const __grid_constant__ Cache8 c, int keep, int recent, int* __restrict__ kept) {
  __shared__ int s_count[256];
  __shared__ int s_sums[33];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const long long bh = blockIdx.x;
  const int b = static_cast<int>(bh / c.heads);
  const int held = held_of(c, b);
  const float* w = c.weight + bh * c.slots;
  int* out = kept + bh * keep;
  if (held <= keep) {
    for (int i = threadIdx.x; i < keep; i += kSelectThreads) out[i] = i < held ? i : -1;
    return;
  }
  const int old = held - recent;  // the slots to choose from
  if (threadIdx.x == 0) {
    s_prefix = 0;
    s_need = keep - recent;
  }
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (threadIdx.x < 256) s_count[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix;
    const int need = s_need;
    for (int i = threadIdx.x; i < old; i += kSelectThreads) {
      const uint32_t u = order_of(w[i]);
      if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_count[(u >> shift) & 255], 1);
    }
    __syncthreads();
    // the digit at which `need` of the largest are reached
    if (threadIdx.x == 0) {
      int above = 0, d = 255;
      while (d > 0 && above + s_count[d] < need) above += s_count[d--];
      s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
      s_need = need - above;
    }
    __syncthreads();
  }
  const uint32_t border = s_prefix;
  const int ties = s_need;  // of the slots at the border, the first so many stay
  int at = 0, seen = 0;
  for (int i0 = 0; i0 < held; i0 += kSelectThreads) {
    const int i = i0 + threadIdx.x;
    const uint32_t u = i < old ? order_of(w[i]) : 0;
    const bool tie = i < old && u == border && keep > recent;
    const int before = block_scan(tie, s_sums) + seen;
    seen += s_sums[32];
    const bool stays = i < held && (i >= old || (keep > recent && u > border) || (tie && before < ties));
    const int place = block_scan(stays, s_sums) + at;
    at += s_sums[32];
    if (stays) out[place] = i;
  }
}

// A CTA takes one block of one head of the smaller cache.
constexpr int kMoveThreads = 128;

__global__ void __launch_bounds__(kMoveThreads)
    cache8_move_kernel(const __grid_constant__ Cache8 c, const __grid_constant__ Cache8 to, int keep, const int* __restrict__ kept, int* __restrict__ index_out,
                       int* __restrict__ dropped_out) {
  const int b = blockIdx.z, h = blockIdx.y, blk = blockIdx.x;
  const int held = held_of(c, b), n = min(held, keep);
  if (h == 0 && blk == 0 && threadIdx.x == 0) {
    index_out[b] = n;
    dropped_out[b] = (c.position != nullptr ? c.dropped[b] : 0) +
                     (max(c.index[static_cast<long long>(b) * c.index_stride], 0) - n);
  }
  const int block = 1 << to.block_log2;
  const int lo = blk << to.block_log2, hi = min(lo + block, n);
  if (lo >= hi) return;
  const long long bh = static_cast<long long>(b) * c.heads + h;
  const int* from = kept + bh * keep;
  const int dim = c.dim;
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    const float* absmax = c.absmax[what] + bh * (c.slots >> c.block_log2);
    uint32_t most = 0;
    for (int i = lo + (threadIdx.x & 31); i < hi; i += 32) most = max(most, abs_bits(absmax[from[i] >> c.block_log2]));
    most = __reduce_max_sync(0xffffffffu, most);
    const float a = __uint_as_float(most);
    if (threadIdx.x == 0) to.absmax[what][bh * (to.slots >> to.block_log2) + blk] = a;
    const int8_t* src = c.codes[what] + bh * c.slots * dim;
    int8_t* dst = to.codes[what] + bh * to.slots * dim;
    const int words = dim / 4;
    for (int i = threadIdx.x; i < (hi - lo) * words; i += kMoveThreads) {
      const int tok = lo + i / words, d = i % words;
      const int s = from[tok];
      const float before = absmax[s >> c.block_log2];
      char4 v = reinterpret_cast<const char4*>(src + static_cast<long long>(s) * dim)[d];
      if (abs_bits(before) != most) {
        const Coder again(before, a);
        v = make_char4(again(v.x), again(v.y), again(v.z), again(v.w));
      }
      reinterpret_cast<char4*>(dst + static_cast<long long>(tok) * dim)[d] = v;
    }
  }
  for (int i = lo + threadIdx.x; i < hi; i += kMoveThreads) {
    const int s = from[i];
    to.weight[bh * to.slots + i] = c.weight[bh * c.slots + s];
    to.position[bh * to.slots + i] = c.position != nullptr ? c.position[bh * c.slots + s] : s;
  }
}

}  // namespace

// What every entry asks of a cache.
int check_cache8(const char* what, const Cache8& c) {
  if (c.batch < 0 || c.heads < 1 || c.slots < 1 || (c.dim != 64 && c.dim != 128))
    return set_error("%s: a cache of %d rows, %d heads, %d slots, %d channels (64 or 128)", what, c.batch, c.heads, c.slots,
                     c.dim);
  if (c.block_log2 < 4 || c.block_log2 > 7 || c.slots % (1 << c.block_log2) != 0)
    return set_error("%s: blocks of 2^%d tokens (16 to 128) over %d slots", what, c.block_log2, c.slots);
  if (c.heads > 65535 || c.batch > 65535) return set_error("%s: over 65535 rows or heads", what);
  if (!aligned_to(16, {c.codes[0], c.codes[1]}) ||
      !aligned_to(4, {c.absmax[0], c.absmax[1], c.index, c.weight, c.position, c.dropped}))
    return set_error("%s: codes must lie at multiples of 16 bytes, the others at multiples of 4", what);
  if (!c.codes[0] || !c.codes[1] || !c.absmax[0] || !c.absmax[1] || !c.index || (c.position && !c.dropped))
    return set_error("%s: null pointer", what);
  return 0;
}

Cache8 make_cache8(const T5xCache8* in) {
  Cache8 c;
  for (int i = 0; i < 2; ++i) {
    c.codes[i] = static_cast<int8_t*>(in->codes[i]);
    c.absmax[i] = static_cast<float*>(in->absmax[i]);
  }
  c.index = static_cast<const int*>(in->index);
  c.index_stride = in->index_stride;
  c.weight = static_cast<float*>(in->weight);
  c.position = static_cast<int*>(in->position);
  c.dropped = static_cast<const int*>(in->dropped);
  c.batch = in->batch;
  c.heads = in->heads;
  c.slots = in->slots;
  c.dim = in->dim;
  c.block_log2 = in->block_log2;
  return c;
}

namespace {

template <typename T>
int launch_append(const Cache8& c, const T5xNewTokens* in, cudaStream_t stream) {
  const NewTokens<T> n = make_tokens<T>(in);
  const int block = 1 << c.block_log2;
  const long long touched = std::min((static_cast<long long>(n.count) + block - 2) / block + 1,
                                     static_cast<long long>(c.slots >> c.block_log2));
  const dim3 grid(2 * static_cast<unsigned>(touched), c.heads, c.batch);
  if (c.dim == 64) cache8_append_kernel<T, 64><<<grid, kAppendThreads, 0, stream>>>(c, n);
  else cache8_append_kernel<T, 128><<<grid, kAppendThreads, 0, stream>>>(c, n);
  count_launches(1);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : set_error("cache8_append launch: %s", cudaGetErrorString(e));
}

}  // namespace

int check_new_tokens(const char* what, const T5xNewTokens* n) {
  if (n->count < 1 || n->type < 0 || n->type > 2) return set_error("%s: %d tokens of type %d", what, n->count, n->type);
  const int bytes = n->type == 2 ? 4 : 2;
  if (!n->x[0] || !n->x[1] || !aligned_to(bytes, {n->x[0], n->x[1]}) || !aligned_to(4, {n->lengths}))
    return set_error("%s: new tokens at a null or misaligned pointer", what);
  return 0;
}

int cache8_append(const Cache8& c, const T5xNewTokens* n, cudaStream_t stream) {
  switch (n->type) {
    case 0: return launch_append<__nv_bfloat16>(c, n, stream);
    case 1: return launch_append<__half>(c, n, stream);
    default: return launch_append<float>(c, n, stream);
  }
}

}  // namespace t5x

T5X_API int t5x_cache8_append(const T5xCache8* cache, const T5xNewTokens* tokens, void* stream) {
  if (!cache || !tokens) return t5x::set_error("cache8_append: null pointer");
  const t5x::Cache8 c = t5x::make_cache8(cache);
  if (int e = t5x::check_cache8("cache8_append", c)) return e;
  if (int e = t5x::check_new_tokens("cache8_append", tokens)) return e;
  if (c.batch == 0) return 0;
  return t5x::cache8_append(c, tokens, static_cast<cudaStream_t>(stream));
}

T5X_API int t5x_cache8_evict(const T5xCache8* cache, const T5xCache8* into, int keep, int recent, void* kept,
                             void* index_out, void* dropped_out, void* stream) {
  if (!cache || !into || !kept || !index_out || !dropped_out) return t5x::set_error("cache8_evict: null pointer");
  const t5x::Cache8 c = t5x::make_cache8(cache), to = t5x::make_cache8(into);
  if (int e = t5x::check_cache8("cache8_evict", c)) return e;
  if (int e = t5x::check_cache8("cache8_evict", to)) return e;
  if (!c.weight || !to.weight || !to.position) return t5x::set_error("cache8_evict: weights and positions are needed");
  if (to.batch != c.batch || to.heads != c.heads || to.dim != c.dim || keep < 1 || keep > to.slots || recent < 0 ||
      recent > keep || !t5x::aligned_to(4, {kept, index_out, dropped_out}))
    return t5x::set_error("cache8_evict: %d of %d slots (the last %d) do not fit %d", keep, c.slots, recent, to.slots);
  if (c.batch == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  t5x::cache8_select_kernel<<<static_cast<unsigned>(c.batch) * c.heads, t5x::kSelectThreads, 0, st>>>(
      c, keep, recent, static_cast<int*>(kept));
  const int blocks = (keep + (1 << to.block_log2) - 1) >> to.block_log2;
  t5x::cache8_move_kernel<<<dim3(blocks, c.heads, c.batch), t5x::kMoveThreads, 0, st>>>(
      c, to, keep, static_cast<const int*>(kept), static_cast<int*>(index_out), static_cast<int*>(dropped_out));
  t5x::count_launches(2);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : t5x::set_error("cache8_evict launch: %s", cudaGetErrorString(e));
}
