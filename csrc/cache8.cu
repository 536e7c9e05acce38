// Writing to a cache held in 8 bits: tokens appended, and the tokens that got most attention moved into a smaller one.
#include <algorithm>

#include "cache8.cuh"
#include "t5x_ops.h"

namespace t5x {
namespace {

// ---------------------------------------------------------------------------
// Append. A CTA takes one block of one head, its keys or its values. The block's largest absolute value grows to that
// of the new tokens; the codes that are there are rounded again, relative to it, so that each block keeps one scale. The
// latency of dependent reads bounds it: by itself from a cold L2 11 us for one token of 64 heads, 14 for 125 tokens of 8, most of
// which the attention behind it begins in.
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
// Eviction: the tokens that stay. A warp takes up to 32 tokens of one block of one head of the smaller cache.
// Tokens of a new block come from many old ones, so nearly all codes are rounded again, 16 at a time: as numbers (a byte under
// the exponent of 2^23), times the ratio of the scales, back under the exponent of 3 * 2^22, which rounds to whole numbers. Near a
// border between two codes as Coder does it. 64 heads of 128 channels, 4096 tokens each: 33 us for 137 MB, 4.2 TB/s; a warp waits for
// tokens that lie apart 53 % of its time. (With scales of 16 bits. With a 32-bit
// model's, where codes near a border are looked at, the whole eviction takes 96 instead of 62.)
// Keys and values requested together were no faster.
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 128;

__device__ __forceinline__ float code_number(uint32_t w, int i) {
  return __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7440 + i)) - 8388736.f;
}
// with short scales (Coder)
__device__ __forceinline__ uint32_t round_four(uint32_t w, float ratio) {
  const uint32_t u = w ^ 0x80808080u;
  const uint64_t less = pair_of(-8388736.f, -8388736.f), by = pair_of(ratio, ratio);
  auto two = [&](int i) {
    return codes_of_two(add2(pair_of(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + i)),
                                     __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441 + i))), less), by);
  };
  return low_bytes(two(0), two(2));
}
// with any; off: how far a quotient is from its code
__device__ __forceinline__ uint32_t round_four(uint32_t w, float ratio, float& off) {
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = code_number(w, i) * ratio, up = q + 12582912.f;
    off = fmaxf(off, fabsf(q - (up - 12582912.f)));
    r[i] = __float_as_uint(up);
  }
  return low_bytes(r);
}

__device__ __forceinline__ uint32_t round_four_exactly(uint32_t w, const Coder& again) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r |= static_cast<uint32_t>(again.of<true>(static_cast<float>(static_cast<int8_t>(w >> (8 * i)))) & 0xff) << (8 * i);
  return r;
}

// What a token's codes go through: their scale is the block's (kAsIs), else times the ratio of the two.
constexpr float kAsIs = -1.f, kByCoder = -2.f;
__device__ __forceinline__ float ratio_of(float old, float a) {
  if (abs_bits(old) == abs_bits(a)) return kAsIs;
  return a >= 0x1p-60f && a <= 0x1p100f ? __fdiv_rn(old, a) : kByCoder;
}

__device__ __forceinline__ int span_of(const Cache8& to) { return min(1 << to.block_log2, 32); }  // tokens of a warp

// Tokens lo on, of the n that stay.
template <int D>
__device__ __forceinline__ void move_span(const Cache8& c, const Cache8& to, int keep, const int* kept, int b, int h, int lo, int n) {
  constexpr int L = D / 16, kTokens = 32 / L, U = 4;  // lanes a token, tokens at a time, turns requested at a time
  const int lane = threadIdx.x & 31;
  const int block = 1 << to.block_log2, span = span_of(to);
  const int first = lo & ~(block - 1), count = min(block, n - first), mine = min(span, n - lo);
  const long long bh = static_cast<long long>(b) * c.heads + h;
  const int* from = kept + bh * keep + first;

  // the block's scale; lane i's token is lo + i
  int slot = 0;
  float old[2] = {0.f, 0.f};
  uint32_t most[2] = {0, 0}, bits[2] = {0, 0};
  for (int j0 = 0; j0 < count; j0 += 32) {
    const int j = j0 + lane;
    const int s = j < count ? __ldcg(from + j) : 0;
#pragma unroll
    for (int what = 0; what < 2; ++what) {
      const float x = j < count ? c.absmax[what][bh * (c.slots >> c.block_log2) + (s >> c.block_log2)] : 0.f;
      most[what] = max(most[what], abs_bits(x));
      bits[what] |= abs_bits(x);
      if (j0 == ((lo - first) & ~31)) old[what] = x;
    }
    if (j0 == ((lo - first) & ~31)) slot = s;
  }
  float a[2], ratio[2];
  bool brief[2];
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    a[what] = __uint_as_float(__reduce_max_sync(0xffffffffu, most[what]));
    brief[what] = (__reduce_or_sync(0xffffffffu, bits[what]) & 0x1fffu) == 0;
    ratio[what] = ratio_of(old[what], a[what]);
    if (lo == first && lane == 0) to.absmax[what][bh * (to.slots >> to.block_log2) + (first >> to.block_log2)] = a[what];
  }
  if (lane < mine) {
    to.weight[bh * to.slots + lo + lane] = c.weight[bh * c.slots + slot];
    to.position[bh * to.slots + lo + lane] = c.position != nullptr ? c.position[bh * c.slots + slot] : slot;
  }

  const int tok = lane / L, part = lane % L;
#pragma unroll
  for (int what = 0; what < 2; ++what) {
    const int8_t* src = c.codes[what] + bh * c.slots * D + 16 * part;
    int8_t* dst = to.codes[what] + (bh * to.slots + lo) * D + 16 * part;
    for (int i0 = 0; i0 < mine; i0 += U * kTokens) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kTokens + tok, s = __shfl_sync(0xffffffffu, slot, i & 31);
        if (i < mine) v[u] = *reinterpret_cast<const uint4*>(src + static_cast<long long>(s) * D);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kTokens + tok;
        const float r = __shfl_sync(0xffffffffu, ratio[what], i & 31), before = __shfl_sync(0xffffffffu, old[what], i & 31);
        if (i >= mine) continue;
        uint4 o = v[u];
        if (r != kAsIs) {
          float off = 0.f;
          if (brief[what] && r != kByCoder) {
            o = make_uint4(round_four(o.x, r), round_four(o.y, r), round_four(o.z, r), round_four(o.w, r));
          } else {
            o = make_uint4(round_four(o.x, r, off), round_four(o.y, r, off), round_four(o.z, r, off), round_four(o.w, r, off));
            if (r == kByCoder || off >= 0.4999f) {
              const Coder again(before, a[what]);
              o = make_uint4(round_four_exactly(v[u].x, again), round_four_exactly(v[u].y, again),
                             round_four_exactly(v[u].z, again), round_four_exactly(v[u].w, again));
            }
          }
        }
        *reinterpret_cast<uint4*>(dst + i * D) = o;
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kMoveThreads)
    cache8_move_kernel(const __grid_constant__ Cache8 c, const __grid_constant__ Cache8 to, int keep,
                       const int* __restrict__ kept) {
  const int b = blockIdx.z, lo = (blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5)) * span_of(to);
  const int n = min(held_of(c, b), keep);
  chain_wait();
  if (lo < n) move_span<D>(c, to, keep, kept, b, blockIdx.y, lo, n);
}

// ---------------------------------------------------------------------------
// Eviction: which slots stay.
// ---------------------------------------------------------------------------
// Order of weights as unsigned numbers: NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  if (!(w == w)) return 0xffffffffu;
  uint32_t u = __float_as_uint(w);
  if (u == 0x80000000u) u = 0;
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}

// Of the counts of 256 digits the one at which `need` of the largest are reached; need less those above it. By a warp.
__device__ __forceinline__ int border_digit(const int* counts, int& need) {
  const int lane = threadIdx.x & 31, top = 255 - 8 * lane;  // this lane's digits: top .. top - 7
  int mine[8], sum = 0;
  const int4 high = reinterpret_cast<const int4*>(counts)[63 - 2 * lane], low = reinterpret_cast<const int4*>(counts)[62 - 2 * lane];
  mine[0] = high.w, mine[1] = high.z, mine[2] = high.y, mine[3] = high.x;
  mine[4] = low.w, mine[5] = low.z, mine[6] = low.y, mine[7] = low.x;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += mine[i];
  int run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += u;
  }
  const int who = __ffs(__ballot_sync(0xffffffffu, run >= need)) - 1;  // (there are so many: the last lane has all)
  int above = run - sum, digit = top;
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (digit == top - i && above + mine[i] < need) above += mine[i], --digit;
  need -= __shfl_sync(0xffffffffu, above, who & 31);
  return __shfl_sync(0xffffffffu, digit, who & 31);
}

__device__ __forceinline__ int remote_int(const int* mine, uint32_t cta) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(mine), cta)) : "memory");
  return v;
}

__device__ __forceinline__ void remote_add(int* mine, int v) {  // to the cluster's first CTA
  asm volatile("red.relaxed.cluster.shared::cluster.add.s32 [%0], %1;" ::"r"(mapa_shared(smem_u32(mine), 0)), "r"(v) : "memory");
}

// A CTA, or a cluster, takes the slots of one head of one row and keeps its weights in registers, K adjacent ones a thread
// (through shared memory, so that global reads are of whole lines). The border is found eight bits at a time from counts of
// the digits, behind the first of those alone that are at the border so far; zeros, which may be most, are counted apart.
// A slot's place is the number of larger ones before it, and of those at the border as far as they stay. 64 heads of up to
// 65536 slots: 29 us, 2.6 at the copy rate: a warp waits for memory 21 % of its time, at the cluster's seven meetings 17 %, for an
// instruction's result 17 %, and half of the issue slots are taken. (With ballots by slot, 32
// slots in the lanes of a warp, 50: four times the instructions. One digit for all: 20 more, the list behind it is long.)
constexpr uint32_t kZero = 0x80000000u;  // order_of(0); of no weight 0

template <int T, int K, int kCtas>
__device__ __forceinline__ void select_slots(const Cache8& c, int keep, int recent, int* kept, int* index_out, int* dropped_out) {
  constexpr int kWarps = T / 32;
  constexpr bool kCluster = kCtas > 1;
  static_assert(T * K < 65536, "two counts in 32 bits");
  __shared__ __align__(16) int s_hist[4][256];
  __shared__ __align__(16) uint32_t s_list[T * K];
  __shared__ int s_left;
  __shared__ __align__(16) int s_all[4][256];  // a cluster's sums, in its first CTA; here the copy that is looked at
  __shared__ uint32_t s_sums[kWarps];
  __shared__ int s_total;  // larger | at the border << 16
  const long long bh = blockIdx.x / kCtas;
  const uint32_t rank = kCluster ? cluster_ctarank() : 0;
  const int b = static_cast<int>(bh / c.heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int index = max(c.index[static_cast<long long>(b) * c.index_stride], 0), held = min(index, c.slots);
  const float* w = c.weight + bh * c.slots;
  int* out = kept + bh * keep;
  chain_release();
  if (bh == static_cast<long long>(b) * c.heads && rank == 0 && threadIdx.x == 0) {
    index_out[b] = min(held, keep);
    dropped_out[b] = (c.position != nullptr ? c.dropped[b] : 0) + (index - min(held, keep));
  }
  if (held <= keep) {
    for (int i = rank * T + threadIdx.x; i < keep; i += T * kCtas) out[i] = i < held ? i : -1;
    return;
  }
  const int old = held - recent, first = static_cast<int>(rank) * (T * K);  // slots to choose from; this CTA's first
  const int own = first + static_cast<int>(threadIdx.x) * K;                // this thread's first
  // 16 bytes a place, places of a thread's by its number: the banks
  auto place_of = [](int chunk) { return chunk ^ (chunk >> 3 & 7); };
  const bool whole = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
#pragma unroll
  for (int i = 0; i < K / 4; ++i) {
    const int chunk = i * T + threadIdx.x, s = first + 4 * chunk;  // (a cache has whole 16 slots)
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s < old) {
      if (whole) x = *reinterpret_cast<const float4*>(w + s);
      else x = make_float4(w[s], w[s + 1], w[s + 2], w[s + 3]);
    }
    reinterpret_cast<float4*>(s_list)[place_of(chunk)] = x;
  }
  for (int i = threadIdx.x; i < 1024; i += T) s_hist[i >> 8][i & 255] = s_all[i >> 8][i & 255] = 0;
  if (threadIdx.x == 0) s_left = 0;
  __syncthreads();
  uint32_t key[K];
#pragma unroll
  for (int i = 0; i < K / 4; ++i) {
    const float4 x = reinterpret_cast<const float4*>(s_list)[place_of(threadIdx.x * (K / 4) + i)];
    key[4 * i] = own + 4 * i < old ? order_of(x.x) : 0;
    key[4 * i + 1] = own + 4 * i + 1 < old ? order_of(x.y) : 0;
    key[4 * i + 2] = own + 4 * i + 2 < old ? order_of(x.z) : 0;
    key[4 * i + 3] = own + 4 * i + 3 < old ? order_of(x.w) : 0;
  }
  if (kCluster) cluster_sync_all();
  else __syncthreads();

  int need = keep - recent;
  const bool any = need > 0;
  uint32_t border = 0;
  if (any)
    for (int round = 0; round < 4; ++round) {
      const int shift = 24 - 8 * round;
      int zeros = 0;
      if (round == 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
          if (key[i] == kZero) ++zeros;
          else if (key[i] != 0) atomicAdd(&s_hist[0][key[i] >> 24], 1);
        }
      } else {
        for (int j = threadIdx.x; j < s_left; j += T) {
          const uint32_t u = s_list[j];
          if ((u ^ border) >> (shift + 8) != 0) continue;
          if (u == kZero) ++zeros;
          else atomicAdd(&s_hist[round][(u >> shift) & 255], 1);
        }
      }
      zeros = __reduce_add_sync(0xffffffffu, zeros);
      if (lane == 0 && zeros > 0) atomicAdd(&s_hist[round][(kZero >> shift) & 255], zeros);
      __syncthreads();
      if (kCluster) {  // the few digits that occur, to the first CTA
        for (int i = threadIdx.x; i < 256; i += T)
          if (s_hist[round][i] != 0) remote_add(&s_all[round][i], s_hist[round][i]);
        cluster_sync_all();
        for (int i = threadIdx.x; i < 256; i += T) s_hist[round][i] = remote_int(&s_all[round][i], 0);
        __syncthreads();
      }
      border |= static_cast<uint32_t>(border_digit(s_hist[round], need)) << shift;
      if (round == 0) {  // those at the border so far, in any order
        int mine = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) mine += key[i] != 0 && (key[i] ^ border) >> 24 == 0;
        int run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, run, o);
          if (lane >= o) run += u;
        }
        int at = 0;
        if (lane == 31 && run != 0) at = atomicAdd(&s_left, run);
        at = __shfl_sync(0xffffffffu, at, 31) + run - mine;
#pragma unroll
        for (int i = 0; i < K; ++i)
          if (key[i] != 0 && (key[i] ^ border) >> 24 == 0) s_list[at++] = key[i];
        __syncthreads();
      }
    }
  const int ties = need;  // of the slots at the border, the first so many stay

  uint32_t mine = 0;  // larger | at the border << 16
  if (any) {
#pragma unroll
    for (int i = 0; i < K; ++i) mine += key[i] > border ? 1u : key[i] == border && key[i] != 0 ? 0x10000u : 0u;
  }
  uint32_t run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += u;
  }
  if (lane == 31) s_sums[warp] = run;
  __syncthreads();
  uint32_t before = run - mine, all = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += s_sums[i];
    all += s_sums[i];
  }
  int above = before & 0xffff, tie = before >> 16;
  if (kCluster) {
    if (threadIdx.x == 0) s_total = static_cast<int>(all);
    cluster_sync_all();
#pragma unroll
    for (int r = 0; r < kCtas; ++r) {
      const uint32_t u = static_cast<uint32_t>(remote_int(&s_total, r));
      if (r < static_cast<int>(rank)) above += u & 0xffff, tie += u >> 16;
    }
  }
  if (any) {
    int* to = out + above + min(tie, ties);
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const bool at_border = key[i] == border && key[i] != 0;
      if (key[i] > border || (at_border && tie < ties)) *to++ = own + i;
      tie += at_border;
    }
  }
  for (int i = rank * T + threadIdx.x; i < recent; i += T * kCtas) out[keep - recent + i] = old + i;
  if (kCluster) cluster_sync_all();  // nobody leaves while others read its sums
}

template <int T, int K, int kCtas>
__global__ void __launch_bounds__(T, 1024 / T)
    cache8_select_kernel(const __grid_constant__ Cache8 c, int keep, int recent, int* __restrict__ kept,
                         int* __restrict__ index_out, int* __restrict__ dropped_out) {
  select_slots<T, K, kCtas>(c, keep, recent, kept, index_out, dropped_out);
}

// The choice and the move in one launch.
template <int T, int K, int D>
__global__ void __launch_bounds__(T, 1024 / T)
    cache8_evict_kernel(const __grid_constant__ Cache8 c, const __grid_constant__ Cache8 to, int keep, int recent,
                        int* kept, int* index_out, int* dropped_out) {
  const int b = blockIdx.x / c.heads, h = blockIdx.x - b * c.heads, n = min(held_of(c, b), keep), span = span_of(to);
  select_slots<T, K, 1>(c, keep, recent, kept, index_out, dropped_out);
  __syncthreads();
  for (int lo = (threadIdx.x >> 5) * span; lo < n; lo += T / 32 * span) move_span<D>(c, to, keep, kept, b, h, lo, n);
}

// Over more slots than a cluster's registers hold the weights are read once for each digit.
constexpr int kWalkThreads = 1024;

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

__global__ void __launch_bounds__(kWalkThreads)
    cache8_select_walk_kernel(const __grid_constant__ Cache8 c, int keep, int recent, int* __restrict__ kept,
                              int* __restrict__ index_out, int* __restrict__ dropped_out) {
  __shared__ int s_count[256];
  __shared__ int s_sums[33];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const long long bh = blockIdx.x;
  const int b = static_cast<int>(bh / c.heads);
  const int index = max(c.index[static_cast<long long>(b) * c.index_stride], 0), held = min(index, c.slots);
  const float* w = c.weight + bh * c.slots;
  int* out = kept + bh * keep;
  chain_release();
  if (bh == static_cast<long long>(b) * c.heads && threadIdx.x == 0) {
    index_out[b] = min(held, keep);
    dropped_out[b] = (c.position != nullptr ? c.dropped[b] : 0) + (index - min(held, keep));
  }
  if (held <= keep) {
    for (int i = threadIdx.x; i < keep; i += kWalkThreads) out[i] = i < held ? i : -1;
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
    for (int i = threadIdx.x; i < old; i += kWalkThreads) {
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
  for (int i0 = 0; i0 < held; i0 += kWalkThreads) {
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

template <int T, int K, int kCtas>
cudaError_t launch_select_by(const Cache8& c, int keep, int recent, int* kept, int* index_out, int* dropped_out,
                             cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(c.batch) * c.heads * kCtas);
  cfg.blockDim = dim3(T);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCtas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCtas > 1 ? 1 : 0;
  count_launches(1);
  return cudaLaunchKernelEx(&cfg, cache8_select_kernel<T, K, kCtas>, c, keep, recent, kept, index_out, dropped_out);
}

// The weights of a head in the registers of one CTA up to 2048 slots, of up to eight up to 65536. (64 heads, us with the move of
// 512 tokens: 2048 slots 14, 4096 17, 8192 21, 16384 27, 32768 40.)
cudaError_t launch_select(const Cache8& c, int keep, int recent, int* kept, int* index_out, int* dropped_out, cudaStream_t stream) {
  auto by = [&](auto launch) { return launch(c, keep, recent, kept, index_out, dropped_out, stream); };
  if (c.slots <= 2048) return by(launch_select_by<256, 8, 1>);
  if (c.slots <= 4096) return by(launch_select_by<256, 8, 2>);
  if (c.slots <= 8192) return by(launch_select_by<256, 8, 4>);
  if (c.slots <= 16384) return by(launch_select_by<256, 8, 8>);
  if (c.slots <= 65536) return by(launch_select_by<256, 32, 8>);
  cache8_select_walk_kernel<<<static_cast<unsigned>(c.batch) * c.heads, kWalkThreads, 0, stream>>>(c, keep, recent, kept, index_out,
                                                                                               dropped_out);
  count_launches(1);
  return cudaGetLastError();
}

// Both in one launch where a CTA makes the choice and has a turn of its warps to move, and all CTAs are there at a time (four an
// SM): the device takes as long, the host one launch less (11.7 to 10.3 a call). us so / in two: 12 heads of 64 channels, 640 -> 121 9.4 / 9.4,
// 2048 -> 256 10.4 / 9.8, -> 512 13.4 / 9.7; 512 heads of 64, 2048 -> 32 13.5 / 13.5, -> 256 20.9 / 21.9, of 128 16.1 / 16.2 and 27.3 /
// 27.5, -> 512 45 / 40; 640 heads of 128, -> 32 26.3 / 19.3, -> 256 39.4 / 37.3, 2048 heads 64 / 49 and 90 / 90.
bool in_one_launch(const Cache8& c, int keep) {
  return c.slots <= 2048 && keep <= 256 && static_cast<long long>(c.batch) * c.heads <= 4LL * num_sms();
}
template <int D>
cudaError_t launch_both(const Cache8& c, const Cache8& to, int keep, int recent, int* kept, int* index_out, int* dropped_out,
                        cudaStream_t stream) {
  cache8_evict_kernel<256, 8, D><<<static_cast<unsigned>(c.batch) * c.heads, 256, 0, stream>>>(c, to, keep, recent, kept, index_out,
                                                                                          dropped_out);
  count_launches(1);
  return cudaGetLastError();
}

// The tokens behind the choice: the kernel begins while that still runs, and waits for it by itself.
template <typename... Args>
cudaError_t launch_move(void (*kernel)(Args...), dim3 grid, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launches(1);
  return cudaLaunchKernelEx(&cfg, kernel, args...);
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
  int *slots = static_cast<int*>(kept), *index = static_cast<int*>(index_out), *dropped = static_cast<int*>(dropped_out);
  const bool both = t5x::in_one_launch(c, keep);
  cudaError_t e = !both          ? t5x::launch_select(c, keep, recent, slots, index, dropped, st)
                  : c.dim == 64 ? t5x::launch_both<64>(c, to, keep, recent, slots, index, dropped, st)
                                : t5x::launch_both<128>(c, to, keep, recent, slots, index, dropped, st);
  if (e == cudaSuccess && !both) {
    const int tokens = std::min(1 << to.block_log2, 32) * (t5x::kMoveThreads / 32);  // of a CTA
    const dim3 grid((keep + tokens - 1) / tokens, c.heads, c.batch);
    e = t5x::launch_move(c.dim == 64 ? t5x::cache8_move_kernel<64> : t5x::cache8_move_kernel<128>, grid, st, c, to, keep,
                         static_cast<const int*>(slots));
  }
  return e == cudaSuccess ? 0 : t5x::set_error("cache8_evict launch: %s", cudaGetErrorString(e));
}
