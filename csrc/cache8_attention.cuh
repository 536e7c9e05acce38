// What the kernels of attention over a cache in 8 bits share: the arguments of a call, the work's division into pieces, and
// the small operations on codes and fragments (cache8_attention.cu).
#pragma once
#include <utility>

#include "cache8.cuh"

namespace t5x {

constexpr int kMaxDistances = 1024;
constexpr int kMaxBatch = 2048;  // rows of one launch
constexpr int kMaxBiases = 8192;  // values of a bias table
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPeak = 7.f;     // exponent of a probability at the reference
constexpr float kLimit = 15.6f;  // of the largest: an fp16 number
constexpr float kNothing = -3e38f;  // the reference of a row that has seen nothing

struct Cache8Attn {
  Cache8 c;
  const void* q;
  void* out;
  const float* table;
  const uint8_t* mask;
  long long q_sb, q_st, q_sh, mask_stride;
  int table_stride, q_vec;  // q_vec: whole 16 bytes of a query may be loaded
  int count, group, rows;  // queries a row, heads a key head, their product
  int from_end;            // the first query's place, counted from the end of the tokens held: `count`, but for a part of them
  int out_heads;           // key heads of `out`, of which a launch may have a part
  int distances, mask_len, causal;
  int appended;            // tokens of this call behind c.index
  float scale;
  uint32_t low;            // 0x00ff00ff
  unsigned long long by_group;  // 2^32 / group, rounded up: r / group for r below 2^16 by one multiplication
  int pieces;              // that the tiles are cut into
  int row_warps;           // over many query rows: warps of a CTA that take different rows (2 or 4 of few rows, else 4 or 8)
  int least;               // cost of a piece at least, in tiles
  int entry;               // what beginning a (row, head) costs, in tiles
  float* part;             // [row tile, pieces, 2, rows of a tile, dim]
  float2* stats;           // [row tile, pieces, 2, rows of a tile]: reference, sum
  long long* first;        // [batch + 1]: cost in front of a row, in tiles; then that of a piece
  float* scores;           // [batch * heads, rows, slots], times log2 e, where weights are added up; else null
  float2* final_stats;     // [batch * heads, rows]: reference, 1 / sum; with scores
  uint8_t buckets[kMaxDistances];  // column of the bias table by distance
};

constexpr float kRest = 0x1p-11f;  // what the second number of a 32-bit probability counts: it stands above fp16's smallest

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c += a b, b one fp16 number or, of 32-bit operands, two: their sum, or (kApart) the second at 2^-11. Tensor cores cut what they add to an accumulator off, toward zero: over a long
// sum of 32-bit operands (two numbers) that would count more than they do, so theirs are added by an instruction that rounds.
template <int Q2, bool kApart = false>
__device__ __forceinline__ void mma_sum(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b0)[Q2], const uint32_t (&b1)[Q2]) {
  if (Q2 == 1) {
    mma_f16(c, a[0], a[1], a[2], a[3], b0[0], b1[0]);
  } else {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    mma_f16(x, a[0], a[1], a[2], a[3], b0[Q2 - 1], b1[Q2 - 1]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (kApart) x[k] *= kRest;
    mma_f16(x, a[0], a[1], a[2], a[3], b0[0], b1[0]);
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] += x[k];
  }
}
// The same with a the sum.
template <int Q2, bool kApart = false>
__device__ __forceinline__ void mma_sum(float (&c)[4], const uint4 (&a)[Q2], uint32_t b0, uint32_t b1) {
  if (Q2 == 1) {
    mma_f16(c, a[0].x, a[0].y, a[0].z, a[0].w, b0, b1);
  } else {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    mma_f16(x, a[Q2 - 1].x, a[Q2 - 1].y, a[Q2 - 1].z, a[Q2 - 1].w, b0, b1);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (kApart) x[k] *= kRest;
    mma_f16(x, a[0].x, a[0].y, a[0].z, a[0].w, b0, b1);
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] += x[k];
  }
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// (w & low) ^ kFlip in one instruction, with `low` = 0x00ff00ff in a register (the compiler makes two of two constants: the
// kernel reads it from its arguments)
template <uint32_t kFlip>
__device__ __forceinline__ uint32_t low_flipped(uint32_t w, uint32_t low) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(w), "r"(low), "n"(kFlip));
  return r;
}
// bytes 0 and 2 of codes as two numbers
__device__ __forceinline__ uint32_t number_pair(uint32_t w, uint32_t low) {
  return as_u32(__hsub2(as_half2(low_flipped<0x64806480u>(w, low)), as_half2(0x64806480u)));
}
__device__ __forceinline__ float log2_approx(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A probability of 32 bits is two fp16 numbers, the second 2^11 times what the first leaves.
__device__ __forceinline__ uint32_t rest_of(float lo, float hi, __half2 first) {
  return as_u32(__floats2half2_rn((lo - __low2float(first)) * (1.f / kRest), (hi - __high2float(first)) * (1.f / kRest)));
}

// ---- What the probabilities of a query row are relative to ----
//
// The sum that divides adds 2^(s - score). The product with the values takes 2^(s - score - scale) times the largest value of the
// token's block, so that one fp16 number holds both and the sums need no scaling by token. Each of the two is raised only where
// it would come to 2^kLimit, to where its largest is 2^kPeak (the scale to a power of two), and by what the row itself sees, so that
// neither what is hidden nor another row changes a result. Taking the scale of the product's largest term, not of the largest
// block, keeps a block of large values but next to no weight from costing the others their bits: below 2^-14 fp16 numbers are
// steps of 2^-24, at most 2^-30 of the largest term each.
struct Reference {
  float score;
  float by;  // 2^-scale, scale whole, -126 to 126
};
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
__device__ __forceinline__ int scale_of(const Reference& r) { return 127 - static_cast<int>(__float_as_uint(r.by) >> 23); }

// Whether a score of a block goes over a limit; a: the block's largest value, times r.by.
__device__ __forceinline__ bool beyond(const Reference& r, float s, float a) {
  return s - r.score > kLimit - fmaxf(log2_approx(a), 0.f);
}
// The reference of scores of which x is the row's largest here.
__device__ __forceinline__ float raised(const Reference& r, float x) { return x - r.score > kLimit ? x - kPeak : r.score; }
// score: what `raised` gave; term: the row's largest score here relative to that, with the logarithm of its block's largest value.
// (Differences alone: scores may be as large as the lowest masks, beside which a logarithm would vanish.) What the sum that divides and
// the other ones are multiplied by: 1 where nothing changes.
__device__ __forceinline__ float2 raise_to(Reference& r, float score, float term) {
  const float lower = r.score - score, old = lower + static_cast<float>(scale_of(r));  // where the sums are, relative to `score`
  const float scale = fminf(fmaxf(ceilf(term - old > kLimit ? term - kPeak : old), -126.f), 126.f);
  r.score = score;
  r.by = power_of_two(-static_cast<int>(scale));
  return make_float2(exp2_approx(lower), exp2_approx(old - scale));
}

// Where a block's largest value a, relative to the scale, is no factor that 32 bits hold a small probability beside (or no number):
// its part from 1 to 2 and its exponent, which goes into the scores.
constexpr float kFar = 0x1p60f;
__device__ __forceinline__ float2 part_of(const Reference& r, float a) {
  const uint32_t u = __float_as_uint(a);
  return make_float2(u < 0x00800000u ? 0.f : __uint_as_float((u & 0x007fffffu) | 0x3f800000u),
                     static_cast<float>(static_cast<int>(u >> 23) - 127 - scale_of(r)));
}
// A score, relative to the reference, then; of a block that is not finite NaN, unless it is hidden.
__device__ __forceinline__ float far_score(float s, float exponent, float a) {
  return s == -INFINITY ? s : s + exponent + (a - a);
}

__device__ __forceinline__ int token_of(const Cache8Attn& p, int r) { return static_cast<int>((r * p.by_group) >> 32); }

// Slots that query row r (token r / group of this call) sees: up to this one.
__device__ __forceinline__ int last_seen(const Cache8Attn& p, int start, int end, int r) {
  if (r >= p.rows) return -1;
  if (!p.causal) return end - 1;
  const long long first = static_cast<long long>(start) + p.appended - p.from_end;
  return static_cast<int>(min(first + token_of(p, r), static_cast<long long>(end) - 1));
}
__device__ __forceinline__ int end_of(const Cache8Attn& p, int start) {
  return static_cast<int>(min(static_cast<long long>(start) + p.appended, static_cast<long long>(p.c.slots)));
}
template <typename T>
__device__ __forceinline__ T* out_row(const Cache8Attn& p, int b, int h, int r) {
  const int tok = token_of(p, r);
  return static_cast<T*>(p.out) +
         ((static_cast<long long>(b) * p.count + tok) * p.out_heads * p.group + h * p.group + r - tok * p.group) * p.c.dim;
}

// s_first[b]: what all heads of the rows in front of b cost; s_first[batch]: all.
template <int kWarps>
__device__ __forceinline__ void count_tiles(const Cache8Attn& p, long long* s_first) {
  constexpr int kThreads = kWarps * 32;
  __shared__ long long s_sums[kWarps];
  const int each = (p.c.batch + kThreads - 1) / kThreads, from = threadIdx.x * each;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto cost = [&](int b) {
    const int tiles = (end_of(p, held_of(p.c, b)) + 15) >> 4;
    return tiles == 0 ? 0LL : static_cast<long long>(tiles + p.entry) * p.c.heads;
  };
  long long mine = 0;
  for (int b = from; b < min(from + each, p.c.batch); ++b) mine += cost(b);
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += u;
  }
  if (lane == 31) s_sums[warp] = sum;
  __syncthreads();
  for (int w = 0; w < warp; ++w) sum += s_sums[w];
  long long run = sum - mine;
  for (int b = from; b < min(from + each, p.c.batch); ++b) {
    s_first[b] = run;
    run += cost(b);
  }
  if (threadIdx.x == kThreads - 1) s_first[p.c.batch] = run;
  __syncthreads();
}

// What a score column needs beside its reference and sums.
struct Column {
  float scale;
  int lim, where, bias;
};

// Launches a kernel that may begin while the one in front of it still runs; it waits for it by itself (chain_wait).
template <typename... Params, typename... Args>
cudaError_t launch_behind(bool behind, void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                          cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = behind ? 1 : 0;
  count_launches(1);
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

// Attention of many query rows (cache8_rows.cu). type: 0 bf16, 1 fp16, 2 fp32.
constexpr int kRowWarps = 8;
// Few rows are dealt 16 a warp (8 heads of 128 channels over 8192 slots, us with 16 / 32: 16 rows 21 / 33, 64 27 / 35, 128 35 /
// 39, 192 56 / 50).
constexpr int kFewRows = 128;
constexpr int row_tile_of(int type, int rows) { return type == 2 || rows <= kFewRows ? 16 : 32; }  // query rows of a warp
cudaError_t launch_cache8_rows(const Cache8Attn& p, int type, bool behind, cudaStream_t stream);

}  // namespace t5x
