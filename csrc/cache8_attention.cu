// Attention over a key/value cache held in 8 bits (cache8.cuh), for a few query rows a key head: a decode step, the beams
// of a cross attention, a chunk of a prompt.
//
// out = sum_s p_s v_s / sum_s p_s, p_s = exp(scale q.k_s + bias - m), with the reference m and the sum of a streaming
// softmax; k and v are codes times their block's largest value / 127. Bytes bound it: 2 * dim a token and head are read
// once, and a query row does 4 * dim operations on them. So the codes go from global memory straight into the registers
// of mma.sync (whose operand of 8 columns the query rows of a head fill or nearly fill; a tcgen05 tile has 64 rows at
// least, and wants the codes converted in shared memory first), as fp16 numbers, which hold them exactly: S^T = K Q^T
// and O^T = V^T P^T, tokens and channels in the 16-row operand, 8 query rows in the other.
//
//   * Channels of a dot product may come in any order: lane (g, t) (g = lane / 4, t = lane % 4) loads channels
//     64 c + 16 t .. + 15 of tokens g and g + 8, sixteen bytes at a time, and MMA step (c, j) takes bytes 4 j .. 4 j + 3 of
//     them: the even ones as its k positions 2t and 2t + 1, the odd ones as 2t + 8 and 2t + 9. The query lies the same way.
//   * In the second product lane (g, t) loads dim / 8 channels, from g * dim / 8 on, of tokens {2t, 2t+1, 2t+8, 2t+9}; row
//     tile i takes channels 2 i and 2 i + 1 of each lane as its rows g and g + 8. So a lane ends up with adjacent channels.
//   * The probabilities, tokens by query rows in the first product's result, turn into the second one's operand by
//     movmatrix.
//   * Bytes stand under the exponent of 1024, and 1152 is subtracted from each, which leaves the code itself. (Keys as code + 128,
//     with 128 times the query's sum taken off the score, were an instruction a pair less and no faster, 95 us for the long
//     contexts below against 93, and what the two sums had lost stayed in the score, times the scale of its block.)
//
// Queries are scaled by a power of two to just below 2^14, where fp16 holds the values of 16-bit types down to 2^-28 of
// the row's largest without loss; values of 32 bits go in as two fp16 numbers each (22 bits). A probability goes into the
// product with its block's largest value, relative to references that are raised seldom (raising costs a maximum over the
// lanes and a multiplication of all sums; `Reference` has the rule): as one fp16 number, 11 bits (a quarter of the rounding of a bf16
// result, and random in sign), or as two. Sums are in 32 bits.
//
// Two ways to deal out the work. Over short caches, and longer ones where there are many (row, head), a CTA takes one: it
// appends the new tokens, its warps take tiles of 16 tokens in turn and meet in shared memory, and the scores that the
// weights are made from never leave it: one launch. Over long ones (of all lengths) all tiles of all (row, head) laid end to
// end are cut into one equal piece a CTA; what it has of a (row, head) that it does not have whole goes to workspace, and a
// second kernel joins the pieces. Many query rows have a kernel of their own, cache8_rows.cu.
//
// Measured, us on the device of a call with its append: 64 rows x 32 heads of 64 channels, up to 1024 slots of all lengths,
// with biases, positions and weights, 59 (2.5 TB/s; 38 % of the issue slots: a CTA has four steps of tiles, and waits for
// memory before and behind them as long); 8 rows x 8 heads of 128 channels, 8 queries each, up to 65536 slots of all lengths, 94
// (4.7 TB/s; full rows 197, 5.5 TB/s, 83 % of the copy rate: latency, four warps a scheduler wait for codes 38 % of their time and for
// an instruction's result 21 %, with 46 % of the issue slots and 41 % of the ALU pipe taken); 12 heads over 640 slots 8.3, all of it
// latency.
#include <algorithm>
#include <type_traits>

#include "cache8_attention.cuh"

namespace t5x {
namespace {

// The query rows of a (row, head), by one warp: the lanes' parts of the first product's second operand to
// s_query[Q2][CH * 4][32], the columns to s_cols[8].
template <typename T, int D, bool kTwo, bool kFold>
__device__ __forceinline__ void lay_query(const Cache8Attn& p, int b, int h, int start, int end, int first_bias,
                                          uint2* s_query, Column* s_cols) {
  constexpr int CH = D / 64, Q2 = kTwo ? 2 : 1, E = 16 / sizeof(T);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int dropped = p.c.position != nullptr ? p.c.dropped[b] : 0;
  const int q_first = static_cast<int>(static_cast<long long>(start) + p.appended - p.from_end);
  {
    const int r = kFold ? g & 3 : g, i = token_of(p, min(r, p.rows - 1)), in_group = min(r, p.rows - 1) - i * p.group;
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_st + (h * p.group + in_group) * p.q_sh + 16 * t;
    float x[CH][16];
    uint32_t most = 0;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      alignas(16) T part[16];
      if (p.q_vec) {
#pragma unroll
        for (int k = 0; k < 16 / E; ++k)
          *reinterpret_cast<uint4*>(part + k * E) = *reinterpret_cast<const uint4*>(src + 64 * ch + k * E);
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) part[k] = src[64 * ch + k];
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        x[ch][k] = r < p.rows ? to_float(part[k]) : 0.f;
        most = max(most, abs_bits(x[ch][k]));
      }
    }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^up brings the largest to [2^13, 2^14)
    int up = most == 0 || most >= 0x7f800000u ? 0 : 13 - (static_cast<int>(most >> 23) - 127);
    up = max(min(up, 126), -113);
    const float by = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
#pragma unroll
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t f[Q2][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float lo = x[ch][4 * j + k] * by, hi = x[ch][4 * j + 2 + k] * by;
          const __half2 v = __floats2half2_rn(lo, hi);
          f[0][k] = as_u32(v);
          if (kTwo) f[Q2 - 1][k] = as_u32(__floats2half2_rn(lo - __low2float(v), hi - __high2float(v)));
        }
#pragma unroll
        for (int w = 0; w < Q2; ++w) s_query[(w * CH * 4 + ch * 4 + j) * 32 + lane] = make_uint2(f[w][0], f[w][1]);
      }
    if (t == 0) {
      Column col;
      // the scale of a key block is its largest value / 127; scores are times log2 e
      col.scale = __uint_as_float(static_cast<uint32_t>(127 - up) << 23) * p.scale * (kLog2e / 127.f);
      col.lim = r < p.rows ? last_seen(p, start, end, r) : 0x7fffffff;  // (a column without a row hinders nobody)
      col.where = q_first + i + dropped;
      col.bias = first_bias + in_group * p.table_stride;
      s_cols[g] = col;
    }
  }
}

enum Deal {
  kRowHead,  // a CTA takes a (row, head), and appends
  kPieces    // a CTA takes a piece of the tiles
};

// MT: tiles of 16 tokens a step; kTwo: operands as two fp16 numbers each.
// kFold: up to four query rows, twice in the 8 columns: of a step's two tiles the first counts in columns 0 to 3 and the second
// in 4 to 7, so that what is done for scores and probabilities is done once for both.
template <typename T, int D, int MT, bool kTwo, Deal kDeal, int kWarps, bool kFold>
__global__ void __launch_bounds__(kWarps * 32, 16 / kWarps)
    cache8_attention_kernel(const __grid_constant__ Cache8Attn p, const __grid_constant__ NewTokens<T> fresh) {
  constexpr bool kBlock = kDeal == kRowHead;
  static_assert(!kFold || MT == 2, "two tiles fold");
  constexpr int MS = kFold ? 1 : MT;           // tiles of scores that a lane has
  constexpr int kParts = kFold ? 2 : 1;        // columns of a query row
  constexpr int kThreads = kWarps * 32;
  constexpr int CH = D / 64;       // 64-channel pieces
  constexpr int VB = D / 8;        // channels a lane has in the second product
  constexpr int MI = D / 16;       // row tiles of the second product
  constexpr int Q2 = kTwo ? 2 : 1;
  constexpr bool kQueryRegs = D == 64;  // the query's operand is kept in registers
  constexpr int kQuery = Q2 * CH * 4 * 32;
  // the query's operand; the bias table, times log2 e (kRowHead: of the head's rows); the sums
  // of the warps [kWarps][rows][D]; kRowHead: scores [rows][slots]
  extern __shared__ uint2 s_dyn[];
  uint2* s_query = s_dyn;
  float* s_table = reinterpret_cast<float*>(s_dyn + kQuery);
  __shared__ long long s_first[kBlock ? 1 : kMaxBatch + 1];
  __shared__ uint8_t s_buckets[kMaxDistances];
  __shared__ Column s_cols[8];
  __shared__ float2 s_stats[kWarps * kParts][8];
  __shared__ float2 s_rows[8];
  const Cache8& c = p.c;
  const uint32_t low = p.low;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, wid = threadIdx.x >> 5;
  const int unit = blockIdx.x;  // (kPieces)

  const int biases = p.table == nullptr ? 0 : (kBlock ? 1 : c.heads) * p.group * p.table_stride;
  if (p.table != nullptr) {
    for (int i = threadIdx.x; i < p.distances; i += kThreads) s_buckets[i] = p.buckets[i];
    const float* from = p.table + (kBlock ? blockIdx.x * biases : 0);
    for (int i = threadIdx.x; i < biases; i += kThreads) {
      const float x = from[i];  // (finite ones stay finite)
      s_table[i] = fabsf(x) < INFINITY ? fminf(fmaxf(x * kLog2e, -0x1p126f), 0x1p126f) : x;
    }
  }
  float* s_sums = s_table + (biases + 3) / 4 * 4;
  float* s_scores = s_sums + kWarps * kParts * p.rows * D;

  long long at = 0, stop = 1;
  int b = 0;
  if constexpr (kBlock) {
    b = blockIdx.y;
  } else {
    count_tiles<kWarps>(p, s_first);
    const long long all = s_first[c.batch];
    const long long piece = max((all + p.pieces - 1) / p.pieces, static_cast<long long>(p.least));
    if (blockIdx.x == 0 && blockIdx.y == 0) {
      for (int i = threadIdx.x; i <= c.batch; i += kThreads) p.first[i] = s_first[i];
      if (threadIdx.x == 0) p.first[c.batch + 1] = piece;
    }
    chain_wait();  // new tokens are written by the kernel in front
    chain_release();
    at = unit * piece;
    stop = min(at + piece, all);
    if (at >= stop) return;
    for (int step = 1 << 11; step > 0; step >>= 1)  // the last row that begins at or before `at` and holds something
      if (b + step < c.batch && s_first[b + step] <= at) b += step;
  }

  while (at < stop) {
    if constexpr (!kBlock)
      while (s_first[b + 1] <= at) ++b;
    const int start = held_of(c, b), end = end_of(p, start);
    const int tiles = (end + 15) >> 4;
    int h, tile0, tile1;
    long long seg = 0;
    if constexpr (kBlock) {
      h = blockIdx.x;
      tile0 = 0;
      tile1 = tiles;
    } else {
      h = static_cast<int>((at - s_first[b]) / (tiles + p.entry));
      seg = s_first[b] + static_cast<long long>(h) * (tiles + p.entry) + p.entry;  // this (row, head)'s first tile
      tile0 = static_cast<int>(max(at - seg, 0LL));
      tile1 = static_cast<int>(min(stop - seg, static_cast<long long>(tiles)));
      if (tile1 <= 0) break;  // (no more than a part of what the beginning costs)
    }
    constexpr int kStep = kWarps * MT;
    const int mine = tile0 + wid * MT;  // this warp's first tile
    const long long bh = static_cast<long long>(b) * c.heads + h;

    const long long slots0 = bh * c.slots;
    const int8_t* keys = c.codes[0] + slots0 * D + g * D + 16 * t;
    const int8_t* values = c.codes[1] + slots0 * D + 2 * t * D + VB * g;
    const float* k_most = c.absmax[0] + bh * (c.slots >> c.block_log2);
    const float* v_most = c.absmax[1] + bh * (c.slots >> c.block_log2);
    const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + b * p.mask_stride;
    const bool placed = p.table != nullptr && c.position != nullptr;

    uint4 kr[MT][2][CH];         // tokens g, g + 8
    uint32_t vr[MT][4][VB / 4];  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
    float ka[MS], va[MS];
    int place[MS][2];
    const int fold = kFold ? t >> 1 : 0;  // which of the two tiles this lane's columns count
    // (what the kernel in front may have written is read through L2)
    auto get = [](const auto* ptr) { return __ldcg(ptr); };
    // (a tile past the end is read again, and hidden)
    auto load_k = [&](int tile) {
#pragma unroll
      for (int ms = 0; ms < MS; ++ms) {
        const int s0 = min(tile + ms + fold, tile1 - 1) << 4;
        ka[ms] = get(k_most + (s0 >> c.block_log2));
        if (placed) place[ms][0] = get(c.position + slots0 + s0 + g), place[ms][1] = get(c.position + slots0 + s0 + g + 8);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int8_t* src = keys + static_cast<long long>(min(tile + mt, tile1 - 1)) * (16 * D);
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int ch = 0; ch < CH; ++ch) kr[mt][e][ch] = get(reinterpret_cast<const uint4*>(src + 8 * e * D + 64 * ch));
      }
    };
    auto load_v = [&](int tile) {
#pragma unroll
      for (int ms = 0; ms < MS; ++ms) va[ms] = get(v_most + (min(tile + ms + fold, tile1 - 1) << 4 >> c.block_log2));
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int8_t* src = values + static_cast<long long>(min(tile + mt, tile1 - 1)) * (16 * D);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int8_t* from = src + ((e & 1) + 8 * (e >> 1)) * D;
          if (VB == 16) {
            const uint4 u = get(reinterpret_cast<const uint4*>(from));
            vr[mt][e][0] = u.x, vr[mt][e][1] = u.y, vr[mt][e][VB / 4 - 2] = u.z, vr[mt][e][VB / 4 - 1] = u.w;
          } else {
            const uint2 u = get(reinterpret_cast<const uint2*>(from));
            vr[mt][e][0] = u.x, vr[mt][e][1] = u.y;
          }
        }
      }
    };

    const int first_bias = kBlock ? 0 : h * p.group * p.table_stride;
    if constexpr (kBlock) {
      // Keys by one half of the threads, values by the other. Tokens of one block that the threads hold at a time are
      // requested first, the first tiles behind them.
      __shared__ uint32_t s_most[kWarps];
      constexpr int kHalf = kThreads / 2, kLanes = D / 4;
      const int half = threadIdx.x / kHalf, tid = threadIdx.x % kHalf, d = tid % kLanes * 4, own = tid / kLanes;
      const int blk = start >> c.block_log2, touched = blk << c.block_log2;
      const bool few = end > start && end - start <= kHalf / kLanes && end <= touched + (1 << c.block_log2);
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      float before = 0.f;
      float* most_at = c.absmax[half] + bh * (c.slots >> c.block_log2) + blk;
      if (few) {
        if (own < end - start) load_four(fresh.x[half] + b * fresh.sb[half] + h * fresh.sh[half] + own * fresh.st[half] + d, fresh.vec != 0, v);
        if (start > touched) before = __ldcg(most_at);
      }
      if (mine < tile1) {
        load_k(mine);
        load_v(mine);
      }
      if (wid == 0) lay_query<T, D, kTwo, kFold>(p, b, h, start, end, first_bias, s_query, s_cols);
      if (few) {
        uint32_t most = max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) s_most[wid] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps / 2; ++w) most = max(most, s_most[half * (kWarps / 2) + w]);
        most = max(most, abs_bits(before));
        const float a = __uint_as_float(most);
        int8_t* codes = c.codes[half] + slots0 * D + d;
        if (most != abs_bits(before)) {
          const Coder again(before, a);
#pragma unroll 4
          for (int s = touched + own; s < start; s += kHalf / kLanes) {
            char4* to = reinterpret_cast<char4*>(codes + static_cast<long long>(s) * D);
            const char4 u = *to;
            *to = make_char4(again.of<true>(u.x), again.of<true>(u.y), again.of<true>(u.z), again.of<true>(u.w));
          }
        }
        if (tid == 0) *most_at = a;
        if (own < end - start) {
          constexpr bool kShort = sizeof(T) == 2;
          const Coder code(127.f, a);
          *reinterpret_cast<char4*>(codes + static_cast<long long>(start + own) * D) = 
              make_char4(code.of<kShort>(v[0]), code.of<kShort>(v[1]), code.of<kShort>(v[2]), code.of<kShort>(v[3]));
          if (half == 0 && d == 0) {
            if (c.weight != nullptr) c.weight[slots0 + start + own] = 0.f;
            if (c.position != nullptr) c.position[slots0 + start + own] = start + own + c.dropped[b];
          }
        }
      } else {
        for (int lo = start; lo < end;) {
          const int hi = min(end, ((lo >> c.block_log2) + 1) << c.block_log2);
          append_block<T, D, kHalf>(c, fresh, half, b, h, start, lo, hi, tid, s_most + half * (kWarps / 2));
          lo = hi;
        }
      }
      __syncthreads();
      // what was requested of a block that got tokens is requested again
      if (p.appended > 0 && mine < tile1 && min(mine + MT, tile1) << 4 > touched) {
        load_k(mine);
        load_v(mine);
      }
      at = stop;
    } else {
      if (mine < tile1) {
        load_k(mine);
        load_v(mine);
      }
      if (wid == 0) lay_query<T, D, kTwo, kFold>(p, b, h, start, end, first_bias, s_query, s_cols);
      __syncthreads();
    }

    // ---- the query: this lane's part of the operand, and what it needs for score columns 2t and 2t + 1 ----
    uint2 qf[kQueryRegs ? Q2 : 1][kQueryRegs ? CH * 4 : 1];
    if constexpr (kQueryRegs) {
#pragma unroll
      for (int w = 0; w < Q2; ++w)
#pragma unroll
        for (int j = 0; j < CH * 4; ++j) qf[w][j] = s_query[(w * CH * 4 + j) * 32 + lane];
    }
    const Column cols[2] = {s_cols[2 * t], s_cols[2 * t + 1]};
    int all_see = end - 1;  // slots up to this one are seen by every row of the tile
    all_see = min(all_see, min(cols[0].lim, cols[1].lim));
    all_see = __reduce_min_sync(0xffffffffu, all_see);

    float o[MI][4];
    Reference ref[2];
    float l[2];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) ref[e] = {kNothing, 1.f}, l[e] = 0.f;

    for (int tile = mine; tile < tile1; tile += kStep) {
      // ---- S^T = K Q^T ----
      float st[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < 4; ++k) st[mt][k] = 0.f;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t a[MT][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t w = j == 0 ? kr[mt][e][ch].x : j == 1 ? kr[mt][e][ch].y : j == 2 ? kr[mt][e][ch].z : kr[mt][e][ch].w;
              a[mt][e] = number_pair(w, low);
              a[mt][2 + e] = number_pair(w >> 8, low);
            }
          uint32_t q0[Q2], q1[Q2];
#pragma unroll
          for (int w = 0; w < Q2; ++w) {
            uint2 q;
            if constexpr (kQueryRegs) q = qf[w][ch * 4 + j];
            else q = s_query[(w * CH * 4 + ch * 4 + j) * 32 + lane];
            q0[w] = q.x, q1[w] = q.y;
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) mma_sum<Q2>(st[mt], a[mt], q0, q1);
        }
      float s[MS][4], k_scale[MS];
      int here[MS][2];  // positions of tokens g and g + 8
#pragma unroll
      for (int ms = 0; ms < MS; ++ms) {
        k_scale[ms] = ka[ms];
        here[ms][0] = place[ms][0], here[ms][1] = place[ms][1];
#pragma unroll
        for (int k = 0; k < 4; ++k) s[ms][k] = kFold && fold ? st[MT - 1][k] : st[ms][k];
      }
      if (tile + kStep < tile1) load_k(tile + kStep);

      // ---- scores of tokens g (k = 0, 1) and g + 8 (k = 2, 3), columns 2t (k = 0, 2) and 2t + 1 ----
#pragma unroll
      for (int ms = 0; ms < MS; ++ms) {
        const int s0 = (tile + ms + fold) << 4;
        const bool inside = tile + ms + fold < tile1;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float by = k_scale[ms] * cols[e].scale;
          s[ms][e] *= by;
          s[ms][2 + e] *= by;
        }
        if (p.table != nullptr) {
          if (!placed) here[ms][0] = s0 + g, here[ms][1] = s0 + g + 8;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int d = cols[k & 1].where - here[ms][k >> 1];
            s[ms][k] += s_table[cols[k & 1].bias + s_buckets[min(max(d, 0), p.distances - 1)]];
          }
        }
        const int last = tile + (kFold ? MT : ms + 1);  // of the step's tiles that are looked at here, and one
        if (!(last <= tile1 && last * 16 - 1 <= all_see && mask == nullptr)) {
          bool shown[2] = {inside, inside};
          if (mask != nullptr) {
#pragma unroll
            for (int e = 0; e < 2; ++e) shown[e] = inside && s0 + g + 8 * e < p.mask_len && mask[s0 + g + 8 * e] != 0;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (!shown[k >> 1] || s0 + g + 8 * (k >> 1) > cols[k & 1].lim) s[ms][k] = -INFINITY;
        }
        if ((kBlock ? c.weight != nullptr : p.scores != nullptr) && inside) {
          float* to = kBlock ? s_scores : p.scores + bh * p.rows * c.slots;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = kFold ? (2 * t + e) & 3 : 2 * t + e;
            if (r < p.rows) {
              to[r * c.slots + s0 + g] = s[ms][e];
              to[r * c.slots + s0 + g + 8] = s[ms][2 + e];
            }
          }
        }
      }

      // ---- references (all tiles of the step in one question: raise_to asks exactly) ----
      float most = va[0];
#pragma unroll
      for (int ms = 1; ms < MS; ++ms) most = fmaxf(most, va[ms]);
      bool raise = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int ms = 0; ms < MS; ++ms) top = fmaxf(top, fmaxf(s[ms][e], s[ms][2 + e]));
        raise |= beyond(ref[e], top, most * ref[e].by);
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = -INFINITY, term = -INFINITY;
#pragma unroll
          for (int ms = 0; ms < MS; ++ms) x = fmaxf(x, fmaxf(s[ms][e], s[ms][2 + e]));
#pragma unroll
          for (int lanes = 4; lanes < 32; lanes *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, lanes));
          const float score = raised(ref[e], x);
#pragma unroll
          for (int ms = 0; ms < MS; ++ms) term = fmaxf(term, fmaxf(s[ms][e], s[ms][2 + e]) - score + log2_approx(va[ms]));
#pragma unroll
          for (int lanes = 4; lanes < 32; lanes *= 2) term = fmaxf(term, __shfl_xor_sync(0xffffffffu, term, lanes));
          const float2 by = raise_to(ref[e], score, term);
          l[e] *= by.x;
#pragma unroll
          for (int i = 0; i < MI; ++i) o[i][e] *= by.y, o[i][2 + e] *= by.y;
        }
      }

      // ---- probabilities ----
      uint32_t pf[Q2][MT][2];
#pragma unroll
      for (int ms = 0; ms < MS; ++ms) {
#pragma unroll
        for (int k = 0; k < 4; ++k) s[ms][k] -= ref[k & 1].score;
        float r[2] = {va[ms] * ref[0].by, va[ms] * ref[1].by};
        float counts = 1.f;  // in the sum that divides
        if (!(fmaxf(r[0], r[1]) < kFar)) {
          counts = 0.f;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 part = part_of(ref[e], va[ms]);
            r[e] = part.x;
#pragma unroll
            for (int k = e; k < 4; k += 2) {
              l[e] += exp2_approx(s[ms][k]);
              s[ms][k] = far_score(s[ms][k], part.y, va[ms]);
            }
          }
        }
        float pr[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          pr[k] = exp2_approx(s[ms][k]);
          l[k & 1] += pr[k] * counts;
          pr[k] *= r[k & 1];
        }
        const __half2 v0 = __floats2half2_rn(pr[0], pr[1]), v1 = __floats2half2_rn(pr[2], pr[3]);
        uint32_t f[Q2][2];
        f[0][0] = as_u32(v0), f[0][1] = as_u32(v1);
        if (kTwo) {
          f[Q2 - 1][0] = rest_of(pr[0], pr[1], v0);
          f[Q2 - 1][1] = rest_of(pr[2], pr[3], v1);
        }
#pragma unroll
        for (int w = 0; w < Q2; ++w)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t turned = transposed(f[w][e]);  // (column g now)
            if constexpr (kFold) pf[w][0][e] = g < 4 ? turned : 0u, pf[w][1][e] = g < 4 ? 0u : turned;
            else pf[w][ms][e] = turned;
          }
      }

      // ---- O^T += V^T P^T ----
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int w = 0; w < VB / 4; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t x = __byte_perm(vr[mt][0][w], vr[mt][1][w], half ? 0x7632 : 0x5410);
            const uint32_t y = __byte_perm(vr[mt][2][w], vr[mt][3][w], half ? 0x7632 : 0x5410);
            const uint32_t a[4] = {number_pair(x, low), number_pair(x >> 8, low), number_pair(y, low), number_pair(y >> 8, low)};
            uint32_t p0[Q2], p1[Q2];
#pragma unroll
            for (int q2 = 0; q2 < Q2; ++q2) p0[q2] = pf[q2][mt][0], p1[q2] = pf[q2][mt][1];
            mma_sum<Q2, true>(o[2 * w + half], a, p0, p1);
          }
      if (tile + kStep < tile1) load_v(tile + kStep);
    }

    // The whole (row, head), or a piece of it: a unit has one that began before its own first tile at most, and one that goes
    // on behind its last.
    const bool whole = tile0 == 0 && tile1 == tiles;
    const long long slot = (unit * 2LL + (tile0 == 0 ? 1 : 0)) * 8;
    {
      // ---- the warps meet; the weights of the first slots are requested ahead ----
      constexpr int kAhead = 4;
      float weight[kAhead];
      if (kBlock && c.weight != nullptr) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int at_slot = threadIdx.x + i * kThreads;
          weight[i] = at_slot < start ? c.weight[slots0 + at_slot] : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int r = kFold ? (2 * t + e) & 3 : 2 * t + e, part = wid * kParts + fold;
        if (r < p.rows) {
          const float f = power_of_two(scale_of(ref[e])) * (1.f / 127.f);
          float* dst = s_sums + (part * p.rows + r) * D + VB * g;
#pragma unroll
          for (int i = 0; i < MI; i += 2)
            *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[i][e] * f, o[i][2 + e] * f, o[i + 1][e] * f,
                                                                  o[i + 1][2 + e] * f);
          if (g == 0) s_stats[part][r] = make_float2(ref[e].score, sum);
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < p.rows * (D / 4); i += kThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float high = kNothing, sum = 0.f;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps * kParts; ++w) high = fmaxf(high, s_stats[w][r].x);
#pragma unroll
        for (int w = 0; w < kWarps * kParts; ++w) {
          const float2 st = s_stats[w][r];
          if (st.y == 0.f) continue;  // (a warp that saw nothing may have sums of 0 * NaN)
          const float f = exp2_approx(st.x - high);
          const float4 v = *reinterpret_cast<const float4*>(s_sums + (w * p.rows + r) * D + d);
          sum += st.y * f;
          x[0] += v.x * f, x[1] += v.y * f, x[2] += v.z * f, x[3] += v.w * f;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (whole || kBlock) {
          T* dst = out_row<T>(p, b, h, r) + d;
#pragma unroll
          for (int k = 0; k < 4; ++k) dst[k] = from_float<T>(x[k] * inv);
          if (d == 0) {
            if (kBlock) s_rows[r] = make_float2(high, inv);
            else if (p.scores != nullptr) p.final_stats[bh * p.rows + r] = make_float2(high, inv);
          }
        } else {
          *reinterpret_cast<float4*>(p.part + (slot + r) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
          if (d == 0) p.stats[slot + r] = make_float2(high, sum);
        }
      }
      if (kBlock && c.weight != nullptr) {
        __syncthreads();
        auto given = [&](int s) {
          float sum = 0.f;
          for (int r = 0; r < p.rows; ++r) {
            const float x = s_scores[r * c.slots + s];
            if (x > -INFINITY || x != x) sum += exp2_approx(x - s_rows[r].x) * s_rows[r].y;
          }
          return sum;
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int at_slot = threadIdx.x + i * kThreads;
          if (at_slot < end) c.weight[slots0 + at_slot] = weight[i] + given(at_slot);
        }
#pragma unroll 4
        for (int s = threadIdx.x + kAhead * kThreads; s < end; s += kThreads)
          c.weight[slots0 + s] = (s >= start ? 0.f : c.weight[slots0 + s]) + given(s);
      }
      if (!kBlock) __syncthreads();  // the next piece's query and sums
    }
    if constexpr (!kBlock) at = seg + tile1;
  }
}

// A block a query row: joins its pieces, where it has several, or none. A lane has four adjacent channels. Bound by
// dependent reads: by itself from a cold L2 8 us for 512 rows of long contexts, 17 for 4000 rows of nine pieces each.
constexpr int kJoinThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) cache8_join_kernel(const __grid_constant__ Cache8Attn p, int tile_rows) {
  constexpr int L = D / 4, S = kJoinThreads / L;  // lanes a piece, pieces at a time
  __shared__ float4 s_x[S][L];
  __shared__ float2 s_stat[S];
  const int bh = blockIdx.x, r = blockIdx.y, b = bh / p.c.heads, h = bh - b * p.c.heads;
  const int sub = threadIdx.x / L, lane = threadIdx.x % L;
  chain_wait();
  chain_release();
  const long long piece = __ldcg(p.first + p.c.batch + 1), from = __ldcg(p.first + b);
  const long long cost = (__ldcg(p.first + b + 1) - from) / p.c.heads;  // tiles + p.entry, or 0
  const long long seg = from + h * cost + p.entry;  // its first tile
  const int w0 = static_cast<int>(seg / piece), w1 = cost == 0 ? w0 - 1 : static_cast<int>((seg + cost - p.entry - 1) / piece);
  if (w0 == w1) return;  // one unit had it whole
  // the first piece is its unit's second, the others are their units' first ones
  const long long base = (static_cast<long long>(r / tile_rows) * p.pieces) * 2 * tile_rows + r % tile_rows;
  auto slot = [&](int w) { return base + (w * 2LL + (w == w0 ? 1 : 0)) * tile_rows; };
  float high = kNothing, sum = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int U = 4;  // pieces requested at a time
  for (int w = w0 + sub; w <= w1; w += S * U) {
    float2 st[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(w + u * S, w1);
      st[u] = __ldcg(p.stats + slot(at));
      v[u] = __ldcg(reinterpret_cast<const float4*>(p.part + slot(at) * D) + lane);
      if (w + u * S > w1) st[u] = make_float2(kNothing, 0.f);
    }
    float top = high;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, st[u].x);
    const float f0 = exp2_approx(high - top);
    high = top;
    sum *= f0, x.x *= f0, x.y *= f0, x.z *= f0, x.w *= f0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (st[u].y == 0.f) continue;
      const float f = exp2_approx(st[u].x - top);
      sum += st[u].y * f;
      x.x += v[u].x * f, x.y += v[u].y * f, x.z += v[u].z * f, x.w += v[u].w * f;
    }
  }
  s_x[sub][lane] = x;
  if (lane == 0) s_stat[sub] = make_float2(high, sum);
  __syncthreads();
  if (sub != 0) return;
  float top = kNothing;
#pragma unroll
  for (int i = 0; i < S; ++i) top = fmaxf(top, s_stat[i].x);
  sum = 0.f;
  x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const float f = s_stat[i].y == 0.f ? 0.f : exp2_approx(s_stat[i].x - top);
    const float4 v = s_x[i][lane];
    sum += s_stat[i].y * f;
    if (f != 0.f) x.x += v.x * f, x.y += v.y * f, x.z += v.z * f, x.w += v.w * f;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* dst = out_row<T>(p, b, h, r) + 4 * lane;
  const float o[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
#pragma unroll
  for (int j = 0; j < 4; ++j) dst[j] = from_float<T>(sum == 0.f ? 0.f : o[j]);
  if (lane == 0 && p.scores != nullptr) p.final_stats[static_cast<long long>(bh) * p.rows + r] = make_float2(top, inv);
}

// weight[slot] += the probabilities that the query rows gave it, from the scores that are in workspace: their bytes bound it.
constexpr int kWeightThreads = 256;
__global__ void __launch_bounds__(kWeightThreads) cache8_weight_kernel(const __grid_constant__ Cache8Attn p) {
  const unsigned all = p.c.batch * p.c.heads, block = blockIdx.x / all;
  const int bh = blockIdx.x - block * all, b = bh / p.c.heads;
  const int s = block * kWeightThreads + threadIdx.x;
  const int start = held_of(p.c, b), end = end_of(p, start);
  chain_wait();
  chain_release();
  if (s >= end) return;
  float* weight = p.c.weight + static_cast<long long>(bh) * p.c.slots + s;
  float sum = 0.f;
  for (int r = 0; r < p.rows; ++r) {
    if (s > last_seen(p, start, end, r)) continue;  // (no score was written)
    const float x = __ldcg(p.scores + (static_cast<long long>(bh) * p.rows + r) * p.c.slots + s);
    const float2 st = __ldcg(p.final_stats + static_cast<long long>(bh) * p.rows + r);
    if (x > -INFINITY || x != x) sum += exp2_approx(x - st.x) * st.y;
  }
  *weight = __ldcg(weight) + sum;
}

// Shared memory of a team, beside the query and the biases.
constexpr int kMaxTeamBytes = 72 * 1024;
size_t team_bytes(const Cache8& c, int rows, bool scores) {
  return 4ull * rows * ((rows <= 4 && c.dim == 64 ? 16ull : 8ull) * c.dim + (scores && c.weight != nullptr ? c.slots : 0));
}
// Whether a CTA takes a whole (row, head): caches of up to 2048 slots, and of up to 8192 where there are three for every two
// SMs. One query a head, most slots held, us so / in pieces: 12 heads of 64 channels over 2048 slots 11.3 / 14.7, over 4096
// 17.2 / 14.5; 8 heads of 128 channels, 8 queries each, 16.8 / 17.0 and 28.2 / 16.9; 128 heads of 64 channels over 8192 slots
// 37.9 / 35.5, 256 of them 47.5 / 55.0; 64 x 32 of them, of all lengths, 237 / 274.
bool by_row_head(const Cache8& c, int rows) {
  const long long bh = static_cast<long long>(c.batch) * c.heads;
  return rows <= 8 && team_bytes(c, rows, true) <= kMaxTeamBytes && (c.slots <= 2048 || (c.slots <= 8192 && 2 * bh >= 3LL * num_sms()));
}

template <typename T, int D, int MT, bool kTwo, Deal kDeal, int kWarps, bool kFold>
cudaError_t launch_tile(const Cache8Attn& p, const NewTokens<T>& fresh, bool behind, cudaStream_t stream) {
  constexpr bool kBlock = kDeal == kRowHead;
  constexpr size_t query = sizeof(uint2) * (kTwo ? 2 : 1) * (D / 64) * 4 * 32;
  const size_t table = p.table == nullptr ? 0 : static_cast<size_t>((kBlock ? 1 : p.c.heads) * p.group * p.table_stride + 3) / 4 * 16;
  const size_t smem = query + table + team_bytes(p.c, p.rows, kBlock);
  static bool set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!set[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(cache8_attention_kernel<T, D, MT, kTwo, kDeal, kWarps, kFold>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(query) + kMaxBiases * 4 + kMaxTeamBytes);
    if (e != cudaSuccess) return e;
    set[dev & 63] = true;
  }
  const dim3 grid = kBlock ? dim3(p.c.heads, p.c.batch) : dim3(p.pieces);
  return launch_behind(behind, cache8_attention_kernel<T, D, MT, kTwo, kDeal, kWarps, kFold>, grid, kWarps * 32, smem, stream, p, fresh);
}

template <typename T, bool kTwo>
cudaError_t launch_row_heads(const Cache8Attn& p, const T5xNewTokens* tokens, cudaStream_t stream) {
  const NewTokens<T> fresh = make_tokens<T>(tokens);
  // Half the warps where there are two CTAs for every SM: what a CTA does around its tiles overlaps more of the others' tiles.
  // 1024 slots, heads of 64 channels, all lengths, us with 4 warps / 8: 256 (row, head) 11.4 / 10.4, 512 15.9 / 18.8, 2048
  // 48.6 / 65.8 (2 warps: 52 to 63 for 45 to 59).
  const bool many = static_cast<long long>(p.c.batch) * p.c.heads >= 2LL * num_sms();
  auto launch_with = [&](auto kernel_warps) {
    constexpr int W = decltype(kernel_warps)::value;
    if (p.c.dim == 128) return launch_tile<T, 128, 1, kTwo, kRowHead, W, false>(p, fresh, false, stream);
    return p.rows <= 4 ? launch_tile<T, 64, 2, kTwo, kRowHead, W, true>(p, fresh, false, stream)
                       : launch_tile<T, 64, 2, kTwo, kRowHead, W, false>(p, fresh, false, stream);
  };
  return many ? launch_with(std::integral_constant<int, 4>()) : launch_with(std::integral_constant<int, 8>());
}

template <typename T, bool kTwo>
cudaError_t launch_pieces(const Cache8Attn& p, bool behind, cudaStream_t stream) {
  const int type = sizeof(T) == 4 ? 2 : std::is_same<T, __half>::value ? 1 : 0;
  const int tile_rows = p.rows <= 8 ? 8 : row_tile_of(type, p.rows);
  const NewTokens<T> none = {};
  cudaError_t e = p.rows > 8        ? launch_cache8_rows(p, type, behind, stream)
                         : p.c.dim == 128  ? launch_tile<T, 128, 1, kTwo, kPieces, 8, false>(p, none, behind, stream)
                         : p.rows <= 4     ? launch_tile<T, 64, 2, kTwo, kPieces, 8, true>(p, none, behind, stream)
                                           : launch_tile<T, 64, 2, kTwo, kPieces, 8, false>(p, none, behind, stream);
  if (e != cudaSuccess) return e;
  const dim3 rows(static_cast<unsigned>(p.c.batch) * p.c.heads, p.rows);
  e = p.c.dim == 64 ? launch_behind(true, cache8_join_kernel<T, 64>, rows, kJoinThreads, 0, stream, p, tile_rows)
                    : launch_behind(true, cache8_join_kernel<T, 128>, rows, kJoinThreads, 0, stream, p, tile_rows);
  if (e != cudaSuccess || p.scores == nullptr) return e;
  // (a part has so few scores that these are below 2^31)
  const unsigned blocks = (p.c.slots + kWeightThreads - 1u) / kWeightThreads;
  return launch_behind(true, cache8_weight_kernel, dim3(blocks * p.c.batch * p.c.heads), kWeightThreads, 0, stream, p);
}

// What a launch has of a call: batch rows, key heads and queries.
struct Part {
  int row, rows, head, heads, query, queries;
};

// That part of a cache. (Of several rows it has all heads.)
Cache8 cache_of(Cache8 c, const Part& at) {
  const long long by_head = static_cast<long long>(at.row) * c.heads + at.head;
  for (int i = 0; i < 2; ++i) {
    c.codes[i] += by_head * c.slots * c.dim;
    c.absmax[i] += by_head * (c.slots >> c.block_log2);
  }
  c.index += static_cast<long long>(at.row) * c.index_stride;
  if (c.weight) c.weight += by_head * c.slots;
  if (c.position) c.position += by_head * c.slots, c.dropped += at.row;
  c.batch = at.rows;
  c.heads = at.heads;
  return c;
}

// The launches of a call, by f(part) until one is false. Where weights are added up a launch has no more scores than a gigabyte
// (which fills the SMs for long), or those of one query of one head: several rows, or several heads of a row, or several queries of
// a head.
constexpr long long kMaxScores = 1LL << 28;
template <typename F>
bool for_parts(const Cache8& c, int count, int group, F&& f) {
  int rows = kMaxBatch, heads = c.heads, queries = count;
  if (c.weight != nullptr) {
    const long long each = static_cast<long long>(group) * c.slots;  // scores of a query
    auto at_most = [&](int all, long long scores) {  // as many of them, of so many scores each, as fit
      return static_cast<int>(std::min<long long>(all, std::max(1LL, kMaxScores / scores)));
    };
    rows = at_most(kMaxBatch, each * count * c.heads);
    heads = at_most(c.heads, each * count);
    queries = at_most(count, each);
  }
  for (int r = 0; r < c.batch; r += rows)
    for (int h = 0; h < c.heads; h += heads)
      for (int q = 0; q < count; q += queries)
        if (!f(Part{r, std::min(rows, c.batch - r), h, std::min(heads, c.heads - h), q, std::min(queries, count - q)})) return false;
  return true;
}

struct Plan {
  int pieces = 0, least = 0, entry = 0, row_warps = 1;
  size_t part = 0, stats = 0, first = 0, scores = 0, final_stats = 0, total = 0;
};
Plan plan(const Cache8& c, int rows, int type) {
  Plan w = {};
  const int tile_rows = rows <= 8 ? 8 : row_tile_of(type, rows), row_tiles = (rows + tile_rows - 1) / tile_rows;
  // Pieces for all CTAs that the SMs hold at a time, none of under 64 tokens a warp; over many rows, where a CTA has its steps of
  // 64 tokens to itself, none of under one (8 heads of 128 channels over 512 slots, 64 rows: 16.7 us, 18.3 with two steps, 25.1
  // with eight; 500 rows: 39, 44, 64; over 8192 slots the same). Beginning a (row, head) costs as much as
  // 24 tiles where a CTA does some four of them a us (us for long contexts of all lengths / for 4 x 16 heads of 64 channels by
  // up to 16384 tokens with 8: 101 / 42, 16: 93 / 30, 24: 93 / 26, 40: 93 / 25).
  w.entry = rows <= 8 ? 24 : 6;
  w.least = (rows <= 8 ? 32 : 4) + w.entry;
  long long room = 2LL * num_sms();
  if (rows > 8) {
    w.row_warps = row_tiles > 4 ? kRowWarps : row_tiles > 2 ? 4 : 2;
    room = num_sms() / ((row_tiles + w.row_warps - 1) / w.row_warps);
  }
  const long long most = static_cast<long long>(c.batch) * c.heads * (c.slots / 16 + w.entry) / w.least + 1;
  w.pieces = static_cast<int>(std::max<long long>(1, std::min(room, most)));
  const size_t bh = static_cast<size_t>(c.batch) * c.heads;
  auto take = [&](size_t bytes) {
    const size_t at = w.total;
    w.total += (bytes + 15) / 16 * 16;
    return at;
  };
  const size_t parts = static_cast<size_t>(row_tiles) * w.pieces * 2 * tile_rows;
  w.part = take(parts * c.dim * 4);
  w.stats = take(parts * 8);
  w.first = take((static_cast<size_t>(c.batch) + 2) * 8);
  if (c.weight != nullptr) {
    w.scores = take(bh * rows * c.slots * 4);
    w.final_stats = take(bh * rows * 8);
  }
  return w;
}

int check_query(const Cache8& c, const T5xCache8Query* q, const T5xNewTokens* n) {
  if (q->count < 1 || q->group < 1 || q->type < 0 || q->type > 2 ||
      static_cast<long long>(q->count) * q->group > 65535 || c.heads * static_cast<long long>(c.batch) > (1 << 24))
    return set_error("cache8_attention: %d queries of type %d, %d heads a key head", q->count, q->type, q->group);
  const int bytes = q->type == 2 ? 4 : 2;
  if (!q->query || !q->out || !aligned_to(bytes, {q->query, q->out}) || !aligned_to(4, {q->table}))
    return set_error("cache8_attention: a null or misaligned pointer");
  if (q->table && (!q->buckets || q->distances < 1 || q->distances > kMaxDistances ||
                   q->table_stride < 1 || q->table_stride > kMaxBiases || q->table_stride * c.heads * q->group > kMaxBiases ||
                   *std::max_element(q->buckets, q->buckets + q->distances) >= q->table_stride))
    return set_error("cache8_attention: biases of %d distances for %d heads", q->distances, q->group);
  if (q->key_mask && (q->mask_len < 0 || q->mask_len > c.slots)) return set_error("cache8_attention: a mask of %d slots", q->mask_len);
  if (c.weight && static_cast<long long>(q->count) * q->group * c.slots > 0x7fffffffLL)
    return set_error("cache8_attention: %d queries with weights over %d slots", q->count, c.slots);
  if (n && (n->count != q->count || n->lengths)) return set_error("cache8_attention: %d queries, %d new tokens", q->count, n->count);
  return n ? check_new_tokens("cache8_attention", n) : 0;
}

}  // namespace
}  // namespace t5x

T5X_API long long t5x_cache8_attention_bytes(const T5xCache8* cache, const T5xCache8Query* q, const T5xNewTokens* n) {
  if (!cache || !q) return t5x::set_error("cache8_attention: null pointer");
  const t5x::Cache8 c = t5x::make_cache8(cache);
  if (int e = t5x::check_cache8("cache8_attention", c)) return e;
  if (int e = t5x::check_query(c, q, n)) return e;
  if (c.batch == 0) return 0;
  if (t5x::by_row_head(c, q->count * q->group)) return 0;
  size_t most = 0;  // (the launches have the same workspace, one after the other)
  t5x::for_parts(c, q->count, q->group, [&](const t5x::Part& at) {
    most = std::max(most, t5x::plan(t5x::cache_of(c, at), at.queries * q->group, q->type).total);
    return true;
  });
  return static_cast<long long>(most);
}

T5X_API int t5x_cache8_attention(const T5xCache8* cache, const T5xCache8Query* q, const T5xNewTokens* n, void* workspace,
                                 void* stream) {
  if (!cache || !q) return t5x::set_error("cache8_attention: null pointer");
  const t5x::Cache8 c = t5x::make_cache8(cache);
  if (int e = t5x::check_cache8("cache8_attention", c)) return e;
  if (int e = t5x::check_query(c, q, n)) return e;
  if (c.batch == 0) return 0;
  t5x::Cache8Attn p;
  p.c = c;
  p.q = q->query;
  p.out = q->out;
  p.table = static_cast<const float*>(q->table);
  p.mask = static_cast<const uint8_t*>(q->key_mask);
  p.q_sb = q->stride_batch;
  p.q_st = q->stride_token;
  p.q_sh = q->stride_head;
  p.table_stride = static_cast<int>(q->table_stride);
  p.mask_stride = q->mask_stride;
  const int q_size = q->type == 2 ? 4 : 2;
  p.q_vec = t5x::aligned_to(16, {q->query}) && ((q->stride_batch | q->stride_token | q->stride_head) * q_size) % 16 == 0;
  p.count = q->count;
  p.group = q->group;
  p.rows = q->count * q->group;
  p.from_end = q->count;
  p.out_heads = c.heads;
  p.by_group = ((1ull << 32) + q->group - 1) / q->group;
  p.distances = q->table ? q->distances : 0;
  if (q->table) std::copy_n(q->buckets, q->distances, p.buckets);
  p.mask_len = q->mask_len;
  p.causal = q->causal;
  p.appended = n ? n->count : 0;
  p.scale = q->scale;
  p.low = 0x00ff00ffu;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (t5x::by_row_head(c, p.rows)) {
    p.scores = nullptr;
    const cudaError_t e = q->type == 0   ? t5x::launch_row_heads<__nv_bfloat16, false>(p, n, st)
                          : q->type == 1 ? t5x::launch_row_heads<__half, false>(p, n, st)
                                         : t5x::launch_row_heads<float, true>(p, n, st);
    return e == cudaSuccess ? 0 : t5x::set_error("cache8_attention launch: %s", cudaGetErrorString(e));
  }
  if (!workspace || !t5x::aligned_to(16, {workspace}))
    return t5x::set_error("cache8_attention: a null or misaligned workspace");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (n)
    if (int e = t5x::cache8_append(c, n, st)) return e;
  const int size = q->type == 2 ? 4 : 2;
  bool behind = n != nullptr;  // (what follows the append alone may begin while it runs)
  cudaError_t e = cudaSuccess;
  t5x::for_parts(c, q->count, q->group, [&](const t5x::Part& at) {
    t5x::Cache8Attn part = p;
    part.c = t5x::cache_of(c, at);
    part.count = at.queries;
    part.rows = at.queries * q->group;
    part.from_end = q->count - at.query;
    const long long head = static_cast<long long>(at.head) * q->group;
    part.q = static_cast<const char*>(p.q) + (at.row * p.q_sb + at.query * p.q_st + head * p.q_sh) * size;
    part.out = static_cast<char*>(p.out) +
               ((static_cast<long long>(at.row) * q->count + at.query) * c.heads * q->group + head) * c.dim * size;
    part.table = p.table ? p.table + head * p.table_stride : nullptr;
    part.mask = p.mask ? p.mask + at.row * p.mask_stride : nullptr;
    const t5x::Plan w = t5x::plan(part.c, part.rows, q->type);
    part.pieces = w.pieces;
    part.row_warps = w.row_warps;
    part.least = w.least;
    part.entry = w.entry;
    part.part = reinterpret_cast<float*>(ws + w.part);
    part.stats = reinterpret_cast<float2*>(ws + w.stats);
    part.first = reinterpret_cast<long long*>(ws + w.first);
    part.scores = c.weight ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
    part.final_stats = reinterpret_cast<float2*>(ws + w.final_stats);
    e = q->type == 0   ? t5x::launch_pieces<__nv_bfloat16, false>(part, behind, st)
        : q->type == 1 ? t5x::launch_pieces<__half, false>(part, behind, st)
                       : t5x::launch_pieces<float, true>(part, behind, st);
    behind = false;
    return e == cudaSuccess;
  });
  return e == cudaSuccess ? 0 : t5x::set_error("cache8_attention launch: %s", cudaGetErrorString(e));
}
