// Attention over a key/value cache held in 8 bits (cache8.cuh), for a few query rows a key head: a decode step, the beams
// of a cross attention, a chunk of a prompt.
//
// out = sum_s p_s v_s / sum_s p_s, p_s = exp(scale q.k_s + bias - m), with the running maximum m and sum of a streaming
// softmax; k and v are codes times their block's largest value / 127. Bytes bound it: 2 * dim a token and head are read
// once, and a query row does 4 * dim operations on them. So the codes go from global memory straight into the registers
// of mma.sync (whose operand of 8 columns the query rows of a head fill or nearly fill; a tcgen05 tile has 64 rows at
// least, and wants the codes converted in shared memory first), as fp16 numbers, which hold them exactly: S^T = K Q^T
// and O^T = V^T P^T, tokens and channels in the 16-row operand, 8 query rows in the other.
//
//   * Channels of a dot product may come in any order: lane (g, t) (g = lane / 4, t = lane % 4) loads channels
//     64 c + 16 t .. + 15 of tokens g and g + 8, sixteen bytes at a time, and MMA step (c, j) takes bytes 4 j .. 4 j + 3 of
//     them as its k positions {2t, 2t+1, 2t+8, 2t+9}; the query is laid out the same way.
//   * In the second product lane (g, t) loads dim / 8 channels, from g * dim / 8 on, of tokens {2t, 2t+1, 2t+8, 2t+9}; row
//     tile i takes channels 2 i and 2 i + 1 of each lane as its rows g and g + 8. So a lane ends up with adjacent channels.
//   * The probabilities, tokens by query rows in the first product's result, turn into the second one's operand by
//     movmatrix.
//   * A byte u = code + 128 under the exponent of 1024 is the fp16 number 1024 + u; one subtraction gives the code.
//
// Queries are scaled by a power of two to just below 2^14, where fp16 holds the values of 16-bit types down to 2^-28 of
// the row's largest without loss; values of 32 bits go in as two fp16 numbers each (22 bits). Probabilities are 2^14 at
// the maximum, rounded to 11 bits (a quarter of the rounding of a bf16 result, and random in sign), or two numbers
// again. A value block's scale goes into the probability, relative to the largest scale that the row has met where it saw
// something, so that the accumulators need no scaling by token. Sums are in 32 bits.
//
// A block of warps takes a stretch of the slots of one (row, head); its warps take tiles in turn and meet at the end in
// shared memory, the stretches in workspace.
#include <algorithm>

#include "cache8.cuh"

namespace t5x {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxDistances = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPeak = 14.f;  // exponent of the largest probability, and of the largest query value

struct Cache8Attn {
  Cache8 c;
  const void* q;
  void* out;
  const float* table;
  const uint8_t* mask;
  long long q_sb, q_st, q_sh, table_stride, mask_stride;
  int count, group, rows;  // queries a row, heads a key head, their product
  int distances, mask_len, causal;
  int appended;            // tokens of this call behind c.index
  float scale;
  int splits;
  float* part;             // [batch * heads, splits, rows, dim], with splits
  float2* stats;           // [batch * heads, splits, rows]: maximum, sum
  float* scores;           // [batch * heads, rows, slots] where weights are added up, else null
  float2* final_stats;     // [batch * heads, rows]: maximum, 1 / sum; with scores
  uint8_t buckets[kMaxDistances];  // column of the bias table by distance
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t less_1152(uint32_t u) {
  return as_u32(__hsub2(as_half2(u), as_half2(0x64806480u)));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Slots that query row r (token r / group of this call) sees: up to this one.
__device__ __forceinline__ int last_seen(const Cache8Attn& p, int start, int end, int r) {
  if (r >= p.rows) return -1;
  if (!p.causal) return end - 1;
  // the queries are the last `count` tokens held
  const long long first = static_cast<long long>(start) + p.appended - p.count;
  return static_cast<int>(min(first + r / p.group, static_cast<long long>(end) - 1));
}

// NT: tiles of 8 query rows; MT: tiles of 16 tokens a step; kTwo: operands as two fp16 numbers each.
template <typename T, int D, int NT, int MT, bool kTwo>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) cache8_attention_kernel(const __grid_constant__ Cache8Attn p) {
  constexpr int CH = D / 64;       // 64-channel pieces
  constexpr int VB = D / 8;        // channels a lane has in the second product
  constexpr int MI = D / 16;       // row tiles of the second product
  constexpr int Q2 = kTwo ? 2 : 1;
  extern __shared__ float s_dyn[];  // [kWarps][NT * 8][D] at the end; before: bias by head and distance
  __shared__ float s_m[kWarps][NT * 8], s_l[kWarps][NT * 8];
  const Cache8& c = p.c;
  const int bh = blockIdx.x, split = blockIdx.y, row0 = blockIdx.z * NT * 8;
  const int b = bh / c.heads, h = bh - b * c.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  const int start = held_of(c, b);
  const int end_all = static_cast<int>(min(static_cast<long long>(start) + p.appended, static_cast<long long>(c.slots)));
  // the stretch of this CTA: whole tiles of 16 slots
  const int end = last_seen(p, start, end_all, min(row0 + NT * 8, p.rows) - 1) + 1;
  const int tiles = (end + 15) >> 4;
  const int per = (tiles + p.splits - 1) / p.splits;
  const int tile0 = split * per, tile1 = min(tile0 + per, tiles);

  if (p.table != nullptr) {
    for (int i = threadIdx.x; i < p.group * p.distances; i += kThreads) {
      const int gq = i / p.distances, d = i - gq * p.distances;
      s_dyn[i] = p.table[static_cast<long long>(h * p.group + gq) * p.table_stride + p.buckets[d]];
    }
    __syncthreads();
  }

  // ---- this lane's part of the query rows as the first product's second operand ----
  uint32_t qf[Q2][NT][CH * 4][2];
  float q_scale[NT][2];   // of the score columns 2t and 2t + 1
  int lim[NT][2], where[NT][2], head[NT][2];
  const int dropped = c.position != nullptr ? c.dropped[b] : 0;
  const int q_first = static_cast<int>(static_cast<long long>(start) + p.appended - p.count);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = row0 + nt * 8 + g;
    float x[CH][16];
    uint32_t most = 0;
    const int i = r / p.group;
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_st + (h * p.group + r - i * p.group) * p.q_sh;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        x[ch][k] = r < p.rows ? to_float(src[64 * ch + 16 * t + k]) : 0.f;
        most = max(most, abs_bits(x[ch][k]));
      }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^up brings the largest to [2^13, 2^14)
    int up = most == 0 || most >= 0x7f800000u ? 0 : 13 - (static_cast<int>(most >> 23) - 127);
    up = max(min(up, 126), -113);
    const float by = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
    const float back = __uint_as_float(static_cast<uint32_t>(127 - up) << 23) * p.scale;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lo = x[ch][2 * j] * by, hi = x[ch][2 * j + 1] * by;
        const __half2 v = __floats2half2_rn(lo, hi);
        qf[0][nt][ch * 4 + j / 2][j & 1] = as_u32(v);
        if (kTwo)
          qf[Q2 - 1][nt][ch * 4 + j / 2][j & 1] = as_u32(__floats2half2_rn(lo - __low2float(v), hi - __high2float(v)));
      }
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // lane 4 * row has that row's
      q_scale[nt][e] = __shfl_sync(0xffffffffu, back, (2 * t + e) * 4);
      const int rr = row0 + nt * 8 + 2 * t + e;
      lim[nt][e] = last_seen(p, start, end_all, rr);
      where[nt][e] = q_first + rr / p.group + dropped;
      head[nt][e] = min(rr, p.rows - 1) % p.group * p.distances;
    }
  }
  // slots up to this one are seen by every row of the tile
  int all_see = end - 1;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) all_see = min(all_see, lim[nt][e]);
  all_see = __reduce_min_sync(0xffffffffu, all_see);

  const long long at = static_cast<long long>(bh) * c.slots;
  const int8_t* keys = c.codes[0] + at * D;
  const int8_t* values = c.codes[1] + at * D;
  const float* k_most = c.absmax[0] + static_cast<long long>(bh) * (c.slots >> c.block_log2);
  const float* v_most = c.absmax[1] + static_cast<long long>(bh) * (c.slots >> c.block_log2);
  const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + b * p.mask_stride;

  float o[NT][MI][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[nt][i][k] = 0.f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }
  float v_ref[NT][2];  // largest value scale that a column met where it saw something
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) v_ref[nt][0] = v_ref[nt][1] = 0.f;

  uint4 kr[MT][2][CH];                 // tokens g, g + 8
  uint32_t vr[MT][4][VB / 4];          // tokens 2t, 2t + 1, 2t + 8, 2t + 9
  float ka[MT], va[MT];
  auto load_k = [&](int tile) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int s0 = min(tile + mt, tile1 - 1) << 4;  // (a tile past the end is read again, and hidden)
      ka[mt] = k_most[s0 >> c.block_log2];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int ch = 0; ch < CH; ++ch)
          kr[mt][e][ch] =
              *reinterpret_cast<const uint4*>(keys + static_cast<long long>(s0 + g + 8 * e) * D + 64 * ch + 16 * t);
    }
  };
  auto load_v = [&](int tile) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int s0 = min(tile + mt, tile1 - 1) << 4;
      va[mt] = v_most[s0 >> c.block_log2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int8_t* src = values + static_cast<long long>(s0 + 2 * t + (e & 1) + 8 * (e >> 1)) * D + VB * g;
        if (VB == 16) {
          const uint4 u = *reinterpret_cast<const uint4*>(src);
          vr[mt][e][0] = u.x, vr[mt][e][1] = u.y, vr[mt][e][VB / 4 - 2] = u.z, vr[mt][e][VB / 4 - 1] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(src);
          vr[mt][e][0] = u.x, vr[mt][e][1] = u.y;
        }
      }
    }
  };

  int tile = tile0 + warp * MT;
  if (tile < tile1) {
    load_k(tile);
    load_v(tile);
  }
  for (; tile < tile1; tile += kWarps * MT) {
    const int next = tile + kWarps * MT;
    // ---- S^T = K Q^T ----
    float s[MT][NT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[mt][nt][k] = 0.f;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const uint32_t w0[4] = {kr[mt][0][ch].x, kr[mt][0][ch].y, kr[mt][0][ch].z, kr[mt][0][ch].w};
        const uint32_t w1[4] = {kr[mt][1][ch].x, kr[mt][1][ch].y, kr[mt][1][ch].z, kr[mt][1][ch].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u0 = w0[j] ^ 0x80808080u, u1 = w1[j] ^ 0x80808080u;
          const uint32_t a0 = less_1152(__byte_perm(u0, 0x64646464u, 0x4140));
          const uint32_t a2 = less_1152(__byte_perm(u0, 0x64646464u, 0x4342));
          const uint32_t a1 = less_1152(__byte_perm(u1, 0x64646464u, 0x4140));
          const uint32_t a3 = less_1152(__byte_perm(u1, 0x64646464u, 0x4342));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int w = 0; w < Q2; ++w)
              mma_f16(s[mt][nt], a0, a1, a2, a3, qf[w][nt][ch * 4 + j][0], qf[w][nt][ch * 4 + j][1]);
        }
      }
    }
    float k_scale[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) k_scale[mt] = ka[mt] * (1.f / 127.f);
    if (next < tile1) load_k(next);

    bool some[MT];  // whether the mask shows a token of the tile
    // ---- scores of tokens g (k = 0, 1) and g + 8 (k = 2, 3), query rows 2t (k = 0, 2) and 2t + 1 ----
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int s0 = (tile + mt) << 4;
      const bool inside = tile + mt < tile1;
      const bool whole = inside && s0 + 15 <= all_see && mask == nullptr;
      bool shown[2] = {true, true};
      some[mt] = inside;
      if (mask != nullptr) {
#pragma unroll
        for (int e = 0; e < 2; ++e) shown[e] = s0 + g + 8 * e < p.mask_len && mask[s0 + g + 8 * e] != 0;
        some[mt] = inside && __any_sync(0xffffffffu, shown[0] || shown[1]);
      }
      int place[2] = {s0 + g, s0 + g + 8};
      if (p.table != nullptr && c.position != nullptr) {
#pragma unroll
        for (int e = 0; e < 2; ++e) place[e] = c.position[at + min(s0 + g + 8 * e, c.slots - 1)];
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x = s[mt][nt][k] * (k_scale[mt] * q_scale[nt][k & 1]);
          if (p.table != nullptr) {
            const int d = where[nt][k & 1] - place[k >> 1];
            x += s_dyn[head[nt][k & 1] + min(max(d, 0), p.distances - 1)];
          }
          if (!whole && !(inside && shown[k >> 1] && s0 + g + 8 * (k >> 1) <= lim[nt][k & 1])) x = -INFINITY;
          s[mt][nt][k] = x;
        }
      if (p.scores != nullptr && inside) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = row0 + nt * 8 + 2 * t + (k & 1);
            if (r < p.rows)
              p.scores[(static_cast<long long>(bh) * p.rows + r) * c.slots + s0 + g + 8 * (k >> 1)] = s[mt][nt][k];
          }
      }
    }

    // ---- running maximum, probabilities ----
    bool moved = false;
    float shrink[NT][2];
    uint32_t pf[Q2][MT][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float base[2], v_inv[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = m[nt][e];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) x = fmaxf(x, fmaxf(s[mt][nt][e], s[mt][nt][2 + e]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        base[e] = x == -INFINITY ? 0.f : x;
        const float f = exp2_approx((m[nt][e] - base[e]) * kLog2e);  // (0 at first)
        float v_new = v_ref[nt][e];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          if (some[mt] && lim[nt][e] >= (tile + mt) << 4 && va[mt] < INFINITY) v_new = fmaxf(v_new, va[mt]);
        moved |= x != m[nt][e] || v_new != v_ref[nt][e];
        v_inv[e] = v_new > 0.f ? __frcp_rn(v_new) : 0.f;
        shrink[nt][e] = f * (v_ref[nt][e] * v_inv[e]);  // (0 where nothing had been met)
        v_ref[nt][e] = v_new;
        m[nt][e] = x;
        l[nt][e] *= f;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float r[2] = {va[mt] * v_inv[0], va[mt] * v_inv[1]};
        float pr[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = s[mt][nt][k];
          const float e = exp2_approx(fmaf(x - base[k & 1], kLog2e, kPeak));
          l[nt][k & 1] += e;
          // (a hidden token counts for nothing whatever its block holds)
          pr[k] = x == -INFINITY ? 0.f : e * r[k & 1];
        }
        const __half2 v0 = __floats2half2_rn(pr[0], pr[1]), v1 = __floats2half2_rn(pr[2], pr[3]);
        pf[0][mt][nt][0] = transposed(as_u32(v0));
        pf[0][mt][nt][1] = transposed(as_u32(v1));
        if (kTwo) {
          pf[Q2 - 1][mt][nt][0] =
              transposed(as_u32(__floats2half2_rn(pr[0] - __low2float(v0), pr[1] - __high2float(v0))));
          pf[Q2 - 1][mt][nt][1] =
              transposed(as_u32(__floats2half2_rn(pr[2] - __low2float(v1), pr[3] - __high2float(v1))));
        }
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[nt][i][k] *= shrink[nt][k & 1];
    }

    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int w = 0; w < VB / 4; ++w) {
        const uint32_t u0 = vr[mt][0][w] ^ 0x80808080u, u1 = vr[mt][1][w] ^ 0x80808080u;
        const uint32_t u2 = vr[mt][2][w] ^ 0x80808080u, u3 = vr[mt][3][w] ^ 0x80808080u;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t x = __byte_perm(u0, u1, half ? 0x7362 : 0x5140), y = __byte_perm(u2, u3, half ? 0x7362 : 0x5140);
          const uint32_t a0 = less_1152(__byte_perm(x, 0x64646464u, 0x4140));
          const uint32_t a1 = less_1152(__byte_perm(x, 0x64646464u, 0x4342));
          const uint32_t a2 = less_1152(__byte_perm(y, 0x64646464u, 0x4140));
          const uint32_t a3 = less_1152(__byte_perm(y, 0x64646464u, 0x4342));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q2 = 0; q2 < Q2; ++q2)
              mma_f16(o[nt][2 * w + half], a0, a1, a2, a3, pf[q2][mt][nt][0], pf[q2][mt][nt][1]);
        }
      }
    if (next < tile1) load_v(next);
  }

  // ---- the warps meet ----
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[nt][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) {
        s_m[warp][nt * 8 + 2 * t + e] = m[nt][e];
        s_l[warp][nt * 8 + 2 * t + e] = x;
      }
    }
  __syncthreads();  // (and the bias table is read for the last time)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = nt * 8 + 2 * t + e;
      float most = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) most = fmaxf(most, s_m[w][col]);
      const float f = m[nt][e] == -INFINITY ? 0.f : exp2_approx((m[nt][e] - most) * kLog2e) * (v_ref[nt][e] * (1.f / 127.f));
      float* dst = s_dyn + (static_cast<long long>(warp) * NT * 8 + col) * D + VB * g;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        // a row that nothing was seen of has sums of 0, or of 0 * NaN
        const float x = m[nt][e] == -INFINITY && l[nt][e] == 0.f ? 0.f : o[nt][i][e] * f;
        const float y = m[nt][e] == -INFINITY && l[nt][e] == 0.f ? 0.f : o[nt][i][2 + e] * f;
        *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(x, y);
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 8 * D; i += kThreads) {
    const int col = i / D, r = row0 + col;
    if (r >= p.rows) break;
    float most = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most = fmaxf(most, s_m[w][col]);
    const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      sum += s_l[w][col] * exp2_approx((s_m[w][col] - base) * kLog2e);
      x += s_dyn[w * NT * 8 * D + i];
    }
    const int d = i - col * D;
    if (p.splits == 1) {
      const int tok = r / p.group;
      T* dst = static_cast<T*>(p.out) +
               ((static_cast<long long>(b) * p.count + tok) * c.heads * p.group + h * p.group + r - tok * p.group) * D + d;
      *dst = from_float<T>(sum == 0.f ? 0.f : x / sum);
      if (d == 0 && p.scores != nullptr)
        p.final_stats[static_cast<long long>(bh) * p.rows + r] = make_float2(base, sum == 0.f ? 0.f : 1.f / sum);
    } else {
      const long long part = (static_cast<long long>(bh) * p.splits + split) * p.rows + r;
      p.part[part * D + d] = x;
      if (d == 0) p.stats[part] = make_float2(most, sum);
    }
  }
}

// One warp a query row: joins the stretches.
template <typename T>
__global__ void __launch_bounds__(kThreads) cache8_join_kernel(const __grid_constant__ Cache8Attn p, long long total) {
  const long long at = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (at >= total) return;
  const int lane = threadIdx.x & 31, D = p.c.dim;
  const long long bh = at / p.rows;
  const int r = static_cast<int>(at - bh * p.rows);
  const float2* stats = p.stats + bh * p.splits * p.rows + r;
  float most = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) most = fmaxf(most, stats[static_cast<long long>(s) * p.rows].x);
  most = warp_max(most);
  const float base = most == -INFINITY ? 0.f : most;
  float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  const float* part = p.part + (bh * p.splits * p.rows + r) * D;
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = stats[static_cast<long long>(s) * p.rows];
    const float f = exp2_approx((ml.x - base) * kLog2e);
    sum += ml.y * f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j * 32 < D) x[j] += f * part[static_cast<long long>(s) * p.rows * D + j * 32 + lane];
  }
  const int b = static_cast<int>(bh / p.c.heads), h = static_cast<int>(bh - static_cast<long long>(b) * p.c.heads);
  const int tok = r / p.group;
  T* dst = static_cast<T*>(p.out) +
           ((static_cast<long long>(b) * p.count + tok) * p.c.heads * p.group + h * p.group + r - tok * p.group) * D;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j * 32 < D) dst[j * 32 + lane] = from_float<T>(sum == 0.f ? 0.f : x[j] / sum);
  if (lane == 0 && p.scores != nullptr) p.final_stats[at] = make_float2(base, sum == 0.f ? 0.f : 1.f / sum);
}

// weight[slot] += the probabilities that the query rows gave it
__global__ void __launch_bounds__(kThreads) cache8_weight_kernel(const __grid_constant__ Cache8Attn p) {
  const int bh = blockIdx.x, b = bh / p.c.heads;
  const int s = blockIdx.y * kThreads + threadIdx.x;
  const int start = held_of(p.c, b);
  const int end = static_cast<int>(min(static_cast<long long>(start) + p.appended, static_cast<long long>(p.c.slots)));
  if (s >= end) return;
  float sum = 0.f;
  for (int r = 0; r < p.rows; ++r) {
    if (s > last_seen(p, start, end, r)) continue;  // (no score was written)
    const float x = p.scores[(static_cast<long long>(bh) * p.rows + r) * p.c.slots + s];
    const float2 st = p.final_stats[static_cast<long long>(bh) * p.rows + r];
    // (the sums are of probabilities 2^kPeak times as large)
    sum += exp2_approx(fmaf(x - st.x, kLog2e, kPeak)) * st.y;
  }
  p.c.weight[static_cast<long long>(bh) * p.c.slots + s] += sum;
}

template <typename T, int D, int NT, int MT, bool kTwo>
cudaError_t launch_tile(const Cache8Attn& p, cudaStream_t stream) {
  const size_t smem = std::max(static_cast<size_t>(kWarps) * NT * 8 * D * 4,
                               p.table == nullptr ? size_t{0} : static_cast<size_t>(p.group) * p.distances * 4);
  static bool set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!set[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(cache8_attention_kernel<T, D, NT, MT, kTwo>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != cudaSuccess) return e;
    set[dev & 63] = true;
  }
  const int row_tiles = (p.rows + NT * 8 - 1) / (NT * 8);
  cache8_attention_kernel<T, D, NT, MT, kTwo>
      <<<dim3(static_cast<unsigned>(p.c.batch) * p.c.heads, p.splits, row_tiles), kThreads, smem, stream>>>(p);
  count_launches(1);
  return cudaGetLastError();
}

template <typename T, bool kTwo>
cudaError_t launch_all(const Cache8Attn& p, int nt, cudaStream_t stream) {
  cudaError_t e;
  if (p.c.dim == 64)
    e = nt == 1 ? launch_tile<T, 64, 1, 2, kTwo>(p, stream) : launch_tile<T, 64, 4, 1, kTwo>(p, stream);
  else
    e = nt == 1 ? launch_tile<T, 128, 1, 1, kTwo>(p, stream) : launch_tile<T, 128, kTwo ? 2 : 4, 1, kTwo>(p, stream);
  if (e != cudaSuccess) return e;
  if (p.splits > 1) {
    const long long total = static_cast<long long>(p.c.batch) * p.c.heads * p.rows;
    cache8_join_kernel<T><<<static_cast<unsigned>((total + kWarps - 1) / kWarps), kThreads, 0, stream>>>(p, total);
    count_launches(1);
  }
  if (p.scores != nullptr) {
    cache8_weight_kernel<<<dim3(static_cast<unsigned>(p.c.batch) * p.c.heads, (p.c.slots + kThreads - 1) / kThreads),
                           kThreads, 0, stream>>>(p);
    count_launches(1);
  }
  return cudaGetLastError();
}

// Tiles of 8 query rows a block takes, and stretches that the slots are cut into.
void plan(const Cache8& c, int rows, bool two, int& nt, int& splits) {
  nt = rows <= 8 ? 1 : 4;
  const int tile_rows = nt == 1 ? 8 : c.dim == 128 && two ? 16 : 32;
  const long long blocks = static_cast<long long>(c.batch) * c.heads * ((rows + tile_rows - 1) / tile_rows);
  // enough blocks for a few rounds over the SMs, none of under 256 slots
  const long long wanted = (4LL * num_sms() + blocks - 1) / blocks;
  splits = static_cast<int>(std::max(1LL, std::min({wanted, static_cast<long long>(c.slots) / 256, 1024LL})));
}

struct Workspace {
  size_t part = 0, stats = 0, scores = 0, final_stats = 0, total = 0;
};
Workspace workspace(const Cache8& c, int rows, int splits) {
  Workspace w;
  const size_t bh = static_cast<size_t>(c.batch) * c.heads;
  auto take = [&](size_t bytes) {
    const size_t at = w.total;
    w.total += (bytes + 15) / 16 * 16;
    return at;
  };
  if (splits > 1) {
    w.part = take(bh * splits * rows * c.dim * 4);
    w.stats = take(bh * splits * rows * 8);
  }
  if (c.weight != nullptr) {
    w.scores = take(bh * rows * c.slots * 4);
    w.final_stats = take(bh * rows * 8);
  }
  return w;
}

int check_query(const Cache8& c, const T5xCache8Query* q, const T5xNewTokens* n) {
  if (q->count < 1 || q->group < 1 || q->type < 0 || q->type > 2 ||
      static_cast<long long>(q->count) * q->group > (1 << 20) || c.heads * static_cast<long long>(c.batch) > (1 << 24))
    return set_error("cache8_attention: %d queries of type %d, %d heads a key head", q->count, q->type, q->group);
  const int bytes = q->type == 2 ? 4 : 2;
  if (!q->query || !q->out || !aligned_to(bytes, {q->query, q->out}) || !aligned_to(4, {q->table}))
    return set_error("cache8_attention: a null or misaligned pointer");
  if (q->table && (!q->buckets || q->distances < 1 || q->distances > kMaxDistances ||
                   static_cast<long long>(q->group) * q->distances > 40000))
    return set_error("cache8_attention: biases of %d distances for %d heads", q->distances, q->group);
  if (q->key_mask && (q->mask_len < 0 || q->mask_len > c.slots)) return set_error("cache8_attention: a mask of %d slots", q->mask_len);
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
  int nt, splits;
  t5x::plan(c, q->count * q->group, q->type == 2, nt, splits);
  return static_cast<long long>(t5x::workspace(c, q->count * q->group, splits).total);
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
  p.table_stride = q->table_stride;
  p.mask_stride = q->mask_stride;
  p.count = q->count;
  p.group = q->group;
  p.rows = q->count * q->group;
  p.distances = q->table ? q->distances : 0;
  if (q->table) std::copy_n(q->buckets, q->distances, p.buckets);
  p.mask_len = q->mask_len;
  p.causal = q->causal;
  p.appended = n ? n->count : 0;
  p.scale = q->scale;
  int nt;
  t5x::plan(c, p.rows, q->type == 2, nt, p.splits);
  const t5x::Workspace w = t5x::workspace(c, p.rows, p.splits);
  if (w.total && (!workspace || !t5x::aligned_to(16, {workspace})))
    return t5x::set_error("cache8_attention: a null or misaligned workspace");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.stats = reinterpret_cast<float2*>(ws + w.stats);
  p.scores = c.weight ? reinterpret_cast<float*>(ws + w.scores) : nullptr;
  p.final_stats = reinterpret_cast<float2*>(ws + w.final_stats);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n)
    if (int e = t5x::cache8_append(c, n, st)) return e;
  const cudaError_t e = q->type == 0   ? t5x::launch_all<__nv_bfloat16, false>(p, nt, st)
                        : q->type == 1 ? t5x::launch_all<__half, false>(p, nt, st)
                                       : t5x::launch_all<float, true>(p, nt, st);
  return e == cudaSuccess ? 0 : t5x::set_error("cache8_attention launch: %s", cudaGetErrorString(e));
}
