// Attention over a key/value cache held in 8 bits (cache8.cuh), for many query rows a key head: a chunk of a prompt, a
// prompt behind one that is held. cache8_attention.cu has the formulas, the scales and the streaming softmax.
//
// Here the products count more than the bytes: a code is converted once for all rows of a CTA. The CTA takes a piece of the
// tokens (all tokens of all (row, head), laid end to end, cut into equal pieces) in steps of 64: its threads load the codes
// of the next step while the warps compute on this one's, which lie in shared memory as fp16 numbers (exactly), 16 bytes
// swizzled by token. A warp has 32 query rows (16 of 32-bit types, as two fp16 numbers each): S = Q K^T with the rows in the
// 16-row operand, whose result is, lane for lane, the first operand of O = P V. Where there are fewer rows than eight warps
// take, warps share rows, take different tokens of a step, and meet in shared memory at the end.
//
// Bound by latency between the products: two warps a scheduler (128 sums a lane leave no room for more) keep the matrix pipe
// 37 % busy, the issue slots 30 %, and wait for an instruction's result 29 % of their time. Measured, us for 2 x 4 heads of 128 channels with
// the append and the join: 500 rows over 8192 slots, four fifths of them held, 87 (in 32 bits 135), over 32768 242, all held 286 (234
// TFLOP/s); 256 rows over 8192 55, 64 rows 26. Two tiles of tokens at a time instead of one took 4 and 9 % off, operands requested a step
// ahead 6.
#include <algorithm>
#include <type_traits>

#include "cache8_attention.cuh"

namespace t5x {
namespace {

constexpr int kThreads = kRowWarps * 32;
constexpr int kTokens = 64;  // of a step

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address));
}
__device__ __forceinline__ void load_transposed(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(address));
}
// four codes as fp16 numbers, in order: under the exponent of 1024 first
__device__ __forceinline__ uint2 numbers(uint32_t codes) {
  const uint32_t u = codes ^ 0x80808080u;
  const __half2 offset = as_half2(0x64806480u);
  return make_uint2(as_u32(__hsub2(as_half2(__byte_perm(u, 0x64646464u, 0x4140)), offset)),
                    as_u32(__hsub2(as_half2(__byte_perm(u, 0x64646464u, 0x4342)), offset)));
}

// What a query row needs.
struct Row {
  float scale;
  int lim, where, bias;  // (the last two are read where there are biases)
};

// The 16 * M query rows from row0 on of a (row, head), by one warp, a row to 4 lanes: the first operand of Q K^T to
// s_query[Q2][D / 16][M][32], the rows' own to s_rows[16 * M].
template <typename T, int D, int M, bool kTwo>
__device__ __forceinline__ void lay_rows(const Cache8Attn& p, int b, int h, int row0, int start, int end, uint4* s_query,
                                         Row* s_rows) {
  constexpr int J = D / 16;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int dropped = p.c.position != nullptr ? p.c.dropped[b] : 0;
  const int q_first = static_cast<int>(static_cast<long long>(start) + p.appended - p.from_end);
  uint32_t* to = reinterpret_cast<uint32_t*>(s_query);
  using Pair = typename std::conditional<sizeof(T) == 4, uint2, uint32_t>::type;
  Pair part[2 * M][J][2];  // channels 16 j + 2 t, + 1, + 8, + 9 of row 8 i + g
#pragma unroll
  for (int i = 0; i < 2 * M; ++i) {
    const int r = min(row0 + 8 * i + g, p.rows - 1), token = token_of(p, r), in_group = r - token * p.group;
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + token * p.q_st + (h * p.group + in_group) * p.q_sh + 2 * t;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (p.q_vec) part[i][j][k] = *reinterpret_cast<const Pair*>(src + 16 * j + 8 * k);
        else {
          T* pair = reinterpret_cast<T*>(&part[i][j][k]);
          pair[0] = src[16 * j + 8 * k], pair[1] = src[16 * j + 8 * k + 1];
        }
      }
  }
#pragma unroll
  for (int i = 0; i < 2 * M; ++i) {
    const int r = row0 + 8 * i + g, real = min(r, p.rows - 1), token = token_of(p, real), in_group = real - token * p.group;
    float x[J][4];
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[j][k] = r < p.rows ? to_float(reinterpret_cast<const T*>(&part[i][j][k >> 1])[k & 1]) : 0.f;
        most = max(most, abs_bits(x[j][k]));
      }
    }
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^up brings the largest to [2^13, 2^14)
    int up = most == 0 || most >= 0x7f800000u ? 0 : 13 - (static_cast<int>(most >> 23) - 127);
    up = max(min(up, 126), -113);
    const float by = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float lo = x[j][2 * k] * by, hi = x[j][2 * k + 1] * by;
        const __half2 v = __floats2half2_rn(lo, hi);
        const int at = ((j * M + (i >> 1)) * 32 + lane) * 4 + 2 * k + (i & 1);
        to[at] = as_u32(v);
        if (kTwo) to[J * M * 32 * 4 + at] = as_u32(__floats2half2_rn(lo - __low2float(v), hi - __high2float(v)));
      }
    if (t == 0) {
      Row row;
      // the scale of a key block is its largest value / 127; scores are times log2 e
      row.scale = __uint_as_float(static_cast<uint32_t>(127 - up) << 23) * p.scale * (kLog2e / 127.f);
      row.lim = r < p.rows ? last_seen(p, start, end, r) : 0x7fffffff;  // (one that is none hinders nobody)
      row.where = q_first + token + dropped;
      row.bias = (h * p.group + in_group) * p.table_stride;
      s_rows[8 * i + g] = row;
    }
  }
}

template <int D>
constexpr size_t fixed_bytes() {  // codes as numbers, the scales of two steps' tiles
  return 2ull * 2 * kTokens * D * 2 + 2 * 2 * (kTokens / 16) * 4;
}
template <int D, int M, bool kTwo>
constexpr size_t query_bytes() {  // of a warp's rows
  return (kTwo ? 2ull : 1ull) * (D / 16) * M * 32 * 16 + 16 * M * sizeof(Row);
}

template <typename T, int D, int M, bool kTwo, int MT>
__global__ void __launch_bounds__(kThreads, 1) cache8_rows_kernel(const __grid_constant__ Cache8Attn p) {
  constexpr int Q2 = kTwo ? 2 : 1, J = D / 16, R = 16 * M;
  constexpr int kTiles = kTokens / 16;
  constexpr int kLoads = kTokens * D / 16 / kThreads;  // of 16 bytes, a thread, of keys
  constexpr int kChunks = D / 8;                       // of 16 bytes in a token's numbers
  extern __shared__ uint4 s_dyn[];
  __shared__ long long s_first[kMaxBatch + 1];
  __shared__ uint8_t s_buckets[kMaxDistances];
  __shared__ float2 s_stats[kRowWarps / 2][R];
  uint4* s_numbers = s_dyn;  // [2 buffers][keys, values][kTokens][kChunks]
  float* s_scale = reinterpret_cast<float*>(s_dyn + 2 * 2 * kTokens * kChunks);  // [2][keys, values][kTiles]
  uint4* s_queries = reinterpret_cast<uint4*>(s_scale + 2 * 2 * kTiles);
  constexpr int kQuery = Q2 * J * M * 32;
  Row* s_rows = reinterpret_cast<Row*>(s_queries + p.row_warps * kQuery);
  float* s_table = reinterpret_cast<float*>(s_rows + p.row_warps * R);

  const Cache8& c = p.c;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, wid = threadIdx.x >> 5;
  const int mine = wid % p.row_warps, group = wid / p.row_warps;
  const int row_tile = blockIdx.y * p.row_warps + mine, row0 = row_tile * R;
  const int unit = blockIdx.x;

  const int biases = p.table == nullptr ? 0 : c.heads * p.group * p.table_stride;
  if (p.table != nullptr) {
    for (int i = threadIdx.x; i < p.distances; i += kThreads) s_buckets[i] = p.buckets[i];
    for (int i = threadIdx.x; i < biases; i += kThreads) {
      const float x = p.table[i];  // (finite ones stay finite)
      s_table[i] = fabsf(x) < INFINITY ? fminf(fmaxf(x * kLog2e, -0x1p126f), 0x1p126f) : x;
    }
  }
  count_tiles<kRowWarps>(p, s_first);
  const long long all = s_first[c.batch];
  const long long piece = max((all + p.pieces - 1) / p.pieces, static_cast<long long>(p.least));
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    for (int i = threadIdx.x; i <= c.batch; i += kThreads) p.first[i] = s_first[i];
    if (threadIdx.x == 0) p.first[c.batch + 1] = piece;
  }
  chain_wait();  // new tokens are written by the kernel in front
  chain_release();
  long long at = unit * piece;
  const long long stop = min(at + piece, all);
  if (at >= stop) return;
  int b = 0;
  for (int step = 1 << 11; step > 0; step >>= 1)  // the last row that begins at or before `at` and holds something
    if (b + step < c.batch && s_first[b + step] <= at) b += step;

  // where this lane's rows of 16 bytes begin: tokens by lane & 7 and a half, chunks by the other half
  const uint32_t numbers_at = static_cast<uint32_t>(__cvta_generic_to_shared(s_numbers));
  const int k_token = (lane & 7) + (lane >> 4) * 8, k_half = lane >> 3 & 1;
  const int v_token = (lane & 7) + (lane >> 3 & 1) * 8, v_half = lane >> 4;
  const uint4* query = s_queries + mine * kQuery;

  while (at < stop) {
    while (s_first[b + 1] <= at) ++b;
    const int start = held_of(c, b), end = end_of(p, start);
    const int tiles = (end + 15) >> 4;
    const int h = static_cast<int>((at - s_first[b]) / (tiles + p.entry));
    const long long seg = s_first[b] + static_cast<long long>(h) * (tiles + p.entry) + p.entry;  // its first tile
    const int tile0 = static_cast<int>(max(at - seg, 0LL));
    const int tile1 = static_cast<int>(min(stop - seg, static_cast<long long>(tiles)));
    if (tile1 <= 0) break;  // (no more than a part of what the beginning costs)
    const long long bh = static_cast<long long>(b) * c.heads + h, slots0 = bh * c.slots;
    const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + b * p.mask_stride;
    const bool placed = p.table != nullptr && c.position != nullptr;

    // ---- codes of a step: 16 bytes a load (a tile past the end is read again, and hidden) ----
    uint4 raw[2][kLoads];
    float scale = 0.f;
    const int from_token = threadIdx.x / (D / 16), from_chunk = threadIdx.x % (D / 16);
    auto load = [&](int tile) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int token = from_token + i * (kThreads / (D / 16));
          const long long s = slots0 + (min(tile + (token >> 4), tile1 - 1) << 4 | (token & 15));
          raw[kv][i] = __ldcg(reinterpret_cast<const uint4*>(c.codes[kv] + s * D) + from_chunk);
        }
      if (threadIdx.x < 2 * kTiles)
        scale = __ldcg(c.absmax[threadIdx.x / kTiles] + bh * (c.slots >> c.block_log2) +
                       (min(tile + static_cast<int>(threadIdx.x % kTiles), tile1 - 1) << 4 >> c.block_log2));
    };
    load(tile0);
    if (group == 0 && row0 < p.rows)
      lay_rows<T, D, M, kTwo>(p, b, h, row0, start, end, s_queries + mine * kQuery, s_rows + mine * R);
    __syncthreads();

    struct {
      float scale;
      int lim;
    } row[M][2];
    int all_see = end - 1;  // slots up to this one are seen by every row of the warp
    if (row0 < p.rows) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const Row& r = s_rows[mine * R + 16 * m + 8 * e + g];
          row[m][e] = {r.scale, r.lim};
          all_see = min(all_see, row[m][e].lim);
        }
    }
    all_see = __reduce_min_sync(0xffffffffu, all_see);
    float o[M][D / 8][4];
    Reference ref[M][2];
    float l[M][2];
#pragma unroll
    for (int m = 0; m < M; ++m) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[m][i][k] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) ref[m][e] = {kNothing, 1.f}, l[m][e] = 0.f;
    }

    int buffer = 0;
    for (int tile = tile0; tile < tile1; tile += kTiles, buffer ^= 1) {
      // ---- the step's codes as numbers; the next one's are requested ----
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int token = from_token + i * (kThreads / (D / 16));
          const uint2 n0 = numbers(raw[kv][i].x), n1 = numbers(raw[kv][i].y), n2 = numbers(raw[kv][i].z), n3 = numbers(raw[kv][i].w);
          const uint4 first = make_uint4(n0.x, n0.y, n1.x, n1.y), second = make_uint4(n2.x, n2.y, n3.x, n3.y);
          uint4* to = s_numbers + ((buffer * 2 + kv) * kTokens + token) * kChunks;
          // (lanes of the upper 128 bytes write the other one first: the banks)
          const int odd = D == 128 ? from_chunk >> 2 : 0;
          to[(2 * from_chunk + odd) ^ (token & 7)] = odd ? second : first;
          to[(2 * from_chunk + 1 - odd) ^ (token & 7)] = odd ? first : second;
        }
      if (threadIdx.x < 2 * kTiles) s_scale[buffer * 2 * kTiles + threadIdx.x] = scale;
      if (tile + kTiles < tile1) load(tile + kTiles);
      __syncthreads();
      if (row0 >= p.rows) continue;

      const int per = kTiles * p.row_warps / kRowWarps;  // tiles of this warp
      const uint32_t keys_at = numbers_at + buffer * 2 * kTokens * kChunks * 16, values_at = keys_at + kTokens * kChunks * 16;
      for (int part = group * per; part < (group + 1) * per; part += MT) {
        if (tile + part >= tile1) break;
        // ---- S = Q K^T ----
        float s[MT][M][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < 8; ++k) s[mt][m][k >> 2][k & 3] = 0.f;
        uint32_t kf[2][MT][4];  // (operands are requested a step ahead of their use)
        uint4 qf[2][Q2][M];
        auto operands = [&](int j) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const int token = (part + mt) * 16 + k_token;
            load_matrices(kf[j & 1][mt], keys_at + (token * kChunks + ((2 * j + k_half) ^ (token & 7))) * 16);
          }
#pragma unroll
          for (int w = 0; w < Q2; ++w)
#pragma unroll
            for (int m = 0; m < M; ++m) qf[j & 1][w][m] = query[((w * J + j) * M + m) * 32 + lane];
        };
        operands(0);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (j + 1 < J) operands(j + 1);
#pragma unroll
          for (int m = 0; m < M; ++m) {
            uint4 q[Q2];
#pragma unroll
            for (int w = 0; w < Q2; ++w) q[w] = qf[j & 1][w][m];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_sum<Q2>(s[mt][m][0], q, kf[j & 1][mt][0], kf[j & 1][mt][1]);
              mma_sum<Q2>(s[mt][m][1], q, kf[j & 1][mt][2], kf[j & 1][mt][3]);
            }
          }
        }

        // ---- scores of tokens 2t + {0, 1} and 8 more, rows g (k = 0, 1) and g + 8 (k = 2, 3) ----
        float va[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int tl = tile + part + mt, s0 = (tl << 4) + 2 * t;
          const bool inside = tl < tile1;
          const float ka = s_scale[buffer * 2 * kTiles + min(part + mt, kTiles - 1)];
          va[mt] = s_scale[buffer * 2 * kTiles + kTiles + min(part + mt, kTiles - 1)];
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < 8; ++k) s[mt][m][k >> 2][k & 3] *= ka * row[m][k >> 1 & 1].scale;
          if (p.table != nullptr) {
            int here[2][2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) here[n][e] = placed ? __ldcg(c.position + slots0 + min(s0 + 8 * n + e, c.slots - 1)) : s0 + 8 * n + e;
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const Row& r = s_rows[mine * R + 16 * m + 8 * (k >> 1 & 1) + g];
                const int d = r.where - here[k >> 2][k & 1];
                s[mt][m][k >> 2][k & 3] += s_table[r.bias + s_buckets[min(max(d, 0), p.distances - 1)]];
              }
          }
          if (!(inside && tl * 16 + 15 <= all_see && mask == nullptr)) {
            bool shown[2][2] = {{inside, inside}, {inside, inside}};
            if (mask != nullptr) {
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int slot = s0 + 8 * n + e;
                  shown[n][e] = inside && slot < p.mask_len && mask[slot] != 0;
                }
            }
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (!shown[k >> 2][k & 1] || s0 + 8 * (k >> 2) + (k & 1) > row[m][k >> 1 & 1].lim) s[mt][m][k >> 2][k & 3] = -INFINITY;
          }
          if (p.scores != nullptr && inside) {
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int r = row0 + 16 * m + 8 * e + g;
                if (r < p.rows) {
                  float* to = p.scores + (bh * p.rows + r) * c.slots + s0;
                  *reinterpret_cast<float2*>(to) = make_float2(s[mt][m][0][2 * e], s[mt][m][0][2 * e + 1]);
                  *reinterpret_cast<float2*>(to + 8) = make_float2(s[mt][m][1][2 * e], s[mt][m][1][2 * e + 1]);
                }
              }
          }
        }

        // ---- references (all tiles of the step in one question: raise_to asks exactly) ----
        float most = va[0];
#pragma unroll
        for (int mt = 1; mt < MT; ++mt) most = fmaxf(most, va[mt]);
        bool raise = false;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int k = 0; k < 4; ++k) top = fmaxf(top, s[mt][m][k >> 1][2 * e + (k & 1)]);
            raise |= beyond(ref[m][e], top, most * ref[m][e].by);
          }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              auto high = [&](int mt) {
                return fmaxf(fmaxf(s[mt][m][0][2 * e], s[mt][m][0][2 * e + 1]), fmaxf(s[mt][m][1][2 * e], s[mt][m][1][2 * e + 1]));
              };
              float x = -INFINITY, term = -INFINITY;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) x = fmaxf(x, high(mt));
#pragma unroll
              for (int lanes = 1; lanes < 4; lanes *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, lanes));
              const float score = raised(ref[m][e], x);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) term = fmaxf(term, high(mt) - score + log2_approx(va[mt]));
#pragma unroll
              for (int lanes = 1; lanes < 4; lanes *= 2) term = fmaxf(term, __shfl_xor_sync(0xffffffffu, term, lanes));
              const float2 by = raise_to(ref[m][e], score, term);
              l[m][e] *= by.x;
#pragma unroll
              for (int i = 0; i < D / 8; ++i) o[m][i][2 * e] *= by.y, o[m][i][2 * e + 1] *= by.y;
            }
        }

        // ---- probabilities, and O += P V ----
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint4 pf[M][Q2];
#pragma unroll
          for (int m = 0; m < M; ++m) {
#pragma unroll
            for (int k = 0; k < 8; ++k) s[mt][m][k >> 2][k & 3] -= ref[m][k >> 1 & 1].score;
            float r[2] = {va[mt] * ref[m][0].by, va[mt] * ref[m][1].by};
            float counts = 1.f;  // in the sum that divides
            if (!(fmaxf(r[0], r[1]) < kFar)) {
              counts = 0.f;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float2 part = part_of(ref[m][e], va[mt]);
                r[e] = part.x;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  float& x = s[mt][m][k >> 1][2 * e + (k & 1)];
                  l[m][e] += exp2_approx(x);
                  x = far_score(x, part.y, va[mt]);
                }
              }
            }
            uint32_t f[Q2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float pr[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const float x = s[mt][m][n][2 * e + k];
                  pr[k] = exp2_approx(x);
                  l[m][e] += pr[k] * counts;
                  pr[k] *= r[e];
                }
                const __half2 v = __floats2half2_rn(pr[0], pr[1]);
                f[0][2 * n + e] = as_u32(v);
                if (kTwo) f[Q2 - 1][2 * n + e] = rest_of(pr[0], pr[1], v);
              }
#pragma unroll
            for (int w = 0; w < Q2; ++w) pf[m][w] = make_uint4(f[w][0], f[w][1], f[w][2], f[w][3]);
          }
          const int token = min(part + mt, kTiles - 1) * 16 + v_token;
          uint32_t vf[2][4];
          auto values = [&](int i) { load_transposed(vf[i & 1], values_at + (token * kChunks + ((2 * i + v_half) ^ (token & 7))) * 16); };
          values(0);
#pragma unroll
          for (int i = 0; i < J; ++i) {
            if (i + 1 < J) values(i + 1);
            const uint32_t(&v)[4] = vf[i & 1];
#pragma unroll
            for (int m = 0; m < M; ++m) {
              mma_sum<Q2, true>(o[m][2 * i], pf[m], v[0], v[1]);
              mma_sum<Q2, true>(o[m][2 * i + 1], pf[m], v[2], v[3]);
            }
          }
        }
      }
    }

    // ---- the warps of the same rows meet: the upper half of them gives its sums to the lower one ----
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[m][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        l[m][e] = sum + __shfl_xor_sync(0xffffffffu, sum, 2);
        const float f = power_of_two(scale_of(ref[m][e])) * (1.f / 127.f);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int k = 0; k < 2; ++k)  // (a row that saw nothing may have sums of 0 * NaN)
            o[m][i][2 * e + k] = l[m][e] == 0.f ? 0.f : o[m][i][2 * e + k] * f;
      }
    for (int groups = kRowWarps / p.row_warps; groups > 1; groups /= 2) {
      const int half = groups / 2, from = wid - half * p.row_warps;  // the warp that this one gives to
      float4* given = reinterpret_cast<float4*>(s_numbers);  // [warps][M * D / 8][32]
      constexpr int kGiven = M * D / 8 * 32;
      __syncthreads();
      if (group >= half && group < groups) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i)
            given[from * kGiven + (m * (D / 8) + i) * 32 + lane] = make_float4(o[m][i][0], o[m][i][1], o[m][i][2], o[m][i][3]);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (t == 0) s_stats[from][16 * m + 8 * e + g] = make_float2(ref[m][e].score, l[m][e]);
        }
      }
      __syncthreads();
      if (group < half) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
          float f[2], other[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 st = s_stats[wid][16 * m + 8 * e + g];
            const float top = fmaxf(ref[m][e].score, st.x);
            f[e] = exp2_approx(ref[m][e].score - top);
            other[e] = exp2_approx(st.x - top);
            ref[m][e].score = top;
            l[m][e] = l[m][e] * f[e] + st.y * other[e];
          }
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const float4 v = given[wid * kGiven + (m * (D / 8) + i) * 32 + lane];
            o[m][i][0] = o[m][i][0] * f[0] + v.x * other[0];
            o[m][i][1] = o[m][i][1] * f[0] + v.y * other[0];
            o[m][i][2] = o[m][i][2] * f[1] + v.z * other[1];
            o[m][i][3] = o[m][i][3] * f[1] + v.w * other[1];
          }
        }
      }
    }

    // The whole (row, head), or a piece of it: a unit has one that began before its own first tile at most, and one that goes
    // on behind its last.
    const bool whole = tile0 == 0 && tile1 == tiles;
    const long long slot = ((static_cast<long long>(row_tile) * p.pieces + unit) * 2 + (tile0 == 0 ? 1 : 0)) * R;
    if (group == 0) {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int in_tile = 16 * m + 8 * e + g, r = row0 + in_tile;
          if (r >= p.rows) continue;
          if (whole) {
            const float inv = l[m][e] == 0.f ? 0.f : 1.f / l[m][e];
            T* dst = out_row<T>(p, b, h, r) + 2 * t;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
              dst[8 * i] = from_float<T>(o[m][i][2 * e] * inv);
              dst[8 * i + 1] = from_float<T>(o[m][i][2 * e + 1] * inv);
            }
            if (t == 0 && p.scores != nullptr) p.final_stats[bh * p.rows + r] = make_float2(ref[m][e].score, inv);
          } else {
            float* dst = p.part + (slot + in_tile) * D + 2 * t;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
              *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[m][i][2 * e], o[m][i][2 * e + 1]);
            if (t == 0) p.stats[slot + in_tile] = make_float2(ref[m][e].score, l[m][e]);
          }
        }
    }
    __syncthreads();  // the next piece's query, codes and scales
    at = seg + tile1;
  }
}

template <typename T, int D, int M, int MT>
cudaError_t launch(const Cache8Attn& p, bool behind, cudaStream_t stream) {
  constexpr bool kTwo = sizeof(T) == 4;
  const size_t table = p.table == nullptr ? 0 : static_cast<size_t>(p.c.heads) * p.group * p.table_stride * 4;
  const size_t fixed = fixed_bytes<D>(), query = query_bytes<D, M, kTwo>();
  static bool set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!set[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(cache8_rows_kernel<T, D, M, kTwo, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(fixed + kRowWarps * query) + kMaxBiases * 4);
    if (e != cudaSuccess) return e;
    set[dev & 63] = true;
  }
  const int row_tiles = (p.rows + 16 * M - 1) / (16 * M);
  const dim3 grid(p.pieces, (row_tiles + p.row_warps - 1) / p.row_warps);
  return launch_behind(behind, cache8_rows_kernel<T, D, M, kTwo, MT>, grid, kThreads, fixed + p.row_warps * query + table, stream, p);
}

// Few rows: 16 a warp, and a tile of tokens at a time (warps that share rows have but one of a step).
template <typename T, int D>
cudaError_t launch_for(const Cache8Attn& p, bool behind, cudaStream_t stream) {
  return p.rows <= kFewRows ? launch<T, D, 1, 1>(p, behind, stream) : launch<T, D, sizeof(T) == 4 ? 1 : 2, 2>(p, behind, stream);
}

}  // namespace

cudaError_t launch_cache8_rows(const Cache8Attn& p, int type, bool behind, cudaStream_t stream) {
  if (p.c.dim == 64)
    return type == 0   ? launch_for<__nv_bfloat16, 64>(p, behind, stream)
           : type == 1 ? launch_for<__half, 64>(p, behind, stream)
                       : launch_for<float, 64>(p, behind, stream);
  return type == 0   ? launch_for<__nv_bfloat16, 128>(p, behind, stream)
         : type == 1 ? launch_for<__half, 128>(p, behind, stream)
                     : launch_for<float, 128>(p, behind, stream);
}

}  // namespace t5x
