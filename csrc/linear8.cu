// Products in 8-bit integers: y = (sum_k cx cw) * sx * sw / 127^2 (+ residual), activations scaled by token (sx, the
// largest |x| of the row, cx = 127 x / sx rounded) and weights by output channel. The sums of products are whole numbers
// below 2^31 for up to 131072 channels and exact. The rest is in 32 bits: the sum's conversion, a scale's division and the product
// with each, the residual's addition, some 2^-21 of the result's parts together; then the rounding to y's type. Scales beyond
// 2^40 or below 2^-40, with which a part of that could leave the normal numbers where y does not, go through 64 bits.
//
// Two launches, for more than two rows: the rows are turned into codes, and tcgen05 (kind::i8, sums in 32 bits in tensor memory)
// multiplies them.
// It runs at twice the rate of bf16, so that a large product has half the time of `native.gemm`; over few rows both are
// bound by the weights' bytes, which are half of bf16's. 8192 x 10240 x 4096: 260 us, 41 for the codes and some 217 for the product
// (3.2 POP/s; the tensor pipe is 91 % busy), 210 at twice the measured rate of bf16. 4096 x 64 x 16384: 58 us, 134 MB of outputs at
// 2.4 TB/s; 16001 outputs 99: what a warp does for a tile is a chain of trips to memory.
#include <algorithm>

#include "cache8.cuh"

namespace t5x {
namespace {

constexpr int kKernelIdLinear8 = 21;
constexpr int kMaxK = 131072;

// Whether sums of products times two such scales stay between 2^-94 and 2^97. (0, and what is not finite, need no care.)
__device__ __forceinline__ bool ordinary(float a) {
  const uint32_t u = __float_as_uint(a);
  return u - (87u << 23) <= (80u << 23) || u == 0 || u >= 0x7f800000u;  // 2^-40 to 2^40
}
// sum * sx * sw / 127^2 + add
__device__ __noinline__ float in_64_bits(int sum, float sx, float sw, float add) {
  double x, w, r;  // (conversions that the build's flags do not let lose numbers below the normal ones)
  asm("cvt.f64.f32 %0, %1;" : "=d"(x) : "f"(sx));
  asm("cvt.f64.f32 %0, %1;" : "=d"(w) : "f"(sw));
  asm("cvt.f64.f32 %0, %1;" : "=d"(r) : "f"(add));
  r += sum * x * w / 16129.0;
  float y;
  asm("cvt.rn.f32.f64 %0, %1;" : "=f"(y) : "d"(r));
  return y;
}
// The same for V values; sx, sw: the largest values of their rows and channels.
template <int V>
__device__ __forceinline__ void scaled(const int (&sum)[V], const float (&sx)[V], const float (&sw)[V], const float (&add)[V],
                                       float (&y)[V]) {
  bool far = false;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    far |= !ordinary(sx[i]) || !ordinary(sw[i]);
    y[i] = static_cast<float>(sum[i]) * (sx[i] * (1.f / 127.f)) * (sw[i] * (1.f / 127.f)) + add[i];
  }
  if (far) {
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = in_64_bits(sum[i], sx[i], sw[i], add[i]);
  }
}

// D (+)= A * B on signed 8-bit integers over a CTA pair, issued by one thread of the even CTA.
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  const uint32_t z = 0;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t"
      "}\n"
      :
      : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(z)
      : "memory");
}
// Instruction descriptor of kind::i8: both operands signed, K-major, sums in signed 32 bits.
__host__ __device__ constexpr uint32_t make_idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// ---------------------------------------------------------------------------
// Rows to codes
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;
constexpr int kRowHeld = 8;  // pieces of 16 bytes that a thread keeps

// One CTA a row, which it reads once where a thread's pieces fit its registers: 16384 values of 16 bits where whole 16 bytes may
// be loaded (kVec), else 4096. `ld` codes a row, those behind the last channel 0. 8192 x 10240 bf16: 42 us for 252 MB, 6.0 TB/s,
// 92 % of the copy rate.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowThreads)
    quantize_rows_kernel(const T* __restrict__ x, long long stride, int k, int ld, int8_t* __restrict__ codes,
                         float* __restrict__ absmax) {
  constexpr int E = 16 / sizeof(T);
  __shared__ uint32_t s_most[kRowThreads / 32];
  const long long row = blockIdx.x;
  const T* src = x + row * stride;
  int8_t* dst = codes + row * ld;
  uint32_t most = 0;
  uint4 held[kVec ? kRowHeld : 1];
  T single[kVec ? 1 : 2 * kRowHeld];
  chain_release();
  if (kVec) {
    uint32_t two = 0;  // of 16-bit values, the largest of each half
#pragma unroll
    for (int i = 0; i < kRowHeld; ++i) {
      const int at = (i * kRowThreads + threadIdx.x) * E;
      if (at < k) held[i] = *reinterpret_cast<const uint4*>(src + at);
    }
#pragma unroll
    for (int i = 0; i < kRowHeld; ++i) {
      const int at = (i * kRowThreads + threadIdx.x) * E;
      if (at < k) {
        const uint32_t w[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (sizeof(T) == 2) two = __vmaxu2(two, w[j] & 0x7fff7fffu);
          else most = max(most, w[j] & 0x7fffffffu);
        }
      }
    }
    if (sizeof(T) == 2) {
      const uint16_t half = static_cast<uint16_t>(max(two >> 16, two & 0xffffu));
      most = abs_bits(to_float(*reinterpret_cast<const T*>(&half)));
    }
  }
  if (!kVec) {
#pragma unroll
    for (int i = 0; i < 2 * kRowHeld; ++i)
      if (i * kRowThreads + static_cast<int>(threadIdx.x) < k) single[i] = src[i * kRowThreads + threadIdx.x];
#pragma unroll
    for (int i = 0; i < 2 * kRowHeld; ++i)
      if (i * kRowThreads + static_cast<int>(threadIdx.x) < k) most = max(most, abs_bits(to_float(single[i])));
  }
  const int rest = min(k, kVec ? kRowHeld * kRowThreads * E : 2 * kRowHeld * kRowThreads);  // from here on read twice
  for (int i = rest + threadIdx.x; i < k; i += kRowThreads) most = max(most, abs_bits(to_float(src[i])));
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) most = max(most, s_most[w]);
  const float a = __uint_as_float(most);
  const Coder code(127.f, a);
  auto of = [&](T v) { return code.template of<sizeof(T) == 2>(to_float(v)); };
  if constexpr (kVec && sizeof(T) == 2) {
    if (code.brief) {
      const uint64_t factor = pair_of(code.factor, code.factor);
#pragma unroll
      for (int i = 0; i < kRowHeld; ++i) {
        const int at = (i * kRowThreads + threadIdx.x) * E;
        if (at < k) {
          const uint4 w = held[i];
          *reinterpret_cast<uint2*>(dst + at) =
              make_uint2(low_bytes(codes_of_two(values_of<T>(w.x), factor), codes_of_two(values_of<T>(w.y), factor)),
                         low_bytes(codes_of_two(values_of<T>(w.z), factor), codes_of_two(values_of<T>(w.w), factor)));
        }
      }
    }
  }
  if (kVec && !(sizeof(T) == 2 && code.brief)) {
#pragma unroll
    for (int i = 0; i < kRowHeld; ++i) {
      const int at = (i * kRowThreads + threadIdx.x) * E;
      if (at < k) {
        const T* v = reinterpret_cast<const T*>(&held[i]);
#pragma unroll
        for (int e = 0; e < E; e += 4) *reinterpret_cast<char4*>(dst + at + e) = make_char4(of(v[e]), of(v[e + 1]), of(v[e + 2]), of(v[e + 3]));
      }
    }
  }
  if (!kVec) {
#pragma unroll
    for (int i = 0; i < 2 * kRowHeld; ++i)
      if (i * kRowThreads + static_cast<int>(threadIdx.x) < k) dst[i * kRowThreads + threadIdx.x] = static_cast<int8_t>(of(single[i]));
  }
  for (int i = rest + threadIdx.x; i < ld; i += kRowThreads) dst[i] = static_cast<int8_t>(i < k ? of(src[i]) : 0);
  if (threadIdx.x == 0) absmax[row] = a;
}

template <typename T>
void launch_rows(const void* x, long long stride, unsigned rows, int k, int ld, int8_t* codes, float* absmax, cudaStream_t stream) {
  const T* src = static_cast<const T*>(x);
  // (rows of whole pieces at multiples of 16 bytes, codes at multiples of 8)
  if (k % (16 / sizeof(T)) == 0 && aligned_to(16, {x}) && stride * sizeof(T) % 16 == 0 && aligned_to(8, {codes}) &&
      ld % 8 == 0)
    quantize_rows_kernel<T, true><<<rows, kRowThreads, 0, stream>>>(src, stride, k, ld, codes, absmax);
  else
    quantize_rows_kernel<T, false><<<rows, kRowThreads, 0, stream>>>(src, stride, k, ld, codes, absmax);
  count_launches(1);
}

// Signals a barrier of the cluster that tensor memory has been read. (Relaxed: it is the fence of tcgen05 in front that orders the
// reads, and a release would wait for all rows that this thread has stored: 7 of 77 us at 4096 x 64 x 16384.)
__device__ __forceinline__ void arrive_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// 32 bytes at a multiple of 32
__device__ __forceinline__ void store_sector(void* to, const uint4& lo, const uint4& hi) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w),
               "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w)
               : "memory");
}

// ---------------------------------------------------------------------------
// The product
// ---------------------------------------------------------------------------
struct Linear8 {
  const float* x_absmax;  // [M]
  const float* w_absmax;  // [N]
  const void* residual;   // [M, N] rows `ld_res` apart, or null
  void* y;                // [M, N] rows N apart
  long long ld_res;
  int M, N, K;            // K: channels, filled up to whole 16
  int tiles_m, tiles_n;
  int vec;                // whole 16 bytes of y and of the residual may be accessed; 2: whole 32 bytes of y
  int* status;
};
struct Linear8Maps {
  CUtensorMap x, w;
};

constexpr int kRows = 128;     // rows of an operand that a CTA stages
constexpr int kTileRows = 256, kTileCols = 256;
constexpr int kBytes = 128;    // channels of a stage
constexpr int kStages = 6;
constexpr int kOperand = kRows * kBytes;
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 64 + 32 * kEpilogueWarps;
constexpr int kPatch = 32 * 33 * 4;  // a warp's 32 x 32 values, rows 33 apart
constexpr int kSmem = kStages * 2 * kOperand + 1024 + 1024 + kEpilogueWarps * kPatch;
static_assert(kSmem <= 232448, "shared memory per CTA");

__device__ __forceinline__ void tile_at(const Linear8& p, int tile, int& mt, int& nt) {
  // eight tiles of rows by all columns at a time: their codes stay in L2 while the weights go by
  const int group = 8 * p.tiles_n, first = tile / group * 8;
  const int high = min(8, p.tiles_m - first), in = tile - tile / group * group;
  mt = first + in % high;
  nt = in / high;
}

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    linear8_kernel(const __grid_constant__ Linear8Maps maps, const __grid_constant__ Linear8 p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_x = smem;
  uint8_t* s_w = smem + kStages * kOperand;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * 2 * kOperand);
  uint64_t* empty = full + kStages;
  uint64_t* tmem_full = empty + kStages;
  uint64_t* tmem_empty = tmem_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* patches = reinterpret_cast<float*>(smem + kStages * 2 * kOperand + 1024);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();  // 0 issues the products
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = p.tiles_m * p.tiles_n, steps = (p.K + kBytes - 1) / kBytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 2 * kEpilogueWarps);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&maps.x);
    tma_prefetch_desc(&maps.w);
  }
  __syncthreads();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are there before anyone signals them
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---- loads: this CTA's 128 rows of the codes and 128 rows of the weights ----
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs) {
        int mt, nt;
        tile_at(p, tile, mt, nt);
        const int m0 = mt * kTileRows + static_cast<int>(cta) * kRows, n0 = nt * kTileCols + static_cast<int>(cta) * kRows;
        for (int k = 0; k < steps; ++k) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag)) {
            report_status(p.status, kStatusTimeoutProducer, kKernelIdLinear8, tile, k);
            *abort_flag = 1;
            ok = false;
            break;
          }
          if (cta == 0) mbar_expect_tx(&full[stage], 4 * kOperand);
          const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);
          tma_load_3d_pair(s_x + stage * kOperand, &maps.x, bar, k * kBytes, m0, 0);
          tma_load_3d_pair(s_w + stage * kOperand, &maps.w, bar, k * kBytes, n0, 0);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---- products ----
    if (lane == 0 && cta == 0) {
      constexpr uint32_t idesc = make_idesc_i8(kTileRows, kTileCols);
      int stage = 0, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < tiles; tile += pairs, ++local) {
        const int acc = local & 1;
        if (!mbar_wait(&tmem_empty[acc], ((local >> 1) & 1) ^ 1, abort_flag)) {
          report_status(p.status, kStatusTimeoutMma, kKernelIdLinear8, tile, -1);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        for (int k = 0; k < steps; ++k) {
          if (!mbar_wait(&full[stage], phase, abort_flag)) {
            report_status(p.status, kStatusTimeoutMma, kKernelIdLinear8, tile, k);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t xa = smem_u32(s_x + stage * kOperand), wa = smem_u32(s_w + stage * kOperand);
#pragma unroll
          for (int s = 0; s < kBytes / 32; ++s)
            umma_i8_pair(tmem + acc * kTileCols, make_smem_desc_sw128(xa + s * 32, 16, 1024),
                         make_smem_desc_sw128(wa + s * 32, 16, 1024), idesc, k > 0 || s > 0);
          umma_commit_pair(&empty[stage], 0x3);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
        if (ok) umma_commit_pair(&tmem_full[acc], 0x3);
      }
    }
  } else {
    // ---- this CTA's 128 rows of the sums: scaled, and stored as whole pieces of rows ----
    const int q = warp & 3, part = (warp - 2) >> 2;  // TMEM lanes 32 q ..; half of the columns
    float* patch = patches + (warp - 2) * (kPatch / 4);
    const uint32_t drained = mapa_shared(smem_u32(&tmem_empty[0]), 0);
    T* y = static_cast<T*>(p.y);
    const T* residual = static_cast<const T*>(p.residual);
    int local = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++local) {
      const int acc = local & 1;
      int mt, nt;
      tile_at(p, tile, mt, nt);
      const int m0 = mt * kTileRows + static_cast<int>(cta) * kRows + q * 32;
      const float most = m0 + lane < p.M ? p.x_absmax[m0 + lane] : 0.f, sx = most * (1.f / 127.f);
      bool far = !ordinary(most);
      const long long row = m0 + lane;
      const int col0 = part * (kTileCols / 2), first = nt * kTileCols + col0;
      constexpr int kBlocks = kTileCols / 64;  // of 32 channels
      float sw[kBlocks];  // the channels' scales
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const int n = first + i * 32 + lane;
        const float most_n = n < p.N ? p.w_absmax[n] : 0.f;
        far |= !ordinary(most_n);
        sw[i] = most_n * (1.f / 127.f);
      }
      if (p.vec == 2) {  // in the patch
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) patch[i * 32 + lane] = sw[i];
        __syncwarp();
      }
      if (!mbar_wait(&tmem_full[acc], (local >> 1) & 1, abort_flag)) {
        if (lane == 0) report_status(p.status, kStatusTimeoutEpilogue, kKernelIdLinear8, tile, 0);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t t_row = tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * kTileCols;
      far = __any_sync(0xffffffffu, far);  // (one value at a time then, below)
      // A lane stores its row's channels where they are whole sectors. (In 32 bits, 4096 x 64 x 16384: 101 us so, 114 by patches; 4096 x
      // 57 x 16004, whole 16 bytes alone: 176 and 130.)
      if (p.vec == 2 && !far) {
        constexpr int E = 16 / sizeof(T), W = sizeof(T) == 4 ? 32 : 64, L = W / E;  // values of 16 bytes, channels at a time, 16 bytes of a lane
#pragma unroll 1
        for (int c = 0; c < kTileCols / 2; c += W) {
          const int n0 = first + c;
          if (n0 >= p.N || m0 >= p.M) break;
          uint4 add[L];
          if (residual != nullptr) {
#pragma unroll
            for (int i = 0; i < L; ++i)
              if (row < p.M && n0 + i * E < p.N) add[i] = *reinterpret_cast<const uint4*>(residual + row * p.ld_res + n0 + i * E);
          }
          uint32_t r[W / 32][32];
          tmem_ld32(t_row + col0 + c, r[0]);
          if (W == 64) tmem_ld32(t_row + col0 + c + 32, r[W / 32 - 1]);
          tmem_ld_wait();
          T* to = y + row * p.N + n0;
#pragma unroll
          for (int i = 0; i < L; i += 2) {
            alignas(16) T o[2 * E];
#pragma unroll
            for (int j = 0; j < 2 * E; j += 4) {
              const int at = i * E + j;
              const float4 sw = *reinterpret_cast<const float4*>(patch + c + at);
              const float ws[4] = {sw.x, sw.y, sw.z, sw.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float v = static_cast<float>(static_cast<int>(r[(at + e) / 32][(at + e) % 32])) * sx * ws[e];
                if (residual != nullptr) v += to_float(reinterpret_cast<const T*>(add)[at + e]);
                o[j + e] = from_float<T>(v);
              }
            }
            const uint4 *lo = reinterpret_cast<const uint4*>(o), *hi = lo + 1;
            if (row < p.M && n0 + i * E < p.N) store_sector(to + i * E, *lo, *hi);
          }
        }
      }
      // Rows at any address: by patches of 32 x 32, a lane a channel. The next sums are requested before these are stored.
      if (p.vec != 2 && !far && first < p.N && m0 < p.M) {
        const int rows = min(32, p.M - m0);
        uint32_t r[32];
        tmem_ld32(t_row + col0, r);
#pragma unroll
        for (int cb = 0; cb < kBlocks; ++cb) {
          const int n0 = first + cb * 32;
          if (n0 >= p.N) break;
          const bool mine = n0 + lane < p.N;
          T add[32];
          if (residual != nullptr && mine) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < rows) add[i] = residual[(m0 + i) * p.ld_res + n0 + lane];
          }
          tmem_ld_wait();
          __syncwarp();  // the patch's last readers are done
#pragma unroll
          for (int j = 0; j < 32; ++j) patch[lane * 33 + j] = static_cast<float>(static_cast<int>(r[j])) * sx;
          __syncwarp();
          if (cb + 1 < kBlocks && n0 + 32 < p.N) tmem_ld32(t_row + col0 + (cb + 1) * 32, r);
          if (mine) {
            T* to = y + static_cast<long long>(m0) * p.N + n0 + lane;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float v = patch[i * 33 + lane] * sw[cb];
              if (residual != nullptr) v += to_float(add[i]);
              if (i < rows) *to = from_float<T>(v);
              to += p.N;
            }
          }
        }
      }
      if (far && m0 < p.M) {
#pragma unroll 1
        for (int n0 = first; n0 < min(first + kTileCols / 2, p.N); n0 += 32) {
          uint32_t r[32];
          tmem_ld32(t_row + col0 + (n0 - first), r);
          tmem_ld_wait();
          __syncwarp();  // the patch's last readers are done
#pragma unroll
          for (int j = 0; j < 32; ++j) patch[lane * 33 + j] = __uint_as_float(r[j]);
          __syncwarp();
          if (n0 + lane >= p.N) continue;
          const float most_n = p.w_absmax[n0 + lane];
#pragma unroll 1
          for (int i = 0; i < min(32, p.M - m0); ++i) {
            const float plus = residual != nullptr ? to_float(residual[(m0 + i) * p.ld_res + n0 + lane]) : 0.f;
            y[static_cast<long long>(m0 + i) * p.N + n0 + lane] =
                from_float<T>(in_64_bits(__float_as_int(patch[i * 33 + lane]), p.x_absmax[m0 + i], most_n, plus));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_relaxed(drained + acc * 8);
    }
  }

  // neither CTA leaves (or frees tensor memory) while its partner may still use its memory or barriers
  __syncwarp();
  if (*abort_flag && warp == 0 && lane == 0)
    for (int it = 0; it < 2000; ++it) __nanosleep(1000);  // ~2 ms for copies in flight to land
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Products of few rows, as of a decode step: bound by the weights' bytes. A cluster takes 128 output channels by NR tokens and
// cuts the input channels into one piece a CTA, so that all SMs stream weights at the same time. The weights are the 128-row
// operand (tokens, of which there may be one, the other), and are requested while the rows are still turned into codes (a
// programmatic dependent launch). The sums, whole numbers, meet through distributed shared memory, in no particular order:
// they are exact. 61 x 4096 x 10240: 15 us with the rows' codes, 6.7 at the copy rate. What a
// CTA begins and ends with (the rows' codes, the sums of a cluster) is as long as the weights take.
// ---------------------------------------------------------------------------
constexpr int kFewThreads = 128;
constexpr int kMaxSplits = 8;  // CTAs of a cluster
// Two CTAs an SM.
template <int NR>
constexpr int few_stages() { return NR <= 32 ? 5 : NR <= 64 ? 4 : 3; }
template <int NR>
constexpr int few_smem() { return few_stages<NR>() * (kOperand + NR * kBytes) + 1024; }
static_assert(2 * (few_smem<32>() + 2048) <= 233472 && 2 * (few_smem<64>() + 2048) <= 233472 && 2 * (few_smem<128>() + 2048) <= 233472,
              "two CTAs an SM");

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ int4 remote_int4(const int* mine, uint32_t cta) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(mapa_shared(smem_u32(mine), cta))
               : "memory");
  return v;
}
__device__ __forceinline__ int remote_int(const int* mine, uint32_t cta) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(mine), cta)) : "memory");
  return v;
}
// 32 lanes x 16 columns
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

template <typename T, int NR>
__global__ void __launch_bounds__(kFewThreads)
    linear8_few_kernel(const __grid_constant__ Linear8Maps maps, const __grid_constant__ Linear8 p, int splits) {
  static_assert(few_smem<NR>() >= 1024 + NR * 128 * 4, "the sums take the place of the stages");
  constexpr int kFewStages = few_stages<NR>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_w = smem;
  uint8_t* s_x = smem + kFewStages * kOperand;
  __shared__ uint64_t full[kFewStages], empty[kFewStages], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_word;
  volatile int* abort_flag = &abort_word;
  constexpr int kColumns = NR < 32 ? 32 : NR;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int piece = static_cast<int>(cluster_ctarank());
  const int n0 = static_cast<int>(blockIdx.x / splits) * kRows, m0 = blockIdx.y * NR;
  const int steps = (p.K + kBytes - 1) / kBytes, per = (steps + splits - 1) / splits;
  const int k0 = min(piece * per, steps), k1 = min(k0 + per, steps);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    abort_word = 0;
    mbar_fence_init();
    tma_prefetch_desc(&maps.x);
    tma_prefetch_desc(&maps.w);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0 && lane == 0) {
    constexpr uint32_t kStage = kOperand + NR * kBytes;
    const int ahead = min(kFewStages, k1 - k0);
    for (int i = 0; i < ahead; ++i) {
      mbar_expect_tx(&full[i], kStage);
      tma_load_3d(s_w + i * kOperand, &maps.w, &full[i], (k0 + i) * kBytes, n0, 0);
    }
    chain_wait();  // the codes are the kernel's in front
    for (int i = 0; i < ahead; ++i) tma_load_3d(s_x + i * NR * kBytes, &maps.x, &full[i], (k0 + i) * kBytes, m0, 0);
    for (int i = ahead; i < k1 - k0; ++i) {
      const int stage = i % kFewStages;
      if (!mbar_wait(&empty[stage], (i / kFewStages - 1) & 1, abort_flag)) {
        report_status(p.status, kStatusTimeoutProducer, kKernelIdLinear8, n0, i);
        *abort_flag = 1;
        break;
      }
      mbar_expect_tx(&full[stage], kStage);
      tma_load_3d(s_w + stage * kOperand, &maps.w, &full[stage], (k0 + i) * kBytes, n0, 0);
      tma_load_3d(s_x + stage * NR * kBytes, &maps.x, &full[stage], (k0 + i) * kBytes, m0, 0);
    }
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = make_idesc_i8(kRows, NR);
    bool ok = true;
    for (int i = 0; i < k1 - k0; ++i) {
      const int stage = i % kFewStages;
      if (!mbar_wait(&full[stage], (i / kFewStages) & 1, abort_flag)) {
        report_status(p.status, kStatusTimeoutMma, kKernelIdLinear8, n0, i);
        *abort_flag = 1;
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t wa = smem_u32(s_w + stage * kOperand), xa = smem_u32(s_x + stage * NR * kBytes);
#pragma unroll
      for (int s = 0; s < kBytes / 32; ++s)
        umma_i8(tmem, make_smem_desc_sw128(wa + s * 32, 16, 1024), make_smem_desc_sw128(xa + s * 32, 16, 1024), idesc, i > 0 || s > 0);
      umma_commit(&empty[stage]);
    }
    if (ok) umma_commit(&done);
  }
  __syncwarp();
  chain_wait();  // the rows' scales are read below
  bool good = true;
  if (k1 > k0) {
    good = mbar_wait(&done, 0, abort_flag);
    if (!good) {
      if (lane == 0) report_status(p.status, kStatusTimeoutEpilogue, kKernelIdLinear8, n0, 0);
      *abort_flag = 1;
    }
  }
  tc_fence_after();
  // The sums by token and channel, over the stages: all of them have been read (`done`). (After a wait that ran out copies may
  // still land there: nothing is written then.)
  int* s_sums = reinterpret_cast<int*>(smem);
  if (good) {
#pragma unroll
    for (int c = 0; c < NR; c += 16) {
      uint32_t r[16];
      if (k1 > k0) {
        tmem_ld16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, r);
        tmem_ld_wait();
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) s_sums[(c + j) * 128 + threadIdx.x] = k1 > k0 ? static_cast<int>(r[j]) : 0;
    }
  } else if (lane == 0) {
    for (int it = 0; it < 2000; ++it) __nanosleep(1000);  // ~2 ms for copies in flight to land
  }
  tc_fence_before();
  cluster_sync_all();

  // each CTA of the cluster finishes a share of the tokens
  T* y = static_cast<T*>(p.y);
  const T* residual = static_cast<const T*>(p.residual);
  const int tokens = min(NR, p.M - m0);
  if (p.vec) {  // four channels a thread (there are whole fours of them)
    for (int i = piece * kFewThreads + threadIdx.x; i < tokens * 32; i += splits * kFewThreads) {
      const int tok = i >> 5, ch = (i & 31) * 4, n = n0 + ch;
      if (n >= p.N) continue;
      int4 v[kMaxSplits], sum = make_int4(0, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < kMaxSplits; ++r)
        if (r < splits) v[r] = remote_int4(s_sums + tok * 128 + ch, r);
      const long long row = m0 + tok;
      float add[4] = {0.f, 0.f, 0.f, 0.f};
      if (residual != nullptr) load_four(residual + row * p.ld_res + n, true, add);
      const float most = ld_chained(p.x_absmax + row);
      const float sx[4] = {most, most, most, most};
      const float sw[4] = {p.w_absmax[n], p.w_absmax[n + 1], p.w_absmax[n + 2], p.w_absmax[n + 3]};
#pragma unroll
      for (int r = 0; r < kMaxSplits; ++r)
        if (r < splits) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
      const int sums[4] = {sum.x, sum.y, sum.z, sum.w};
      float out[4];
      scaled(sums, sx, sw, add, out);
      alignas(16) T o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = from_float<T>(out[k]);
      if (sizeof(T) == 4) *reinterpret_cast<uint4*>(y + row * p.N + n) = *reinterpret_cast<uint4*>(o);
      else *reinterpret_cast<uint2*>(y + row * p.N + n) = *reinterpret_cast<uint2*>(o);
    }
  } else if (n0 + static_cast<int>(threadIdx.x) < p.N) {  // one channel a thread, four tokens at a time
    const int n = n0 + threadIdx.x;
    const float most_n = p.w_absmax[n];
    constexpr int U = 4;
    for (int tok = piece * U; tok < tokens; tok += splits * U) {
      int v[U][kMaxSplits], sum[U];
      float add[U], sx[U], sw[U], out[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long row = m0 + min(tok + u, tokens - 1);
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r)
          if (r < splits) v[u][r] = remote_int(s_sums + (tok + u) * 128 + threadIdx.x, r);
        add[u] = residual != nullptr ? to_float(residual[row * p.ld_res + n]) : 0.f;
        sx[u] = ld_chained(p.x_absmax + row);
        sw[u] = most_n;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        sum[u] = 0;
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r)
          if (r < splits) sum[u] += v[u][r];
      }
      scaled(sum, sx, sw, add, out);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (tok + u < tokens) y[(m0 + tok + u) * static_cast<long long>(p.N) + n] = from_float<T>(out[u]);
    }
  }
  cluster_sync_all();  // nobody leaves while others read its sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kColumns);
  }
}

// ---------------------------------------------------------------------------
// One row or two in one launch: each CTA turns them into codes for itself (they are in L2), behind its first requests for
// weights; two CTAs an SM take output channels in turn, two a warp, 512 bytes of both at a time, by dot products of four bytes. The
// weights' bytes bound it: 1 x 4096 x 32128 takes 21.8 us, 92 % of the copy rate.
// ---------------------------------------------------------------------------
constexpr int kOneThreads = 256;
constexpr int kOneWarps = kOneThreads / 32;
constexpr int kOneChannels = 2;          // of a warp
constexpr int kOneHeld = 4;              // pieces of 16 bytes of a row that a thread keeps

template <typename T, int R>
__global__ void __launch_bounds__(kOneThreads)
    linear8_one_kernel(const __grid_constant__ Linear8 p, const T* __restrict__ x, long long stride, int k, int vec,
                       const int8_t* __restrict__ w) {
  constexpr int E = 16 / sizeof(T), C = kOneChannels, U = 4;  // steps of 512 bytes requested at a time
  constexpr int kHeld = kOneHeld;
  extern __shared__ uint4 s_codes[];                          // [R][K / 16]
  __shared__ uint32_t s_most[R][kOneWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pieces = p.K / 16, stride_n = gridDim.x * kOneWarps * C;
  int n0 = (blockIdx.x * kOneWarps + warp) * C;
  uint4 next[U][C];
  auto request = [&](int n, int at) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const uint4* row = reinterpret_cast<const uint4*>(w + static_cast<long long>(min(n + c, p.N - 1)) * p.K);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (at + u * 32 + lane < pieces) next[u][c] = __ldcs(row + at + u * 32 + lane);
    }
  };
  if (n0 < p.N) request(n0, 0);

  // ---- codes ----
  uint4 held[R][kHeld];
  const int whole = vec ? min(k, kHeld * kOneThreads * E) : 0;  // values in registers; the rest is read twice
  uint32_t most[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    most[r] = 0;
    {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int at = (i * kOneThreads + threadIdx.x) * E;
        if (at < whole) held[r][i] = *reinterpret_cast<const uint4*>(x + r * stride + at);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if ((i * kOneThreads + static_cast<int>(threadIdx.x)) * E < whole) {
          const T* v = reinterpret_cast<const T*>(&held[r][i]);
#pragma unroll
          for (int e = 0; e < E; ++e) most[r] = max(most[r], abs_bits(to_float(v[e])));
        }
      for (int i = whole + threadIdx.x; i < k; i += kOneThreads) most[r] = max(most[r], abs_bits(to_float(x[r * stride + i])));
    }
    most[r] = __reduce_max_sync(0xffffffffu, most[r]);
    if (lane == 0) s_most[r][warp] = most[r];
  }
  __syncthreads();
  float scale[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int i = 0; i < kOneWarps; ++i) most[r] = max(most[r], s_most[r][i]);
    const float a = __uint_as_float(most[r]);
    scale[r] = a;
    {
      const Coder code(127.f, a);
      auto of = [&](T v) { return code.template of<sizeof(T) == 2>(to_float(v)); };
      int8_t* dst = reinterpret_cast<int8_t*>(s_codes) + r * p.K;
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int at = (i * kOneThreads + threadIdx.x) * E;
        if (at < whole) {
          const T* v = reinterpret_cast<const T*>(&held[r][i]);
#pragma unroll
          for (int e = 0; e < E; e += 4) *reinterpret_cast<char4*>(dst + at + e) = make_char4(of(v[e]), of(v[e + 1]), of(v[e + 2]), of(v[e + 3]));
        }
      }
      for (int i = whole + threadIdx.x; i < p.K; i += kOneThreads) dst[i] = static_cast<int8_t>(i < k ? of(x[r * stride + i]) : 0);
    }
  }
  __syncthreads();

  // ---- products ----
  for (; n0 < p.N; n0 += stride_n) {
    int sum[R][C];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) sum[r][c] = 0;
    for (int at = 0; at < pieces; at += U * 32) {
      uint4 here[U][C];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c) here[u][c] = next[u][c];
      if (at + U * 32 < pieces) request(n0, at + U * 32);
      else if (n0 + stride_n < p.N) request(n0 + stride_n, 0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int piece = at + u * 32 + lane;
        if (piece >= pieces) break;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint4 q = s_codes[r * pieces + piece];
#pragma unroll
          for (int c = 0; c < C; ++c) {
            sum[r][c] = __dp4a(static_cast<int>(here[u][c].x), static_cast<int>(q.x), sum[r][c]);
            sum[r][c] = __dp4a(static_cast<int>(here[u][c].y), static_cast<int>(q.y), sum[r][c]);
            sum[r][c] = __dp4a(static_cast<int>(here[u][c].z), static_cast<int>(q.z), sum[r][c]);
            sum[r][c] = __dp4a(static_cast<int>(here[u][c].w), static_cast<int>(q.w), sum[r][c]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int all = __reduce_add_sync(0xffffffffu, sum[r][c]), n = n0 + c;
        if (lane == r * C + c && n < p.N) {
          const float add = p.residual != nullptr ? to_float(static_cast<const T*>(p.residual)[r * p.ld_res + n]) : 0.f;
          float out[1];
          scaled({all}, {scale[r]}, {p.w_absmax[n]}, {add}, out);
          static_cast<T*>(p.y)[r * static_cast<long long>(p.N) + n] = from_float<T>(out[0]);
        }
      }
  }
}

bool alone(int rows, int k) { return rows == 1 && k <= 32768; }  // a row that needs no workspace, whatever its type

template <typename T, int R>
cudaError_t launch_one(const T* x, long long stride, int k, const void* w, const Linear8& p, cudaStream_t stream) {
  const int vec = k % (16 / static_cast<int>(sizeof(T))) == 0 && aligned_to(16, {x}) && stride * static_cast<long long>(sizeof(T)) % 16 == 0;
  const int channels = kOneWarps * kOneChannels, most = 2 * num_sms();
  linear8_one_kernel<T, R><<<std::min((p.N + channels - 1) / channels, most), kOneThreads, static_cast<size_t>(R) * p.K, stream>>>(
      p, x, stride, k, vec, static_cast<const int8_t*>(w));
  count_launches(1);
  return cudaGetLastError();
}

bool map_of(CUtensorMap* map, const void* codes, int rows, int k, uint32_t box_rows = kRows) {
  const uint64_t dims[3] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(k) * rows};
  const uint32_t box[3] = {kBytes, box_rows, 1};
  return get_tensor_map(map, codes, 1, 3, dims, strides, box, 1);
}

template <typename T, int NR>
cudaError_t launch_few(const Linear8Maps& maps, const Linear8& p, int splits, cudaStream_t stream) {
  static bool set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!set[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(linear8_few_kernel<T, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, few_smem<NR>());
    if (e != cudaSuccess) return e;
    set[dev & 63] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + kRows - 1) / kRows * splits, (p.M + NR - 1) / NR);
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = few_smem<NR>();
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  count_launches(1);
  return cudaLaunchKernelEx(&cfg, linear8_few_kernel<T, NR>, maps, p, splits);
}

template <typename T>
int launch(const void* x, long long stride, int k, int8_t* codes, const void* w, Linear8 p, cudaStream_t stream) {
  // us in one launch / as below, rows x in x out: 1 x 1024 x 2816 3.1 / 5.4, 1 x 4096 x 10240 9.9 / 12.4, 1 x 10240 x 4096 11.1 /
  // 12.4, 2 x 1024 x 2816 4.2 / 5.4, 2 x 4096 x 32128 23.5 / 25.8, 2 x 10240 x 4096 (two rows of which a CTA reads a part twice)
  // 13.8 / 12.3; four rows 6 to 11 / 5.5.
  constexpr int kOneValues = kOneHeld * kOneThreads * 16 / static_cast<int>(sizeof(T));  // of a row in a CTA's registers
  if (alone(p.M, p.K) || (p.M == 2 && p.K <= kOneValues)) {
    const T* rows = static_cast<const T*>(x);
    const cudaError_t e = p.M == 1   ? launch_one<T, 1>(rows, stride, k, w, p, stream)
                                     : launch_one<T, 2>(rows, stride, k, w, p, stream);
    return e == cudaSuccess ? 0 : set_error("linear8 launch: %s", cudaGetErrorString(e));
  }
  float* absmax = const_cast<float*>(p.x_absmax);
  launch_rows<T>(x, stride, p.M, k, p.K, codes, absmax, stream);
  Linear8Maps maps;
  p.tiles_m = (p.M + kTileRows - 1) / kTileRows;
  p.tiles_n = (p.N + kTileCols - 1) / kTileCols;
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
  const int nr = p.M <= 16 ? 16 : p.M <= 32 ? 32 : p.M <= 64 ? 64 : 128;
  const long long all = static_cast<long long>((p.N + kRows - 1) / kRows) * ((p.M + nr - 1) / nr);
  // One tile of tokens, or fewer tiles than SMs. us so / in tiles of 256 x 256, rows x in x out: 1 x 4096 x 32128 26 / 41,
  // 61 x 4096 x 32128 33 / 36, 128 x 4096 x 20480 35 / 36, 128 x 4096 x 32128 41 / 39, 200 x 4096 x 4096 13 / 20, 200 x 4096 x
  // 10240 31 / 23, 509 x 4096 x 4096 20 / 21, 1024 x 1024 x 2816 23 / 15.
  if (p.M <= 128 || all <= num_sms()) {
    if (!map_of(&maps.x, codes, p.M, p.K, nr) || !map_of(&maps.w, w, p.N, p.K)) return -1;
    // as many pieces of the input channels as there are CTAs for at a time (two an SM), of two steps at least
    const int steps = (p.K + kBytes - 1) / kBytes;
    const int splits = static_cast<int>(std::max(1LL, std::min({2LL * num_sms() / all, steps / 2LL, static_cast<long long>(kMaxSplits)})));
    const cudaError_t e = nr == 16   ? launch_few<T, 16>(maps, p, splits, stream)
                          : nr == 32 ? launch_few<T, 32>(maps, p, splits, stream)
                          : nr == 64 ? launch_few<T, 64>(maps, p, splits, stream)
                                     : launch_few<T, 128>(maps, p, splits, stream);
    return e == cudaSuccess ? 0 : set_error("linear8 launch: %s", cudaGetErrorString(e));
  }
  if (!map_of(&maps.x, codes, p.M, p.K) || !map_of(&maps.w, w, p.N, p.K)) return -1;
  static bool set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e;
  if (!set[dev & 63]) {
    e = cudaFuncSetAttribute(linear8_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return set_error("linear8: %s", cudaGetErrorString(e));
    set[dev & 63] = true;
  }
  const int pairs = static_cast<int>(std::min<long long>(num_sms() / 2, tiles));
  linear8_kernel<T><<<2 * pairs, kThreads, kSmem, stream>>>(maps, p);
  count_launches(1);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : set_error("linear8 launch: %s", cudaGetErrorString(e));
}

}  // namespace
}  // namespace t5x

T5X_API int t5x_quantize_rows(const void* x, int type, long long rows, int k, long long stride, void* codes, int ld,
                              void* absmax, void* stream) {
  if (rows < 0 || rows > 0x7fffffffLL || k < 1 || ld < k || type < 0 || type > 2)
    return t5x::set_error("quantize_rows: %lld rows of %d values, type %d", rows, k, type);
  if (rows == 0) return 0;
  if (!x || !codes || !absmax || !t5x::aligned_to(type == 2 ? 4 : 2, {x}) || !t5x::aligned_to(4, {absmax}))
    return t5x::set_error("quantize_rows: a null or misaligned pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int8_t* c = static_cast<int8_t*>(codes);
  float* a = static_cast<float*>(absmax);
  const unsigned grid = static_cast<unsigned>(rows);
  if (type == 0) t5x::launch_rows<__nv_bfloat16>(x, stride, grid, k, ld, c, a, st);
  else if (type == 1) t5x::launch_rows<__half>(x, stride, grid, k, ld, c, a, st);
  else t5x::launch_rows<float>(x, stride, grid, k, ld, c, a, st);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : t5x::set_error("quantize_rows launch: %s", cudaGetErrorString(e));
}

T5X_API long long t5x_linear8_workspace_bytes(int rows, int k) {
  if (t5x::alone(rows, (k + 15) / 16 * 16)) return 0;
  return (static_cast<long long>(rows) * ((k + 15) / 16 * 16) + 127) / 128 * 128 + static_cast<long long>(rows) * 4;
}

T5X_API int t5x_linear8(const void* x, int type, int rows, int k, long long stride, const void* w, const void* w_absmax,
                        int n, const void* residual, long long ld_res, void* y, void* workspace, void* stream) {
  if (rows < 0 || k < 1 || k > t5x::kMaxK || n < 1 || type < 0 || type > 2 ||
      static_cast<long long>((rows + 255LL) / 256) * ((n + 255LL) / 256) > 0x7fffffffLL)
    return t5x::set_error("linear8: %d rows, %d -> %d channels (at most %d), type %d", rows, k, n, t5x::kMaxK, type);
  if (rows == 0) return 0;
  const int size = type == 2 ? 4 : 2;
  if (!x || !w || !w_absmax || !y || (!workspace && t5x_linear8_workspace_bytes(rows, k) > 0) ||
      !t5x::aligned_to(size, {x, y, residual}) || !t5x::aligned_to(16, {w, workspace}) || !t5x::aligned_to(4, {w_absmax}))
    return t5x::set_error("linear8: a null or misaligned pointer");
  t5x::Linear8 p = {};
  p.M = rows;
  p.N = n;
  p.K = (k + 15) / 16 * 16;
  int8_t* codes = static_cast<int8_t*>(workspace);
  p.x_absmax = reinterpret_cast<float*>(codes + (static_cast<long long>(rows) * p.K + 127) / 128 * 128);
  p.w_absmax = static_cast<const float*>(w_absmax);
  p.residual = residual;
  p.ld_res = ld_res;
  p.y = y;
  p.vec = n * static_cast<long long>(size) % 16 == 0 && t5x::aligned_to(16, {y, residual}) &&
          (residual == nullptr || ld_res * size % 16 == 0);
  if (p.vec && n * static_cast<long long>(size) % 32 == 0 && t5x::aligned_to(32, {y})) p.vec = 2;
  p.status = t5x::device_status_buffer();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (type) {
    case 0: return t5x::launch<__nv_bfloat16>(x, stride, k, codes, w, p, st);
    case 1: return t5x::launch<__half>(x, stride, k, codes, w, p, st);
    default: return t5x::launch<float>(x, stride, k, codes, w, p, st);
  }
}
