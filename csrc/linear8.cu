// Products in 8-bit integers: y = (sum_k cx cw) * sx * sw / 127^2 (+ residual), activations scaled by token (sx, the
// largest |x| of the row, cx = 127 x / sx rounded) and weights by output channel. The sums of products are whole numbers
// below 2^31 for up to 131072 channels and exact; one rounding at the end.
//
// Two kernels: the rows are turned into codes, and tcgen05 (kind::i8, sums in 32 bits in tensor memory) multiplies them.
// It runs at twice the rate of bf16, so that a large product has half the time of `native.gemm`; over few rows both are
// bound by the weights' bytes, which are half of bf16's.
#include <algorithm>

#include "cache8.cuh"

namespace t5x {
namespace {

constexpr int kKernelIdLinear8 = 21;
constexpr int kMaxK = 131072;

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

// One CTA a row; `ld` codes a row, those behind the last channel 0.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
    quantize_rows_kernel(const T* __restrict__ x, long long stride, int k, int ld, int8_t* __restrict__ codes,
                         float* __restrict__ absmax) {
  __shared__ uint32_t s_most[kRowThreads / 32];
  const long long row = blockIdx.x;
  const T* src = x + row * stride;
  uint32_t most = 0;
  for (int i = threadIdx.x; i < k; i += kRowThreads) most = max(most, abs_bits(to_float(src[i])));
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) most = max(most, s_most[w]);
  const float a = __uint_as_float(most);
  const Coder code(127.f, a);
  for (int i = threadIdx.x; i < ld; i += kRowThreads)
    codes[row * ld + i] = static_cast<int8_t>(i < k ? code.template of<sizeof(T) == 2>(to_float(src[i])) : 0);
  if (threadIdx.x == 0) absmax[row] = a;
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
  int vec;                // whole 16 bytes of y and of the residual may be accessed
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
      const float sx = m0 + lane < p.M ? p.x_absmax[m0 + lane] * (1.f / 127.f) : 0.f;
      if (!mbar_wait(&tmem_full[acc], (local >> 1) & 1, abort_flag)) {
        if (lane == 0) report_status(p.status, kStatusTimeoutEpilogue, kKernelIdLinear8, tile, 0);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t t_row = tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * kTileCols;
      for (int cb = 0; cb < kTileCols / 64; ++cb) {
        const int col = part * (kTileCols / 2) + cb * 32, n0 = nt * kTileCols + col;
        if (n0 >= p.N || m0 >= p.M) break;
        const float sw = n0 + lane < p.N ? p.w_absmax[n0 + lane] * (1.f / 127.f) : 0.f;
        uint32_t r[32];
        tmem_ld32(t_row + col, r);
        tmem_ld_wait();
        __syncwarp();  // the patch's last readers are done
#pragma unroll
        for (int j = 0; j < 32; ++j)
          patch[lane * 33 + j] = static_cast<float>(static_cast<int>(r[j])) * sx * __shfl_sync(0xffffffffu, sw, j);
        __syncwarp();
        const int rows = min(32, p.M - m0);
        if (p.vec && n0 + 32 <= p.N) {
          constexpr int E = 16 / sizeof(T), L = 32 / E;  // values a lane stores at a time, lanes a row
          const int j = lane % L * E;
          for (int i = lane / L; i < rows; i += 32 / L) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = patch[i * 33 + j + e];
            alignas(16) T o[E];
            if (residual != nullptr) {
              *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(residual + (m0 + i) * p.ld_res + n0 + j);
#pragma unroll
              for (int e = 0; e < E; ++e) v[e] += to_float(o[e]);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = from_float<T>(v[e]);
            *reinterpret_cast<uint4*>(y + static_cast<long long>(m0 + i) * p.N + n0 + j) = *reinterpret_cast<uint4*>(o);
          }
        } else if (n0 + lane < p.N) {
          for (int i = 0; i < rows; ++i) {
            float v = patch[i * 33 + lane];
            if (residual != nullptr) v += to_float(residual[(m0 + i) * p.ld_res + n0 + lane]);
            y[static_cast<long long>(m0 + i) * p.N + n0 + lane] = from_float<T>(v);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(drained + acc * 8);
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

bool map_of(CUtensorMap* map, const void* codes, int rows, int k) {
  const uint64_t dims[3] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows), 1};
  const uint64_t strides[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(k) * rows};
  const uint32_t box[3] = {kBytes, kRows, 1};
  return get_tensor_map(map, codes, 1, 3, dims, strides, box, 1);
}

template <typename T>
int launch(const void* x, long long stride, int k, int8_t* codes, const void* w, Linear8 p, cudaStream_t stream) {
  float* absmax = const_cast<float*>(p.x_absmax);
  quantize_rows_kernel<T><<<p.M, kRowThreads, 0, stream>>>(static_cast<const T*>(x), stride, k, p.K, codes, absmax);
  count_launches(1);
  Linear8Maps maps;
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
  p.tiles_m = (p.M + kTileRows - 1) / kTileRows;
  p.tiles_n = (p.N + kTileCols - 1) / kTileCols;
  const long long tiles = static_cast<long long>(p.tiles_m) * p.tiles_n;
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
  if (type == 0)
    t5x::quantize_rows_kernel<<<grid, t5x::kRowThreads, 0, st>>>(static_cast<const __nv_bfloat16*>(x), stride, k, ld, c, a);
  else if (type == 1)
    t5x::quantize_rows_kernel<<<grid, t5x::kRowThreads, 0, st>>>(static_cast<const __half*>(x), stride, k, ld, c, a);
  else
    t5x::quantize_rows_kernel<<<grid, t5x::kRowThreads, 0, st>>>(static_cast<const float*>(x), stride, k, ld, c, a);
  t5x::count_launches(1);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : t5x::set_error("quantize_rows launch: %s", cudaGetErrorString(e));
}

T5X_API long long t5x_linear8_workspace_bytes(int rows, int k) {
  return (static_cast<long long>(rows) * ((k + 15) / 16 * 16) + 127) / 128 * 128 + static_cast<long long>(rows) * 4;
}

T5X_API int t5x_linear8(const void* x, int type, int rows, int k, long long stride, const void* w, const void* w_absmax,
                        int n, const void* residual, long long ld_res, void* y, void* workspace, void* stream) {
  if (rows < 0 || k < 1 || k > t5x::kMaxK || n < 1 || type < 0 || type > 2 ||
      static_cast<long long>((rows + 255LL) / 256) * ((n + 255LL) / 256) > 0x7fffffffLL)
    return t5x::set_error("linear8: %d rows, %d -> %d channels (at most %d), type %d", rows, k, n, t5x::kMaxK, type);
  if (rows == 0) return 0;
  const int size = type == 2 ? 4 : 2;
  if (!x || !w || !w_absmax || !y || !workspace || !t5x::aligned_to(size, {x, y, residual}) ||
      !t5x::aligned_to(16, {w, workspace}) || !t5x::aligned_to(4, {w_absmax}))
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
  p.status = t5x::device_status_buffer();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (type) {
    case 0: return t5x::launch<__nv_bfloat16>(x, stride, k, codes, w, p, st);
    case 1: return t5x::launch<__half>(x, stride, k, codes, w, p, st);
    default: return t5x::launch<float>(x, stride, k, codes, w, p, st);
  }
}
