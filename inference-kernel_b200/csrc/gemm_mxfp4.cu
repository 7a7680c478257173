// Product of two microscaled 4-bit matrices: C[m, n] = sum_k A[m, k] B[n, k],
// A [M, K / 2] and B [N, K / 2] codes with scale tiles as in mxfp4.cu, fp32
// accumulation, one rounding to the output type.
//
// Persistent tcgen05 kernel, one CTA per SM, 128 x BN tiles of C:
//   * codes are read as bytes by TMA, 256 elements of K (one 128-byte swizzle
//     row) per stage, both operands K-major; scale tiles (512 bytes per 128
//     rows x 4 blocks, already in the order of TMEM) by untiled bulk copies;
//   * per stage the MMA thread copies the scales to TMEM and issues up to four
//     K = 64 MMAs (kind::mxf4).  TMEM holds one scale area per stage of the
//     ring, so a stage's scales are overwritten only when its barrier has shown
//     that the MMAs which read them are done;
//   * two accumulators, so that a tile's read-out overlaps the next tile's
//     MMAs.  At BN = 256 they and the scales do not fit into the 512 columns
//     side by side: they overlap by 96 columns, which each read-out empties
//     first (accumulator 0 from its top, 1 from its bottom).
// A block of zeros pads K (TMA zero fill); MMAs stop at the last 64 elements
// that exist.  Rows beyond M or N may multiply stale scales, and are not stored.
#include <type_traits>

#include "common.h"
#include "gemm_internal.h"
#include "sm100.cuh"
#include "tmap.h"
#include "vec.cuh"

namespace aotk {
namespace {

using namespace sm100;

__device__ unsigned g_mx_watchdog;

constexpr int kBM = 128;
constexpr int kBK = 256;       // elements of K per stage (128 bytes of codes)
constexpr int kStepK = 64;     // elements of K per MMA
constexpr int kThreads = 192;  // producer, MMA and 4 epilogue warps
constexpr int kGroupM = 16;    // M tiles per raster group
constexpr uint32_t kScaleTile = 512;

enum : unsigned { kWdProducer = 4096u, kWdMma = 8192u, kWdEpilogue = 16384u };

template <int BN, int STAGES>
struct MxLayout {
  static constexpr int kScaleTilesN = BN > 128 ? 2 : 1;  // scale tiles along N
  static constexpr uint32_t kABytes = kBM * 128;
  static constexpr uint32_t kBBytes = BN * 128;
  static constexpr uint32_t kSfaBytes = 2 * kScaleTile;
  static constexpr uint32_t kSfbBytes = kScaleTilesN * 2 * kScaleTile;
  static constexpr uint32_t kOffA = 0;
  static constexpr uint32_t kOffB = kOffA + STAGES * kABytes;
  static constexpr uint32_t kOffSfa = kOffB + STAGES * kBBytes;
  static constexpr uint32_t kOffSfb = kOffSfa + STAGES * kSfaBytes;
  static constexpr uint32_t kCBuf = 32 * 128;
  static constexpr uint32_t kOffC = kOffSfb + STAGES * kSfbBytes;
  static constexpr uint32_t kOffBar = kOffC + 4 * kCBuf;
  static constexpr uint32_t kNumBars = 2 * STAGES + 5;  // full, empty, tfull x2, release x2, drain
  static constexpr uint32_t kOffMisc = kOffBar + kNumBars * 8;
  static constexpr uint32_t kAlloc = kOffMisc + 16 + 1024;
  static_assert(kAlloc <= 232448, "227 KB of shared memory");
  // TMEM columns: accumulators, then 4 columns per scale tile and stage.
  static constexpr int kSfCols = 2 * 4 * (1 + kScaleTilesN);
  static constexpr bool kOverlap = 2 * BN + STAGES * kSfCols > 512;
  static constexpr int kSfBase = kOverlap ? 512 - STAGES * kSfCols : 2 * BN;
  static constexpr int kAcc1 = kOverlap ? kSfBase - BN : BN;
  static constexpr int kShared = BN - kAcc1;  // columns of both accumulators
  static constexpr int kTmemCols = kSfBase + STAGES * kSfCols > 256 ? 512 : 256;
  static_assert(kSfBase + STAGES * kSfCols <= kTmemCols, "TMEM columns");
};

__device__ __forceinline__ void tile_coords(int tile, int tiles_m, int tiles_n, int& mb, int& nb) {
  const int per_group = kGroupM * tiles_n;
  const int g = tile / per_group;
  const int first_m = g * kGroupM;
  const int gm = min(tiles_m - first_m, kGroupM);
  const int local = tile - g * per_group;
  mb = first_m + local % gm;
  nb = local / gm;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_word(const uint32_t* r, int i) {
  if constexpr (std::is_same_v<T, float>)
    return r[i];
  else
    return Elem<T>::pack2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
}

template <typename T, int BN, int STAGES>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmA,
                      const __grid_constant__ CUtensorMap tmB,
                      const __grid_constant__ CUtensorMap tmC, const uint8_t* __restrict__ a_scales,
                      const uint8_t* __restrict__ b_scales, T* __restrict__ c, int M, int N, int K,
                      int tma_store) {
  using L = MxLayout<BN, STAGES>;
  constexpr int kChunk = 128 / sizeof(T);  // output columns per staged box
  constexpr int kChunks = BN / kChunk;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t bar0 = base + L::kOffBar;
  const uint32_t drain_bar = bar0 + 8u * (2 * STAGES + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  unsigned* wd = &g_mx_watchdog;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + a); };
  auto release_bar = [&](int a) { return bar0 + 8u * (2 * STAGES + 2 + a); };

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform
  const int lane = threadIdx.x & 31;
  const int tiles_m = (M + kBM - 1) / kBM;
  const int tiles_n = (N + BN - 1) / BN;
  const int num_tiles = tiles_m * tiles_n;
  const int kblocks = (K + kBK - 1) / kBK;
  const int sf_tiles_k = (K + 127) / 128;
  const int sf_tiles_n = (N + 127) / 128;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(release_bar(a), 4);  // the epilogue warps
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_addr(tmem_slot), L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Global memory is touched only from here on, once the previous kernel on
  // the stream has completed (programmatic dependent launch).
  pdl_wait_prior();

  if (warp == 0) {
    // ---------------- producer ----------------
    const bool elected = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
      int mb, nb;
      tile_coords(tile, tiles_m, tiles_n, mb, nb);
      const int sn0 = nb * BN / 128;  // first scale tile along N
      const bool second = L::kScaleTilesN == 2 && sn0 + 1 < sf_tiles_n;
      const uint8_t* sfa_row = a_scales + static_cast<int64_t>(mb) * sf_tiles_k * kScaleTile;
      const uint8_t* sfb_row = b_scales + static_cast<int64_t>(sn0) * sf_tiles_k * kScaleTile;
      for (int kb = 0; kb < kblocks; ++kb) {
        ok = mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, wd, kWdProducer);
        if (!ok) break;
        // Both scale tiles of the K block are neighbours in memory; the last
        // block may have one, the last N tile too.
        const int sk = 2 * kb;
        const uint32_t sf_bytes = (sk + 1 < sf_tiles_k ? 2 : 1) * kScaleTile;
        const uint32_t fb = full_bar(stage);
        const uint32_t sfb = base + L::kOffSfb + stage * L::kSfbBytes;
        if (elected) {
          mbar_arrive_expect_tx(fb, L::kABytes + L::kBBytes + (second ? 3 : 2) * sf_bytes);
          tma_load_2d(base + L::kOffA + stage * L::kABytes, &tmA, kb * 128, mb * kBM, fb);
          tma_load_2d(base + L::kOffB + stage * L::kBBytes, &tmB, kb * 128, nb * BN, fb);
          bulk_load(base + L::kOffSfa + stage * L::kSfaBytes, sfa_row + sk * kScaleTile, sf_bytes,
                    fb);
          bulk_load(sfb, sfb_row + sk * kScaleTile, sf_bytes, fb);
          if (second)
            bulk_load(sfb + 2 * kScaleTile,
                      sfb_row + (static_cast<int64_t>(sf_tiles_k) + sk) * kScaleTile, sf_bytes, fb);
        }
        __syncwarp();
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (elected) {
      int s = stage;
      uint32_t p = phase;
      for (int i = 0; i < STAGES && i < issued; ++i) {
        if (--s < 0) {
          s = STAGES - 1;
          p ^= 1u;
        }
        mbar_drain(full_bar(s), p);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA ----------------
    const bool elected = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    int it = 0;  // tiles of this CTA
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x, ++it) {
      int mb, nb;
      tile_coords(tile, tiles_m, tiles_n, mb, nb);
      const int acc = it & 1;
      // Overlapping accumulators: the previous tile's read-out has left the
      // shared columns.  Else: the read-out before it has left this one.
      const int need = L::kOverlap ? it - 1 : it - 2;
      if (need >= 0) {
        ok = mbar_wait_warp(release_bar(L::kOverlap ? 0 : acc),
                            (L::kOverlap ? need : need >> 1) & 1, abort_flag, wd, kWdMma);
        if (!ok) break;
      }
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + (acc ? L::kAcc1 : 0);
      // A 64-column tile may be the upper half of its scale tile: 2 columns on.
      const uint32_t sfb_shift = BN == 64 ? (nb & 1) * 2 : 0;
      for (int kb = 0; kb < kblocks; ++kb) {
        ok = mbar_wait_warp(full_bar(stage), phase, abort_flag, wd, kWdMma);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sfa = tmem_base + L::kSfBase + stage * L::kSfCols;
        const uint32_t sfb = sfa + 8;
        const uint64_t sa = sdesc_scales(base + L::kOffSfa + stage * L::kSfaBytes);
        const uint64_t sb = sdesc_scales(base + L::kOffSfb + stage * L::kSfbBytes);
        const uint64_t ad = sdesc_sw128(base + L::kOffA + stage * L::kABytes, 16, 1024);
        const uint64_t bd = sdesc_sw128(base + L::kOffB + stage * L::kBBytes, 16, 1024);
        const int steps = min(kBK / kStepK, (K - kb * kBK + kStepK - 1) / kStepK);
        if (elected) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {  // halves of 128 elements: one scale tile each
            if (2 * t < steps) {
              // Descriptors count addresses in units of 16 bytes.
              tmem_cp_scales(sfa + 4 * t, sa + t * (kScaleTile / 16));
#pragma unroll
              for (int j = 0; j < L::kScaleTilesN; ++j)
                tmem_cp_scales(sfb + 4 * (L::kScaleTilesN * t + j),
                               sb + (2 * j + t) * (kScaleTile / 16));
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int k = 2 * t + h;
                if (k < steps)
                  umma_mxf4(d_tmem, ad + k * 2, bd + k * 2, idesc_mxf4(kBM, BN, 2 * h), sfa + 4 * t,
                            sfb + 4 * L::kScaleTilesN * t + sfb_shift, kb > 0 || k > 0);
              }
            }
          }
          umma_commit(empty_bar(stage));
        }
        __syncwarp();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      if (elected) umma_commit(tfull_bar(acc));
      __syncwarp();
    }
    if (elected) {
      umma_commit(drain_bar);
      mbar_drain(drain_bar, 0);
    }
    __syncwarp();
  } else {
    // ---------------- epilogue (warps 2..5) ----------------
    const int q = warp & 3;
    const uint32_t buf = base + L::kOffC + (warp - 2) * L::kCBuf;
    uint8_t* buf_ptr = smem + L::kOffC + (warp - 2) * L::kCBuf;
    int it = 0;
    bool stored = false;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x, ++it) {
      int mb, nb;
      tile_coords(tile, tiles_m, tiles_n, mb, nb);
      const int acc = it & 1;
      int ok = 1;
      if (lane == 0)
        ok = mbar_wait_bounded(tfull_bar(acc), (it >> 1) & 1, abort_flag, wd, kWdEpilogue);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      const uint32_t trow = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + (acc ? L::kAcc1 : 0);
      const int y = mb * kBM + q * 32;
      // Chunks after which the columns of both accumulators have been read.
      constexpr int kRelease = L::kOverlap ? (L::kShared + kChunk - 1) / kChunk : kChunks;
#pragma unroll 1
      for (int i = 0; i < kChunks; ++i) {
        const int ch = L::kOverlap && acc == 0 ? kChunks - 1 - i : i;
        uint32_t r[kChunk];
#pragma unroll
        for (int j = 0; j < kChunk; j += 32) tmem_ld_32x32b_x32(trow + ch * kChunk + j, r + j);
        tmem_wait_ld();
        if (i == kRelease - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(release_bar(L::kOverlap ? 0 : acc));
        }
        const int x = nb * BN + ch * kChunk;
        if (x >= N || y >= M) continue;
        if (stored && tma_store && lane == 0) bulk_wait_read<0>();
        __syncwarp();
        const uint32_t srow = buf + lane * 128;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          st_shared_v4(srow + ((j ^ (lane & 7)) << 4), pack_word<T>(r, 4 * j),
                       pack_word<T>(r, 4 * j + 1), pack_word<T>(r, 4 * j + 2),
                       pack_word<T>(r, 4 * j + 3));
        if (tma_store) {
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmC, buf, x, y);
            bulk_commit();
          }
          stored = true;
        } else {
          // Row strides or a base that TMA cannot address: element stores, a
          // row at a time.
          __syncwarp();
          const int rows = min(32, M - y);
          for (int rr = 0; rr < rows; ++rr) {
            T* crow = c + static_cast<int64_t>(y + rr) * N + x;
#pragma unroll
            for (int e = lane; e < kChunk; e += 32) {
              const int b = e * static_cast<int>(sizeof(T));
              const T v = *reinterpret_cast<const T*>(
                  buf_ptr + rr * 128 + (((b >> 4) ^ (rr & 7)) << 4) + (b & 15));
              if (x + e < N) crow[e] = v;
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

template <typename T>
int output_map(CUtensorMap* tm, const void* c, int M, int N, int* tma_store) {
  *tma_store = aligned16(c) && static_cast<int64_t>(N) * sizeof(T) % 16 == 0;
  if (!*tma_store) return AOTK_OK;
  if constexpr (std::is_same_v<T, float>)
    return make_tmap_2d_f32(tm, c, M, N, N, 32, 32);
  else
    return make_tmap_2d_16bit(tm, c, std::is_same_v<T, __nv_bfloat16>, M, N, N, 64, 32);
}

template <typename T, int BN, int STAGES>
int launch_tiles(void* c, const void* a, const void* as, const void* b, const void* bs, int M,
                 int N, int K, cudaStream_t stream, const DeviceInfo& info) {
  using L = MxLayout<BN, STAGES>;
  auto kernel = gemm_mxfp4_kernel<T, BN, STAGES>;
  if (int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kAlloc, info)) return st;
  CUtensorMap ta, tb, tc = {};
  int tma_store = 0;
  if (int st = make_tmap_2d_8bit(&ta, a, M, K / 2, K / 2, 128, kBM)) return st;
  if (int st = make_tmap_2d_8bit(&tb, b, N, K / 2, K / 2, 128, BN)) return st;
  if (int st = output_map<T>(&tc, c, M, N, &tma_store)) return st;
  const int64_t tiles = static_cast<int64_t>((M + kBM - 1) / kBM) * ((N + BN - 1) / BN);
  if (tiles > 0x7fffffffLL)
    return fail(AOTK_ERR_UNSUPPORTED, "aotk_mxfp4_gemm: output of %d x %d has too many tiles", M, N);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles < info.sm_count ? tiles : info.sm_count), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kAlloc;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(
      &cfg, kernel, ta, tb, tc, static_cast<const uint8_t*>(as), static_cast<const uint8_t*>(bs),
      static_cast<T*>(c), M, N, K, tma_store);
  if (e != cudaSuccess)
    return fail(AOTK_ERR_CUDA, "aotk_mxfp4_gemm launch: %s", cudaGetErrorString(e));
  return check_launch("aotk_mxfp4_gemm");
}

template <typename T>
int dispatch(void* c, const void* a, const void* as, const void* b, const void* bs, int M, int N,
             int K, cudaStream_t s, const DeviceInfo& info) {
  // Rounds of tiles on the SMs, in units of 256 columns.
  auto rounds = [&](int bn) {
    const int64_t tiles = static_cast<int64_t>((M + kBM - 1) / kBM) * ((N + bn - 1) / bn);
    return static_cast<double>((tiles + info.sm_count - 1) / info.sm_count) * bn / 256;
  };
  const double r256 = rounds(256), r128 = 1.1 * rounds(128), r64 = 1.3 * rounds(64);
  if (r256 <= r128 && r256 <= r64)
    return launch_tiles<T, 256, 4>(c, a, as, b, bs, M, N, K, s, info);
  if (r128 <= r64) return launch_tiles<T, 128, 6>(c, a, as, b, bs, M, N, K, s, info);
  return launch_tiles<T, 64, 7>(c, a, as, b, bs, M, N, K, s, info);
}

}  // namespace

int mxfp4_watchdog(uint32_t* status, bool clear) {
  unsigned v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_mx_watchdog, sizeof(v));
  if (e != cudaSuccess) return fail(AOTK_ERR_CUDA, "watchdog read: %s", cudaGetErrorString(e));
  if (clear) {
    const unsigned zero = 0;
    e = cudaMemcpyToSymbol(g_mx_watchdog, &zero, sizeof(zero));
    if (e != cudaSuccess) return fail(AOTK_ERR_CUDA, "watchdog clear: %s", cudaGetErrorString(e));
  }
  *status |= v;
  return AOTK_OK;
}

}  // namespace aotk

extern "C" int aotk_mxfp4_gemm(void* c, const void* a, const void* a_scales, const void* b,
                               const void* b_scales, int64_t M, int64_t N, int64_t K,
                               int out_dtype, void* stream) {
  using namespace aotk;
  const char* who = "aotk_mxfp4_gemm";
  if (M < 0 || N < 0 || K < 0) return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (!valid_dtype(out_dtype))
    return fail(AOTK_ERR_UNSUPPORTED, "%s: unsupported output dtype %d", who, out_dtype);
  if (K % 32 != 0)
    return fail(AOTK_ERR_UNSUPPORTED, "%s: K = %lld is not a multiple of the block size 32", who,
                (long long)K);
  if (M == 0 || N == 0) return AOTK_OK;
  if (!c || (K > 0 && (!a || !a_scales || !b || !b_scales)))
    return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (M > 0x7fffff00LL || N > 0x7fffff00LL || K > 0x7fffff00LL)
    return fail(AOTK_ERR_UNSUPPORTED, "%s: extents above 2^31 - 256", who);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (K == 0) {  // an empty sum
    const size_t bytes = static_cast<size_t>(M) * static_cast<size_t>(N) * elem_size(out_dtype);
    cudaError_t e = cudaMemsetAsync(c, 0, bytes, s);
    return e == cudaSuccess ? AOTK_OK : fail(AOTK_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  }
  if (!aligned16(a) || !aligned16(b) || !aligned16(a_scales) || !aligned16(b_scales))
    return fail(AOTK_ERR_UNSUPPORTED, "%s: codes and scales must be 16-byte aligned", who);
  DeviceInfo info;
  if (int st = current_device_info(&info)) return st;
  if (int st = require_sm100(info)) return st;
  const int m = (int)M, n = (int)N, k = (int)K;
  if (M <= kSkinnyMaxM)
    return gemm_mxfp4_skinny(c, a, a_scales, b, b_scales, m, n, k, out_dtype, stream, info);
  switch (out_dtype) {
    case AOTK_FLOAT32: return dispatch<float>(c, a, a_scales, b, b_scales, m, n, k, s, info);
    case AOTK_FLOAT16: return dispatch<__half>(c, a, a_scales, b, b_scales, m, n, k, s, info);
    default: return dispatch<__nv_bfloat16>(c, a, a_scales, b, b_scales, m, n, k, s, info);
  }
}
