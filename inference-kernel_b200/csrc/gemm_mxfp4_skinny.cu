// Product of two microscaled 4-bit matrices for few rows of A (decode, M <= 128):
// C[m, n] = sum_k A[m, k] B[n, k], layouts as in mxfp4.cu.
//
// The cost is streaming the weight B and its scales from HBM (17 bytes per 32
// elements), so the kernel is organised around that stream:
//   * swapped operands: 128 rows of B fill the MMA's M, the rows of A, padded to
//     MP = 16..128 by TMA zero fill, are its N;
//   * K is split over a cluster of S <= 8 CTAs so that about two CTAs per SM
//     stream at once; each leaves an fp32 partial tile in its shared memory, and
//     the S partials are added in rank order through distributed shared memory:
//     no workspace, no atomics, one launch, the same sum every time.
// Stages, scale copies and scale areas in TMEM are those of gemm_mxfp4.cu.
#include "common.h"
#include "gemm_internal.h"
#include "sm100.cuh"
#include "tmap.h"
#include "vec.cuh"

namespace aotk {
namespace {

using namespace sm100;

__device__ unsigned g_mxs_watchdog;

constexpr int kThreads = 192;  // producer, MMA and 4 TMEM-reading warps
constexpr int kTileN = 128;    // rows of B per CTA (the MMA's M)
constexpr int kBK = 256;       // elements of K per stage (128 bytes of codes)
constexpr int kStepK = 64;
constexpr int kMaxCluster = 8;
constexpr uint32_t kScaleTile = 512;

enum : unsigned { kWdProducer = 32768u, kWdMma = 65536u, kWdEpilogue = 131072u };

template <int MP, int STAGES>
struct MxsLayout {
  static constexpr uint32_t kWBytes = kTileN * 128;
  static constexpr uint32_t kXBytes = MP * 128;
  static constexpr uint32_t kSfBytes = 2 * kScaleTile;  // per operand
  static constexpr uint32_t kOffW = 0;
  static constexpr uint32_t kOffX = kOffW + STAGES * kWBytes;
  static constexpr uint32_t kOffSfw = kOffX + STAGES * kXBytes;
  static constexpr uint32_t kOffSfx = kOffSfw + STAGES * kSfBytes;
  static constexpr uint32_t kRing = kOffSfx + STAGES * kSfBytes;
  static constexpr uint32_t kPartial = MP * kTileN * 4;  // aliases the drained ring
  static constexpr uint32_t kOffBar = kRing > kPartial ? kRing : kPartial;
  static constexpr uint32_t kNumBars = 2 * STAGES + 1;  // full, empty, done
  static constexpr uint32_t kOffMisc = kOffBar + kNumBars * 8;
  static constexpr uint32_t kAlloc = kOffMisc + 16 + 1024;
  static constexpr int kSfCols = 16;  // 2 scale tiles of 4 columns per operand
  static constexpr int kCols = MP + STAGES * kSfCols;
  static constexpr int kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : 256;
  static_assert(kCols <= 256, "two CTAs share an SM's 512 TMEM columns");
  static_assert(kXBytes % 1024 == 0, "swizzle atoms");
};

template <typename T, int MP, int STAGES>
__global__ void __launch_bounds__(kThreads, 2)
    gemm_mxfp4_skinny_kernel(const __grid_constant__ CUtensorMap tmW,
                             const __grid_constant__ CUtensorMap tmX,
                             const uint8_t* __restrict__ w_scales,
                             const uint8_t* __restrict__ x_scales, T* __restrict__ c, int M, int N,
                             int K, int kb_per_split, int vec_store) {
  using L = MxsLayout<MP, STAGES>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t bar0 = base + L::kOffBar;
  const uint32_t done_bar = bar0 + 8u * (2 * STAGES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  float* partial = reinterpret_cast<float*>(smem);  // [MP][128], after the main loop
  unsigned* wd = &g_mxs_watchdog;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform
  const int lane = threadIdx.x & 31;
  const uint32_t split = cluster_ctarank();
  uint32_t S;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(S));
  const int strip = static_cast<int>(blockIdx.x / S);
  const int n0 = strip * kTileN;
  const int kblocks = (K + kBK - 1) / kBK;
  const int sf_tiles_k = (K + 127) / 128;
  const int kb0 = static_cast<int>(split) * kb_per_split;
  const int kb1 = min(kblocks, kb0 + kb_per_split);  // the host guarantees kb1 > kb0

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
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
  pdl_wait_prior();  // inputs, and the memory under C, may be the previous kernel's

  if (warp == 0) {
    const bool elected = elect_one();
    const uint8_t* w_row = w_scales + static_cast<int64_t>(strip) * sf_tiles_k * kScaleTile;
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, wd, kWdProducer)) break;
      const int sk = 2 * kb;
      const uint32_t sf_bytes = (sk + 1 < sf_tiles_k ? 2 : 1) * kScaleTile;
      const uint32_t fb = full_bar(stage);
      if (elected) {
        mbar_arrive_expect_tx(fb, L::kWBytes + L::kXBytes + 2 * sf_bytes);
        tma_load_2d(base + L::kOffW + stage * L::kWBytes, &tmW, kb * 128, n0, fb);
        bulk_load(base + L::kOffSfw + stage * L::kSfBytes, w_row + sk * kScaleTile, sf_bytes, fb);
        tma_load_2d(base + L::kOffX + stage * L::kXBytes, &tmX, kb * 128, 0, fb);
        bulk_load(base + L::kOffSfx + stage * L::kSfBytes, x_scales + sk * kScaleTile, sf_bytes, fb);
      }
      __syncwarp();
      ++issued;
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
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
    const bool elected = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(full_bar(stage), phase, abort_flag, wd, kWdMma)) break;
      tc_fence_after();
      const uint32_t sfw = tmem_base + MP + stage * L::kSfCols;
      const uint32_t sfx = sfw + 8;
      const uint64_t sw = sdesc_scales(base + L::kOffSfw + stage * L::kSfBytes);
      const uint64_t sx = sdesc_scales(base + L::kOffSfx + stage * L::kSfBytes);
      const uint64_t wdesc = sdesc_sw128(base + L::kOffW + stage * L::kWBytes, 16, 1024);
      const uint64_t xdesc = sdesc_sw128(base + L::kOffX + stage * L::kXBytes, 16, 1024);
      const int steps = min(kBK / kStepK, (K - kb * kBK + kStepK - 1) / kStepK);
      if (elected) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (2 * t < steps) {
            tmem_cp_scales(sfw + 4 * t, sw + t * (kScaleTile / 16));
            tmem_cp_scales(sfx + 4 * t, sx + t * (kScaleTile / 16));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int k = 2 * t + h;
              if (k < steps)
                umma_mxf4(tmem_base, wdesc + k * 2, xdesc + k * 2, idesc_mxf4(kTileN, MP, 2 * h),
                          sfw + 4 * t, sfx + 4 * t, kb > kb0 || k > 0);
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
    if (elected) {
      umma_commit(done_bar);
      mbar_drain(done_bar, 0);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    int ok = 1;
    if (lane == 0) ok = mbar_wait_bounded(done_bar, 0, abort_flag, wd, kWdEpilogue);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    if (ok) {
      tc_fence_after();
      const int nl = q * 32 + lane;  // row of B within the strip = TMEM lane
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < M; c0 += 16) {  // columns of rows that exist
        uint32_t r[16];
        tmem_ld_32x32b_x16(taddr + c0, r);
        tmem_wait_ld();
#pragma unroll
        for (int m = 0; m < 16; ++m) partial[(c0 + m) * kTileN + nl] = __uint_as_float(r[m]);
      }
    }
  }

  tc_fence_before();
  cluster_sync();  // partials of every CTA of the cluster are complete and visible

  // This CTA adds its share of the M x 128 tile's groups of four over all S
  // partials, in rank order.
  {
    const uint32_t groups = static_cast<uint32_t>(M) * (kTileN / 4);
    const uint32_t f_end = groups * (split + 1) / S;
    const uint32_t part_addr = smem_addr(partial);
    for (uint32_t f = groups * split / S + threadIdx.x; f < f_end; f += kThreads) {
      const int m = static_cast<int>(f / (kTileN / 4));
      const int n = n0 + static_cast<int>(f % (kTileN / 4)) * 4;
      if (n >= N) continue;
      // All reads first: each is a trip through another SM's shared memory.
      float4 v[kMaxCluster];
#pragma unroll
      for (uint32_t j = 0; j < kMaxCluster; ++j)
        if (j < S) v[j] = ld_dsmem_f32x4(map_to_rank(part_addr + f * 16u, j));
      float4 acc = v[0];
#pragma unroll
      for (uint32_t j = 1; j < kMaxCluster; ++j) {
        if (j < S) {
          acc.x += v[j].x;
          acc.y += v[j].y;
          acc.z += v[j].z;
          acc.w += v[j].w;
        }
      }
      T* p = c + static_cast<int64_t>(m) * N + n;
      if (vec_store) {  // N % 4 == 0 and c aligned: all four exist
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<float4*>(p) = acc;
        } else {
          uint2 o;
          o.x = Elem<T>::pack2(acc.x, acc.y);
          o.y = Elem<T>::pack2(acc.z, acc.w);
          *reinterpret_cast<uint2*>(p) = o;
        }
      } else {
        const float e4[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N) p[e] = Elem<T>::from_f(e4[e]);
      }
    }
  }

  // No CTA leaves while a peer may still read its shared memory.
  __syncwarp();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

template <typename T, int MP, int STAGES>
int launch_skinny(void* c, const void* a, const void* as, const void* b, const void* bs, int M,
                  int N, int K, cudaStream_t stream, const DeviceInfo& info) {
  using L = MxsLayout<MP, STAGES>;
  auto kernel = gemm_mxfp4_skinny_kernel<T, MP, STAGES>;
  if (int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kAlloc, info)) return st;
  CUtensorMap tw, tx;
  if (int st = make_tmap_2d_8bit(&tw, b, N, K / 2, K / 2, 128, kTileN)) return st;
  if (int st = make_tmap_2d_8bit(&tx, a, M, K / 2, K / 2, 128, MP)) return st;
  const int strips = (N + kTileN - 1) / kTileN;
  const int kblocks = (K + kBK - 1) / kBK;
  // One wave, as in the 16-bit skinny kernel: the largest cluster (<= 8, <= K
  // blocks) whose `strips` clusters are resident together, two CTAs per SM.
  int S = 1;
  for (int cs = kMaxCluster < kblocks ? kMaxCluster : kblocks; cs > 1; --cs) {
    int resident = 0;
    if (int st = resident_clusters(cs, static_cast<int>(L::kAlloc), info, &resident)) return st;
    if (strips <= resident) {
      S = cs;
      break;
    }
  }
  const int kbps = (kblocks + S - 1) / S;
  S = (kblocks + kbps - 1) / kbps;  // every split owns at least one K block
  const int64_t blocks = static_cast<int64_t>(strips) * S;

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kAlloc;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(S);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const int vec_store = N % 4 == 0 && aligned16(c);
  cudaError_t e = cudaLaunchKernelEx(
      &cfg, kernel, tw, tx, static_cast<const uint8_t*>(bs), static_cast<const uint8_t*>(as),
      static_cast<T*>(c), M, N, K, kbps, vec_store);
  if (e != cudaSuccess)
    return fail(AOTK_ERR_CUDA, "aotk_mxfp4_gemm launch (cluster %d): %s", S, cudaGetErrorString(e));
  return check_launch("aotk_mxfp4_gemm");
}

// Ring depth per width of A: two CTAs fit per SM (at most 113 KB each).
template <typename T>
int dispatch(void* c, const void* a, const void* as, const void* b, const void* bs, int M, int N,
             int K, cudaStream_t s, const DeviceInfo& info) {
  if (M <= 16) return launch_skinny<T, 16, 5>(c, a, as, b, bs, M, N, K, s, info);
  if (M <= 32) return launch_skinny<T, 32, 5>(c, a, as, b, bs, M, N, K, s, info);
  if (M <= 64) return launch_skinny<T, 64, 4>(c, a, as, b, bs, M, N, K, s, info);
  return launch_skinny<T, 128, 3>(c, a, as, b, bs, M, N, K, s, info);
}

}  // namespace

int gemm_mxfp4_skinny(void* c, const void* a, const void* as, const void* b, const void* bs, int M,
                      int N, int K, int out_dtype, void* stream, const DeviceInfo& info) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case AOTK_FLOAT32: return dispatch<float>(c, a, as, b, bs, M, N, K, s, info);
    case AOTK_FLOAT16: return dispatch<__half>(c, a, as, b, bs, M, N, K, s, info);
    default: return dispatch<__nv_bfloat16>(c, a, as, b, bs, M, N, K, s, info);
  }
}

int mxfp4_skinny_watchdog(uint32_t* status, bool clear) {
  unsigned v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_mxs_watchdog, sizeof(v));
  if (e != cudaSuccess) return fail(AOTK_ERR_CUDA, "watchdog read: %s", cudaGetErrorString(e));
  if (clear) {
    const unsigned zero = 0;
    e = cudaMemcpyToSymbol(g_mxs_watchdog, &zero, sizeof(zero));
    if (e != cudaSuccess) return fail(AOTK_ERR_CUDA, "watchdog clear: %s", cudaGetErrorString(e));
  }
  *status |= v;
  return AOTK_OK;
}

}  // namespace aotk
