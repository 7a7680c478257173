// Product of two microscaled 4-bit matrices for few rows of A (decode, M <= 128):
// C[m, n] = sum_k A[m, k] B[n, k], layouts as in mxfp4.cu.
//
// The cost is streaming the weight B and its scales from HBM (17 bytes per 32
// elements), so the kernel is organised around that stream:
//   * swapped operands: a strip of 128 rows of B fills the MMA's M, the rows of A,
//     padded to MP = 16..128 by TMA zero fill, are its N;
//   * a cluster of C <= 8 CTAs takes Q strips: the strips' K blocks in one line,
//     cut into C equal parts, so that about two CTAs per SM stream equal shares at
//     once.  A CTA's part is one or two segments, each of one strip;
//   * a segment's fp32 sums go straight from TMEM into the shared memory of the
//     CTAs that hold parts of the same strip (st.async), each of which receives the
//     strip's columns of its own, adds them in rank order, rounds and writes them:
//     no workspace, no atomics, one launch, the same sum every time.  Nobody waits
//     for a cluster barrier at the end; a CTA leaves when it has what is sent to it;
//   * a CTA asks for its first blocks of the weight in L2 before it waits for the
//     previous kernel on the stream (kAhead; graph replays, us: 1 x 28672 x 4096
//     12.6 -> 12.0, 1 x 6144 x 4096 5.45 -> 4.9, 1 x 4096 x 14336 8.0 -> 7.3, after a
//     quantiser 10.2 -> 9.3).
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
constexpr int kTileN = 128;    // rows of B per strip (the MMA's M)
constexpr int kBK = 256;       // elements of K per stage (128 bytes of codes)
constexpr int kStepK = 64;
constexpr int kMaxCluster = 8;
constexpr int kAhead = 4;      // blocks prefetched; 2 gain less, 8 or all of them lose at 48 rows
constexpr uint32_t kScaleTile = 512;

enum : unsigned { kWdProducer = 32768u, kWdMma = 65536u, kWdEpilogue = 131072u };

// SEGS: segments per CTA (1 or 2).  kAlias: the buffer for received sums lies over
// the ring, and is used only when every CTA of the cluster is done with its ring.
template <int MP, int STAGES, int SEGS, bool kAlias>
struct MxsLayout {
  static constexpr uint32_t kWBytes = kTileN * 128;
  static constexpr uint32_t kXBytes = MP * 128;
  static constexpr uint32_t kSfBytes = 2 * kScaleTile;  // per operand
  static constexpr uint32_t kOffW = 0;
  static constexpr uint32_t kOffX = kOffW + STAGES * kWBytes;
  static constexpr uint32_t kOffSfw = kOffX + STAGES * kXBytes;
  static constexpr uint32_t kOffSfx = kOffSfw + STAGES * kSfBytes;
  static constexpr uint32_t kRing = kOffSfx + STAGES * kSfBytes;
  // Received sums of one strip: contributions x columns (their product is at most
  // 128 + kMaxCluster - 1) x MP rows, fp32.
  static constexpr uint32_t kRecv = (kTileN + kMaxCluster - 1) * MP * 4;
  static constexpr uint32_t kOffRecv = kAlias ? 0 : kRing;
  static constexpr uint32_t kOffBar =
      kAlias ? (kRing > kRecv ? kRing : kRecv) : kRing + SEGS * kRecv;
  static constexpr uint32_t kNumBars = 2 * STAGES + 2 * SEGS;  // full, empty, done, received
  static constexpr uint32_t kOffMisc = kOffBar + kNumBars * 8;
  static constexpr uint32_t kAlloc = kOffMisc + 16 + 1024;
  static constexpr int kSfCols = 16;  // 2 scale tiles of 4 columns per operand
  static constexpr int kCols = SEGS * MP + STAGES * kSfCols;
  static constexpr int kTmemCols = kCols <= 64 ? 64 : kCols <= 128 ? 128 : 256;
  static_assert(kCols <= 256, "two CTAs share an SM's 512 TMEM columns");
  static_assert(kAlloc <= (233472 - 2 * 1024) / 2, "two CTAs share an SM's shared memory");
  static_assert(!kAlias || SEGS == 1, "one buffer over the ring");
  static_assert(kOffBar % 16 == 0 && kXBytes % 1024 == 0, "alignment, swizzle atoms");
};

// Parts: unit x of U (K block x % kblocks of strip x / kblocks of the cluster's
// strips) belongs to CTA part_of(x); CTA r has units [part_begin(r), part_begin(r + 1)).
// K <= 2^28: U < 2^20 x 8 and C <= 8, so the products fit 32 bits.
__device__ __forceinline__ int part_begin(int r, int units, int ctas) {
  return static_cast<int>(static_cast<unsigned>(units * r) / static_cast<unsigned>(ctas));
}
__device__ __forceinline__ int part_of(int x, int units, int ctas) {
  return static_cast<int>(static_cast<unsigned>((x + 1) * ctas - 1) / static_cast<unsigned>(units));
}

template <typename T, int MP, int STAGES, int SEGS, bool kAlias>
__global__ void __launch_bounds__(kThreads, 2)
    gemm_mxfp4_skinny_kernel(const __grid_constant__ CUtensorMap tmW,
                             const __grid_constant__ CUtensorMap tmX,
                             const uint8_t* w_scales, const uint8_t* x_scales,
                             T* __restrict__ c, int M, int N, int K, int strips_per_cluster) {
  using L = MxsLayout<MP, STAGES, SEGS, kAlias>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const uint32_t bar0 = base + L::kOffBar;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
  unsigned* wd = &g_mxs_watchdog;
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto done_bar = [&](int i) { return bar0 + 8u * (2 * STAGES + i); };
  auto recv_bar = [&](int i) { return bar0 + 8u * (2 * STAGES + SEGS + i); };

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform
  const int lane = threadIdx.x & 31;
  const int rank = __shfl_sync(0xffffffffu, cluster_ctarank(), 0);
  int C;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(C));
  C = __shfl_sync(0xffffffffu, C, 0);
  const int kblocks = (K + kBK - 1) / kBK;
  const int sf_tiles_k = (K + 127) / 128;
  const int strips = (N + kTileN - 1) / kTileN;
  const int strip0 = static_cast<int>(blockIdx.x / C) * strips_per_cluster;
  const int units = min(strips_per_cluster, strips - strip0) * kblocks;
  const int u0 = part_begin(rank, units, C), u1 = part_begin(rank + 1, units, C);
  const int local0 = u0 / kblocks;  // first strip of this CTA within the cluster's
  const int rows4 = (M + 3) / 4;    // rows of A in fours

  // Segment i is of strip local0 + i; its contributors are CTAs [first, first + n).
  struct Strip {
    int first, n;
  };
  auto contributors = [&](int local) {
    Strip s = {0, C};
    if (strips_per_cluster == 1) return s;
    s.first = part_of(local * kblocks, units, C);
    s.n = part_of((local + 1) * kblocks - 1, units, C) - s.first + 1;
    return s;
  };
  auto segment_end = [&](int i) { return min(u1, (local0 + i + 1) * kblocks); };
  auto segment_begin = [&](int i) { return i == 0 ? u0 : (local0 + i) * kblocks; };
  const int segs = u1 > u0 ? (u1 - 1) / kblocks - local0 + 1 : 0;  // at most SEGS (host)

  // The next kernel may start its own prologue now; this kernel reads global
  // memory only after pdl_wait_prior() below.
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int i = 0; i < SEGS; ++i) {
      mbar_init(done_bar(i), 1);
      mbar_init(recv_bar(i), 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
    for (int i = 0; i < segs; ++i) {  // what this CTA will be sent, if others have parts
      const Strip s = contributors(local0 + i);
      const int mine = rank - s.first;
      const int cols = kTileN * (mine + 1) / s.n - kTileN * mine / s.n;
      if (s.n > 1) mbar_arrive_expect_tx(recv_bar(i), static_cast<uint32_t>(s.n * cols * rows4) * 16u);
    }
  }
  if (warp == 1) {
    tmem_alloc(smem_addr(tmem_slot), L::kTmemCols);
    tmem_relinquish();
  } else if (warp == 2) {
    if (elect_one()) {
      int strip = strip0 + local0, kb = u0 - local0 * kblocks;
      for (int u = u0; u < min(u1, u0 + kAhead); ++u) {
        tma_prefetch_2d(&tmW, kb * 128, strip * kTileN);
        const int sk = 2 * kb;
        bulk_prefetch(w_scales + (static_cast<int64_t>(strip) * sf_tiles_k + sk) * kScaleTile,
                      (sk + 1 < sf_tiles_k ? 2 : 1) * kScaleTile);
        if (++kb == kblocks) {
          kb = 0;
          ++strip;
        }
      }
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  cluster_arrive_relaxed();  // this CTA's barriers may be signalled; the wait is before the first send
  pdl_wait_prior();  // inputs, and the memory under C, may be the previous kernel's

  if (warp == 0) {
    const bool elected = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    int strip = strip0 + local0, kb = u0 - local0 * kblocks;
    for (int u = u0; u < u1; ++u) {
      if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, wd, kWdProducer)) break;
      const int sk = 2 * kb;
      const uint32_t sf_bytes = (sk + 1 < sf_tiles_k ? 2 : 1) * kScaleTile;
      const uint32_t fb = full_bar(stage);
      const uint8_t* ws = w_scales + (static_cast<int64_t>(strip) * sf_tiles_k + sk) * kScaleTile;
      if (elected) {
        mbar_arrive_expect_tx(fb, L::kWBytes + L::kXBytes + 2 * sf_bytes);
        tma_load_2d(base + L::kOffW + stage * L::kWBytes, &tmW, kb * 128, strip * kTileN, fb);
        bulk_load(base + L::kOffSfw + stage * L::kSfBytes, ws, sf_bytes, fb);
        tma_load_2d(base + L::kOffX + stage * L::kXBytes, &tmX, kb * 128, 0, fb);
        bulk_load(base + L::kOffSfx + stage * L::kSfBytes, x_scales + sk * kScaleTile, sf_bytes, fb);
      }
      __syncwarp();
      ++issued;
      if (++kb == kblocks) {
        kb = 0;
        ++strip;
      }
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
    cluster_wait();
  } else if (warp == 1) {
    const bool elected = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; ok && i < segs; ++i) {
      const int begin = segment_begin(i), end = segment_end(i);
      const uint32_t d_tmem = tmem_base + i * MP;
      int kb = begin - (local0 + i) * kblocks;
      for (int u = begin; u < end; ++u, ++kb) {
        ok = mbar_wait_warp(full_bar(stage), phase, abort_flag, wd, kWdMma);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sfw = tmem_base + SEGS * MP + stage * L::kSfCols;
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
                  umma_mxf4(d_tmem, wdesc + k * 2, xdesc + k * 2, idesc_mxf4(kTileN, MP, 2 * h),
                            sfw + 4 * t, sfx + 4 * t, u > begin || k > 0);
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
      if (ok && elected) umma_commit(done_bar(i));
      __syncwarp();
    }
    // Every MMA is done before the CTA leaves; after a wait that gave up, too.
    if (elected && !ok) {
      umma_commit(done_bar(SEGS - 1));
      mbar_drain(done_bar(SEGS - 1), 0);
    }
    __syncwarp();
    cluster_wait();
  } else {
    const int q = warp & 3;
    const int n = q * 32 + lane;  // row of B within the strip = TMEM lane
    // Where this lane's sums of segment i go (worked out while the weight streams):
    // the contributor that adds up this column, and the place in its buffer.
    Strip strip_of[SEGS];
    uint32_t to_bar[SEGS], to_buf[SEGS], to_step[SEGS];
#pragma unroll
    for (int i = 0; i < SEGS; ++i) {
      if (i >= segs) break;
      const int local = local0 + i;
      const Strip s = contributors(local);
      strip_of[i] = s;
      const int to = ((n + 1) * s.n - 1) / kTileN;
      const int col = n - kTileN * to / s.n;
      const int pitch = (kTileN + s.n - 1) / s.n;  // columns
      const int dst = s.first + to;
      const int slot = part_begin(dst, units, C) / kblocks == local ? 0 : 1;
      to_bar[i] = map_to_rank(recv_bar(slot), dst);
      to_buf[i] = map_to_rank(base + L::kOffRecv + slot * L::kRecv, dst) +
                  static_cast<uint32_t>((rank - s.first) * rows4 * pitch + col) * 16u;
      to_step[i] = static_cast<uint32_t>(pitch) * 16u;
    }
    cluster_wait();
    bool ok = true;
#pragma unroll
    for (int i = 0; i < SEGS; ++i) {
      if (!ok || i >= segs) break;
      int done = 1;
      if (lane == 0) done = mbar_wait_bounded(done_bar(i), 0, abort_flag, wd, kWdEpilogue);
      ok = __shfl_sync(0xffffffffu, done, 0) != 0;
      // Every ring has been read, as its MMAs' barrier has shown (also after a wait
      // that gave up); nothing was written for others.
      if constexpr (kAlias) {
        cluster_arrive_relaxed();
        cluster_wait();
      }
      if (!ok) break;
      tc_fence_after();
      const bool alone = strip_of[i].n == 1;
      const int column = (strip0 + local0 + i) * kTileN + n;
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + i * MP;
#pragma unroll 1
      for (int c0 = 0; c0 < M; c0 += 16) {  // columns of rows that exist
        uint32_t r[16];
        tmem_ld_32x32b_x16(taddr + c0, r);
        tmem_wait_ld();
        if (alone) {
          if (column < N) {
            T* p = c + static_cast<int64_t>(c0) * N + column;
#pragma unroll
            for (int m = 0; m < 16; ++m)
              if (c0 + m < M) p[static_cast<int64_t>(m) * N] = Elem<T>::from_f(__uint_as_float(r[m]));
          }
        } else {
#pragma unroll
          for (int m = 0; m < 4; ++m)
            if (c0 / 4 + m < rows4)
              st_async_v4(to_buf[i] + static_cast<uint32_t>(c0 / 4 + m) * to_step[i], r[4 * m],
                          r[4 * m + 1], r[4 * m + 2], r[4 * m + 3], to_bar[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < SEGS; ++i) {
      if (!ok || i >= segs) break;
      const Strip s = strip_of[i];
      if (s.n == 1) continue;
      const int mine = rank - s.first;
      const int n_begin = kTileN * mine / s.n;
      const int cols = kTileN * (mine + 1) / s.n - n_begin;
      const int pitch = (kTileN + s.n - 1) / s.n;
      const int n0 = (strip0 + local0 + i) * kTileN + n_begin;
      const float4* got = reinterpret_cast<const float4*>(smem + L::kOffRecv + i * L::kRecv);
      if (!mbar_wait_bounded(recv_bar(i), 0, abort_flag, wd, kWdEpilogue)) break;
      for (int f = threadIdx.x - 64; f < rows4 * cols; f += kThreads - 64) {
        const int m4 = f / cols, cl = f - m4 * cols;
        if (n0 + cl >= N) continue;
        float4 v[kMaxCluster];
#pragma unroll
        for (int j = 0; j < kMaxCluster; ++j)
          if (j < s.n) v[j] = got[(j * rows4 + m4) * pitch + cl];
        float4 acc = v[0];
#pragma unroll
        for (int j = 1; j < kMaxCluster; ++j) {
          if (j < s.n) {
            acc.x += v[j].x;
            acc.y += v[j].y;
            acc.z += v[j].z;
            acc.w += v[j].w;
          }
        }
        const float e4[4] = {acc.x, acc.y, acc.z, acc.w};
        T* p = c + static_cast<int64_t>(m4) * 4 * N + n0 + cl;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (m4 * 4 + e < M) p[static_cast<int64_t>(e) * N] = Elem<T>::from_f(e4[e]);
      }
    }
  }
  if constexpr (kAlias) {
    if (warp < 2) {
      cluster_arrive_relaxed();
      cluster_wait();
    }
  }

  tc_fence_before();
  __syncthreads();
  // A wait that gave up: stay until no other CTA can send here any more (those
  // that have left count as arrived).
  if (*abort_flag) {
    cluster_arrive_relaxed();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

// How the weight is cut: C CTAs per cluster, Q strips per cluster.  All CTAs stream
// at once, two per SM.  While clusters of two or more find room for every strip, a
// strip is a cluster's and C is the largest (<= 8, <= K blocks) that fits with one
// to spare (the occupancy query's count itself was not always reached, and the last
// cluster then waits for a whole part: 56 clusters of 5 took 15.8 us, not 12).  With
// more strips than that, some SMs would have two whole strips and others one: then
// Q < C strips are shared by C CTAs where that shortens the longest part (224 strips
// of K = 4096: 7 strips to 8 CTAs, 14 K blocks each instead of 16, 256 CTAs on 148 SMs).
int choose_parts(bool two_segments, int smem, int strips, int kblocks, const DeviceInfo& info,
                 int* C, int* Q) {
  *C = *Q = 1;
  const int most = kMaxCluster < kblocks ? kMaxCluster : kblocks;
  int resident[kMaxCluster + 1] = {};
  for (int cs = most; cs > 1; --cs) {
    if (int st = resident_clusters(cs, smem, info, &resident[cs])) return st;
    if (strips < resident[cs]) {
      *C = cs;
      return AOTK_OK;
    }
  }
  if (!two_segments || strips > 2 * info.sm_count) return AOTK_OK;
  int longest = kblocks;
  for (int cs = 3; cs <= most; ++cs) {
    for (int q = 2; q < cs; ++q) {
      const int part = (q * kblocks + cs - 1) / cs;
      if ((strips + q - 1) / q < resident[cs] && part < longest) {
        longest = part;
        *C = cs;
        *Q = q;
      }
    }
  }
  return AOTK_OK;
}

template <typename T, int MP, int STAGES, int SEGS, bool kAlias>
int launch_skinny(void* c, const void* a, const void* as, const void* b, const void* bs, int M,
                  int N, int K, cudaStream_t stream, const DeviceInfo& info) {
  using L = MxsLayout<MP, STAGES, SEGS, kAlias>;
  auto kernel = gemm_mxfp4_skinny_kernel<T, MP, STAGES, SEGS, kAlias>;
  if (int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kAlloc, info)) return st;
  CUtensorMap tw, tx;
  if (int st = make_tmap_2d_8bit(&tw, b, N, K / 2, K / 2, 128, kTileN)) return st;
  if (int st = make_tmap_2d_8bit(&tx, a, M, K / 2, K / 2, 128, MP)) return st;
  const int strips = (N - 1) / kTileN + 1;
  const int kblocks = (K - 1) / kBK + 1;
  int C, Q;
  if (int st = choose_parts(SEGS == 2, static_cast<int>(L::kAlloc), strips, kblocks, info, &C, &Q))
    return st;
  const int64_t blocks = static_cast<int64_t>((strips + Q - 1) / Q) * C;
  if (blocks > 0x7fffffffLL)
    return fail(AOTK_ERR_UNSUPPORTED, "aotk_mxfp4_gemm: N = %d is too large", N);

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kAlloc;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(C);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(
      &cfg, kernel, tw, tx, static_cast<const uint8_t*>(bs), static_cast<const uint8_t*>(as),
      static_cast<T*>(c), M, N, K, Q);
  if (e != cudaSuccess)
    return fail(AOTK_ERR_CUDA, "aotk_mxfp4_gemm launch (cluster %d): %s", C, cudaGetErrorString(e));
  return check_launch("aotk_mxfp4_gemm");
}

// Ring depth per width of A: two CTAs fit per SM.
template <typename T>
int dispatch(void* c, const void* a, const void* as, const void* b, const void* bs, int M, int N,
             int K, cudaStream_t s, const DeviceInfo& info) {
  if (M <= 16) return launch_skinny<T, 16, 4, 2, false>(c, a, as, b, bs, M, N, K, s, info);
  if (M <= 32) return launch_skinny<T, 32, 3, 2, false>(c, a, as, b, bs, M, N, K, s, info);
  if (M <= 64) return launch_skinny<T, 64, 4, 1, true>(c, a, as, b, bs, M, N, K, s, info);
  return launch_skinny<T, 128, 3, 1, true>(c, a, as, b, bs, M, N, K, s, info);
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
