// Product of two microscaled 4-bit matrices: C[m, n] = sum_k A[m, k] B[n, k],
// A [M, K / 2] and B [N, K / 2] codes with scale tiles as in mxfp4.cu, fp32
// accumulation, one rounding to the output type.  (M <= 128: gemm_mxfp4_skinny.cu.)
//
// Persistent tcgen05 kernel on tiles of 128 CG x BN of C, CG = 1 or 2 CTAs (SMs)
// per tile:
//   * codes are read as bytes by TMA in blocks of 256 elements of K (one 128-byte
//     swizzle row), SUB blocks per stage, both operands K-major; scale tiles (512
//     bytes per 128 rows x 4 blocks, already in the order of TMEM) by TMA as rows
//     of 512 bytes;
//   * per stage one thread copies the scales to TMEM and issues up to 4 SUB MMAs of
//     K = 64 (kind::mxf4).  TMEM holds one scale area per stage of the ring, so a
//     stage's scales are overwritten only when its barrier has shown that the
//     MMAs which read them are done;
//   * CG = 2 (cta_group::2): each CTA stages its 128 rows of A, BN / 2 of the rows
//     of B and the scales of its rows of A and of all rows of B; the first CTA
//     holds the stage barriers and issues all MMAs; each reads out its 128 rows;
//   * 8 epilogue warps read a tile out of TMEM at once, 128 columns each at
//     BN = 256, so one accumulator is enough there (it and the scales would not
//     fit twice into 512 columns); narrower tiles have two.  A lane holds a row and
//     writes it in whole 32-byte sectors, without shared memory, which is the
//     ring's (staged TMA stores and a stage less: 8192^3 228 -> 232 us).  Where rows
//     do not start on 16 bytes, the memory of one or two stages turns the rows for
//     stores along them.
// What bounds it: tiles of one CTA by operand traffic out of L2, about 16.5 TB/s
// over the chip.  128 x 256 tiles moved 51 KB per 256 of K, 0.455 us where the MMAs
// take 0.27; the pairs of CTAs that took their place move 35 KB for the same work and
// end at the power cap.  Of the one-CTA tiles left, for grids that do not fill the
// chip with pairs, 128 x 64 ones are bound by the work per stage of the issuing
// warps, hence SUB = 2 there (128 x 6144 x 4096 7.1 -> 6.6 us, 128 x 4096 x 14336
// 15.2 -> 13.3).  Sending the
// scales a stage ahead of their MMAs, or between them, gained nothing or lost.
// K is padded by zeros (TMA fill); MMAs stop at the last 64 elements that exist.
// Rows beyond M or N may multiply stale or foreign scales, and are not stored.
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

constexpr int kBM = 128;          // rows of a tile per CTA
constexpr int kBK = 256;          // elements of K per stage (128 bytes of codes)
constexpr int kStepK = 64;        // elements of K per MMA
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;  // producer, MMA and epilogue warps
constexpr int kGroupRows = 2048;  // rows of A per raster group
constexpr uint32_t kScaleTile = 512;
// A wait for a tile's whole sum lasts as long as K does.  The bound of all waits (2e9
// cycles, sm100.cuh) must not end it: 2^20 K blocks take at most 0.9e9 cycles.
constexpr int64_t kMaxK = int64_t{1} << 28;

enum : unsigned { kWdProducer = 4096u, kWdMma = 8192u, kWdEpilogue = 16384u };

// SUB: K blocks per stage.
template <int CG, int BN, int STAGES, int SUB>
struct MxLayout {
  static constexpr int kScaleTilesN = BN > 128 ? 2 : 1;  // scale tiles along N
  static constexpr uint32_t kABlock = kBM * 128;
  static constexpr uint32_t kBBlock = BN / CG * 128;
  static constexpr uint32_t kABytes = SUB * kABlock;
  static constexpr uint32_t kBBytes = SUB * kBBlock;
  static constexpr uint32_t kSfBox = 2 * SUB * kScaleTile;  // the K tiles of a stage
  static constexpr uint32_t kSfBytes = (1 + kScaleTilesN) * kSfBox;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes + kSfBytes;
  static constexpr uint32_t kOffA = 0;
  static constexpr uint32_t kOffB = kOffA + STAGES * kABytes;
  static constexpr uint32_t kOffSf = kOffB + STAGES * kBBytes;
  static constexpr uint32_t kOffBar = kOffSf + STAGES * kSfBytes;
  // Staging of unaligned rows: 4 KB per epilogue warp in A's last one or two stages.
  static constexpr uint32_t kCBuf = 32 * 128;
  static constexpr int kStagingStages = kABytes >= kEpiWarps * kCBuf ? 1 : 2;
  static constexpr uint32_t kOffC = kOffA + (STAGES - kStagingStages) * kABytes;
  static_assert(kEpiWarps * kCBuf <= kStagingStages * kABytes, "staging fits");
  static_assert(STAGES > kStagingStages + 1, "a ring is left beside the staging");
  static constexpr uint32_t kNumBars = 2 * STAGES + 5;  // full, empty, tfull x2, release x2, drain
  static constexpr uint32_t kOffMisc = kOffBar + kNumBars * 8;
  static constexpr uint32_t kAlloc = kOffMisc + 16 + 1024;
  static_assert(kAlloc <= 232448, "227 KB of shared memory");
  // TMEM columns: accumulators, then 4 columns per scale tile and stage.
  static constexpr int kSfCols = 2 * SUB * 4 * (1 + kScaleTilesN);
  static constexpr int kAccs = 2 * BN + STAGES * kSfCols <= 512 ? 2 : 1;
  static constexpr int kSfBase = kAccs * BN;
  static constexpr int kTmemCols = kSfBase + STAGES * kSfCols > 256 ? 512 : 256;
  static_assert(kSfBase + STAGES * kSfCols <= kTmemCols, "TMEM columns");
};

// Tiles in groups of `group` M tiles, M fastest within a group (L2 reuse).
__device__ __forceinline__ void tile_coords(int tile, int group, int tiles_m, int tiles_n, int& mb,
                                            int& nb) {
  const int per_group = group * tiles_n;
  const int g = tile / per_group;
  const int first_m = g * group;
  const int gm = min(tiles_m - first_m, group);
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

enum : int { kRowsAny = 0, kRows4 = 1, kRows16 = 2, kRows32 = 3 };  // bytes that rows of C start on

// Writes `bytes` of each staged row of 128 bytes as units of type U along the rows,
// eight units per lane at a time.
template <typename U>
__device__ __forceinline__ void write_rows(uint8_t* p, int64_t pitch, const uint8_t* buf, int lane,
                                           int bytes, int rows) {
  constexpr int kUnits = 4 / sizeof(U);  // per lane and row
  constexpr int kRows = 8 / kUnits;
  auto at = [&](int k) { return (lane + 32 * k) * static_cast<int>(sizeof(U)); };
  auto unit = [&](int rr, int k) {
    return *reinterpret_cast<const U*>(buf + rr * 128 + ((at(k) / 16 ^ (rr & 7)) << 4) + at(k) % 16);
  };
  int rr = 0;
  for (; rr + kRows <= rows; rr += kRows, p += kRows * pitch) {
    U v[kRows][kUnits];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int k = 0; k < kUnits; ++k) v[i][k] = unit(rr + i, k);
    if (bytes == 128) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int k = 0; k < kUnits; ++k) *reinterpret_cast<U*>(p + i * pitch + at(k)) = v[i][k];
    } else {
#pragma unroll
      for (int k = 0; k < kUnits; ++k)
        if (at(k) < bytes)
#pragma unroll
          for (int i = 0; i < kRows; ++i) *reinterpret_cast<U*>(p + i * pitch + at(k)) = v[i][k];
    }
  }
  for (; rr < rows; ++rr, p += pitch)
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
      if (at(k) < bytes) *reinterpret_cast<U*>(p + at(k)) = unit(rr, k);
}

// Writes a warp's 32 rows x 128 bytes of accumulators (lane = row) to C at (x, y).
// A lane writes its row's vectors; rows that do not start on 16 bytes are turned
// through 4 KB of shared memory and written along the row in words, if they start on
// 4 bytes, or elements (900 x 28611 x 832 to fp32 from row by row 57 -> 43 us, whole
// sectors 33; bf16 31, 24; pure writes run at about 3.7 TB/s).
template <typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ c, const uint32_t* r, uint8_t* buf,
                                            int lane, int x, int y, int M, int N, int rows_on) {
  constexpr int kChunk = 128 / sizeof(T);
  constexpr int kVec = 16 / sizeof(T);
  auto vec = [&](int j) {
    return make_uint4(pack_word<T>(r, 4 * j), pack_word<T>(r, 4 * j + 1), pack_word<T>(r, 4 * j + 2),
                      pack_word<T>(r, 4 * j + 3));
  };
  if (rows_on >= kRows16) {
    if (y + lane >= M) return;
    T* p = c + static_cast<int64_t>(y + lane) * N + x;
    auto one = [&](int j) {
      if (x + j * kVec < N) st_stream(reinterpret_cast<uint4*>(p + j * kVec), vec(j));
    };
    auto two = [&](int j) {
      if (x + (j + 1) * kVec < N)
        st_stream32(p + j * kVec, vec(j), vec(j + 1));
      else
        one(j);
    };
    // Whole sectors also where every other row starts in the middle of one.
    if (rows_on == kRows32 || reinterpret_cast<uintptr_t>(p) % 32 == 0) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) two(j);
    } else {
      one(0);
#pragma unroll
      for (int j = 1; j < 7; j += 2) two(j);
      one(7);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    *reinterpret_cast<uint4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) = vec(j);
  __syncwarp();
  const int rows = min(32, M - y), bytes = min(kChunk, N - x) * static_cast<int>(sizeof(T));
  uint8_t* p = reinterpret_cast<uint8_t*>(c + static_cast<int64_t>(y) * N + x);
  const int64_t pitch = static_cast<int64_t>(N) * sizeof(T);
  if (sizeof(T) == 4 || rows_on == kRows4)
    write_rows<uint32_t>(p, pitch, buf, lane, bytes, rows);
  else
    write_rows<uint16_t>(p, pitch, buf, lane, bytes, rows);
  __syncwarp();
}

template <typename T, int CG, int BN, int STAGES, int SUB>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmA,
                      const __grid_constant__ CUtensorMap tmB,
                      const __grid_constant__ CUtensorMap tmSa,
                      const __grid_constant__ CUtensorMap tmSb, T* __restrict__ c, int M, int N,
                      int K, int rows_on) {
  using L = MxLayout<CG, BN, STAGES, SUB>;
  constexpr int kTileM = CG * kBM;
  constexpr int kGroup = kGroupRows / kTileM;
  constexpr int kChunk = 128 / sizeof(T);                // columns of 128 bytes of output
  constexpr int kHalves = BN / 2 >= kChunk ? 2 : 1;      // warps that share a row's columns
  constexpr int kRead = BN / kHalves;                    // columns read by a warp
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
  const int rank = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0;  // 0 issues the MMAs
  const int worker = static_cast<int>(blockIdx.x) / CG;
  const int workers = static_cast<int>(gridDim.x) / CG;
  const int tiles_m = (M + kTileM - 1) / kTileM;
  const int tiles_n = (N + BN - 1) / BN;
  const int num_tiles = tiles_m * tiles_n;
  const int kblocks = (K + SUB * kBK - 1) / (SUB * kBK);  // stages
  const int sf_tiles_k = (K + 127) / 128;
  const int stages = rows_on < kRows16 ? STAGES - L::kStagingStages : STAGES;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSa);
    tma_prefetch_desc(&tmSb);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(release_bar(a), 4 * kHalves * CG);  // the epilogue warps of all CTAs
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(smem_addr(tmem_slot), L::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(smem_addr(tmem_slot), L::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) {  // both CTAs' barriers before any use across
    cluster_arrive_relaxed();
    cluster_wait();
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Global memory is touched only from here on, once the previous kernel on
  // the stream has completed (programmatic dependent launch).
  pdl_wait_prior();

  if (warp == 0) {
    // ---------------- producer (every CTA) ----------------
    const bool elected = elect_one();
    int stage = 0;
    uint32_t phase = 0;
    int issued = 0;
    bool ok = true;
    for (int tile = worker; ok && tile < num_tiles; tile += workers) {
      int mb, nb;
      tile_coords(tile, kGroup, tiles_m, tiles_n, mb, nb);
      const int row_a = mb * kTileM + rank * kBM;
      const int row_b = nb * BN + rank * (BN / CG);
      const int sa_row = (CG * mb + rank) * sf_tiles_k;
      const int sb_row = nb * BN / 128 * sf_tiles_k;
      for (int kb = 0; kb < kblocks; ++kb) {
        ok = mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, wd, kWdProducer);
        if (!ok) break;
        // Boxes of scales are always 2 SUB tiles: the last may belong to the next
        // 128 rows, or be zeros beyond the last.  No MMA reads them then.
        const uint32_t a_dst = base + L::kOffA + stage * L::kABytes;
        const uint32_t b_dst = base + L::kOffB + stage * L::kBBytes;
        const uint32_t sf = base + L::kOffSf + stage * L::kSfBytes;
        if (elected) {
          if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), CG * L::kStageBytes);
          if constexpr (CG == 2) {
            const uint32_t fb = map_to_rank(full_bar(stage), 0);
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
              tma_load_2d_pair(a_dst + i * L::kABlock, &tmA, (kb * SUB + i) * 128, row_a, fb);
              tma_load_2d_pair(b_dst + i * L::kBBlock, &tmB, (kb * SUB + i) * 128, row_b, fb);
            }
            tma_load_2d_pair(sf, &tmSa, 0, sa_row + 2 * SUB * kb, fb);
#pragma unroll
            for (int j = 0; j < L::kScaleTilesN; ++j)
              tma_load_2d_pair(sf + (1 + j) * L::kSfBox, &tmSb, 0,
                               sb_row + j * sf_tiles_k + 2 * SUB * kb, fb);
          } else {
            const uint32_t fb = full_bar(stage);
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
              tma_load_2d(a_dst + i * L::kABlock, &tmA, (kb * SUB + i) * 128, row_a, fb);
              tma_load_2d(b_dst + i * L::kBBlock, &tmB, (kb * SUB + i) * 128, row_b, fb);
            }
            tma_load_2d(sf, &tmSa, 0, sa_row + 2 * SUB * kb, fb);
#pragma unroll
            for (int j = 0; j < L::kScaleTilesN; ++j)
              tma_load_2d(sf + (1 + j) * L::kSfBox, &tmSb, 0,
                          sb_row + j * sf_tiles_k + 2 * SUB * kb, fb);
          }
        }
        __syncwarp();
        ++issued;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // The first CTA's full barriers see every load: drain there.  The second is sent
    // commits, and does not leave before the last of them have arrived (those of tfull
    // are the epilogue's).
    if (elected) {
      int s = stage;
      uint32_t p = phase;
      for (int i = 0; i < stages && i < issued; ++i) {
        if (--s < 0) {
          s = stages - 1;
          p ^= 1u;
        }
        if (!mbar_drain(rank == 0 ? full_bar(s) : empty_bar(s), p) && rank != 0) break;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA (first CTA) ----------------
    if (rank == 0) {
      const bool elected = elect_one();
      auto commit = [&](uint32_t bar) {  // on the barrier of every CTA of the tile
        if constexpr (CG == 2)
          umma_commit_pair(bar, 0x3);
        else
          umma_commit(bar);
      };
      auto copy_scales = [&](uint32_t taddr, uint64_t desc) {
        if constexpr (CG == 2)
          tmem_cp_scales_pair(taddr, desc);
        else
          tmem_cp_scales(taddr, desc);
      };
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;  // tiles so far
      bool ok = true;
      for (int tile = worker; ok && tile < num_tiles; tile += workers, ++it) {
        const int acc = it % L::kAccs;
        if (it >= L::kAccs) {  // the accumulator's last tile has been read out
          ok = mbar_wait_warp(release_bar(acc), (it / L::kAccs - 1) & 1, abort_flag, wd, kWdMma);
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        int mb, nb;
        tile_coords(tile, kGroup, tiles_m, tiles_n, mb, nb);
        // A 64-column tile may be the upper half of its scale tile: 2 columns on.
        const uint32_t sfb_shift = BN == 64 ? (nb & 1) * 2 : 0;
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = mbar_wait_warp(full_bar(stage), phase, abort_flag, wd, kWdMma);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sfa = tmem_base + L::kSfBase + stage * L::kSfCols;
          const uint32_t sfb = sfa + 8 * SUB;
          const uint64_t sd = sdesc_scales(base + L::kOffSf + stage * L::kSfBytes);
          const uint64_t ad = sdesc_sw128(base + L::kOffA + stage * L::kABytes, 16, 1024);
          const uint64_t bd = sdesc_sw128(base + L::kOffB + stage * L::kBBytes, 16, 1024);
          const int steps =
              min(SUB * kBK / kStepK, (K - kb * SUB * kBK + kStepK - 1) / kStepK);
          if (elected) {
#pragma unroll
            for (int t = 0; t < 2 * SUB; ++t) {  // 128 elements: one scale tile each
              if (2 * t < steps) {
                // Descriptors count addresses in units of 16 bytes.
                copy_scales(sfa + 4 * t, sd + t * (kScaleTile / 16));
#pragma unroll
                for (int j = 0; j < L::kScaleTilesN; ++j)
                  copy_scales(sfb + 4 * (L::kScaleTilesN * t + j),
                              sd + (2 * SUB * (j + 1) + t) * (kScaleTile / 16));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int k = 2 * t + h;
                  if (k < steps) {
                    const uint32_t sfb_t = sfb + 4 * L::kScaleTilesN * t + sfb_shift;
                    const uint32_t idesc = idesc_mxf4(kTileM, BN, 2 * h);
                    const bool add = kb > 0 || k > 0;
                    // Block k / 4 of the stage, 32 bytes on per step.
                    const uint64_t ak = ad + (k / 4) * (L::kABlock / 16) + (k % 4) * 2;
                    const uint64_t bk = bd + (k / 4) * (L::kBBlock / 16) + (k % 4) * 2;
                    if constexpr (CG == 2)
                      umma_mxf4_pair(d_tmem, ak, bk, idesc, sfa + 4 * t, sfb_t, add);
                    else
                      umma_mxf4(d_tmem, ak, bk, idesc, sfa + 4 * t, sfb_t, add);
                  }
                }
              }
            }
            commit(empty_bar(stage));
          }
          __syncwarp();
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (elected) commit(tfull_bar(acc));
        __syncwarp();
      }
      if (elected) {
        if constexpr (CG == 2)
          umma_commit_pair(drain_bar, 0x1);
        else
          umma_commit(drain_bar);
        mbar_drain(drain_bar, 0);
        // The second CTA signals its last read-outs here, and no further tile waits for
        // them: the cluster's barriers are relaxed, so that they do not show it either.
        if constexpr (CG == 2)
          for (int i = it > L::kAccs ? it - L::kAccs : 0; i < it; ++i)
            if (!mbar_drain(release_bar(i % L::kAccs), (i / L::kAccs) & 1)) break;
      }
    }
    __syncwarp();
  } else if ((warp - 2) / 4 < kHalves) {
    // ---------------- epilogue (every CTA) ----------------
    const int q = warp & 3;            // the quarter of TMEM lanes that this warp may read
    const int half = (warp - 2) / 4;   // its columns of the tile
    uint8_t* buf = smem + L::kOffC + (warp - 2) * L::kCBuf;
    int it = 0;
    for (int tile = worker; tile < num_tiles; tile += workers, ++it) {
      int mb, nb;
      tile_coords(tile, kGroup, tiles_m, tiles_n, mb, nb);
      const int acc = it % L::kAccs;
      int ok = 1;
      if (lane == 0)
        ok = mbar_wait_bounded(tfull_bar(acc), (it / L::kAccs) & 1, abort_flag, wd, kWdEpilogue);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      const uint32_t trow =
          tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * BN + half * kRead;
      uint32_t r[kRead];
#pragma unroll
      for (int j = 0; j < kRead; j += 32) tmem_ld_32x32b_x32(trow + j, r + j);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2)
          mbar_arrive_cluster(map_to_rank(release_bar(acc), 0));
        else
          mbar_arrive(release_bar(acc));
      }
      const int y = mb * kTileM + rank * kBM + q * 32;
#pragma unroll
      for (int j = 0; j < kRead / kChunk; ++j) {
        const int x = nb * BN + half * kRead + j * kChunk;
        if (x < N && y < M)
          store_chunk<T>(c, r + j * kChunk, buf, lane, x, y, M, N, rows_on);
      }
    }
  }

  // No CTA frees TMEM or exits while its pair may still use its shared memory
  // (operands, barriers) or its TMEM.
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) {
    cluster_arrive_relaxed();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2)
      tmem_dealloc_pair(tmem_base, L::kTmemCols);
    else
      tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

int64_t tile_count(int cg, int bn, int M, int N) {
  return static_cast<int64_t>((M - 1) / (cg * kBM) + 1) * ((N - 1) / bn + 1);
}

template <typename T, int CG, int BN, int STAGES, int SUB>
int launch_tiles(void* c, const void* a, const void* as, const void* b, const void* bs, int M,
                 int N, int K, cudaStream_t stream, const DeviceInfo& info) {
  using L = MxLayout<CG, BN, STAGES, SUB>;
  auto kernel = gemm_mxfp4_kernel<T, CG, BN, STAGES, SUB>;
  if (int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kAlloc, info)) return st;
  CUtensorMap ta, tb, tsa, tsb;
  const uint64_t sf_tiles_k = (static_cast<uint64_t>(K) + 127) / 128;
  if (int st = make_tmap_2d_8bit(&ta, a, M, K / 2, K / 2, 128, kBM)) return st;
  if (int st = make_tmap_2d_8bit(&tb, b, N, K / 2, K / 2, 128, BN / CG)) return st;
  if (int st = make_tmap_blocks512(&tsa, as, (static_cast<uint64_t>(M) + 127) / 128 * sf_tiles_k, 2 * SUB))
    return st;
  if (int st = make_tmap_blocks512(&tsb, bs, (static_cast<uint64_t>(N) + 127) / 128 * sf_tiles_k, 2 * SUB))
    return st;
  const uintptr_t start = reinterpret_cast<uintptr_t>(c) | static_cast<uintptr_t>(N * sizeof(T));
  const int rows_on = start % 32 == 0 ? kRows32 : start % 16 == 0 ? kRows16
                      : start % 4 == 0 ? kRows4 : kRowsAny;
  const int64_t tiles = tile_count(CG, BN, M, N);
  if (tiles > 0x3fffffffLL)
    return fail(AOTK_ERR_UNSUPPORTED, "aotk_mxfp4_gemm: output of %d x %d has too many tiles", M, N);
  const int64_t workers = info.sm_count / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(CG * (tiles < workers ? tiles : workers)), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kAlloc;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  cudaError_t e =
      cudaLaunchKernelEx(&cfg, kernel, ta, tb, tsa, tsb, static_cast<T*>(c), M, N, K, rows_on);
  if (e != cudaSuccess)
    return fail(AOTK_ERR_CUDA, "aotk_mxfp4_gemm launch: %s", cudaGetErrorString(e));
  return check_launch("aotk_mxfp4_gemm");
}

// Whether M <= 128 rows go to the kernel that splits K and streams the weight at two
// CTAs per SM (gemm_mxfp4_skinny.cu) or to one-CTA tiles.  The former's exchange of
// partial sums grows with M, the latter go through K one block after the other; up
// to 32 rows the former always won.  Estimates in us from graph replays on 148 SMs,
// weight from HBM (split / 64-column tiles / 128-column tiles measured): 128 rows,
// N x K = 6144 x 4096 12.3 / 6.6 / 7.6, 4096 x 14336 13.2 / 13.3 / 16.7, 28672 x 4096
// 17.2 / 19.0 / 15.8, 1024 x 8192 8.2 / 9.0 / 11.1; 64 rows, 28672 x 4096 14.5 / 18 / 15.
bool prefer_split(int M, int N, int K, int sm_count) {
  if (M <= 32) return true;
  const double weight_kb = static_cast<double>(N) * K * (17.0 / 32) / 1024;
  const int kblocks = (K - 1) / kBK + 1;
  auto tiles = [&](int bn, double per_block) {
    const int64_t rounds = (tile_count(1, bn, M, N) + sm_count - 1) / sm_count;
    const double loop = per_block * kblocks * static_cast<double>(rounds);
    const double stream = weight_kb / 5100;
    return 3.8 + (loop > stream ? loop : stream);
  };
  const double t64 = tiles(64, 0.167), t128 = tiles(128, 0.241);
  const double split = 2.5 + 0.039 * M + weight_kb / 4900;
  return split <= t64 && split <= t128;
}

// The kernel for a problem (AOTK_MXFP4_*).
int path_of(int M, int N, int K, int sm_count) {
  if (M <= kSkinnyMaxM && prefer_split(M, N, K, sm_count)) return AOTK_MXFP4_SPLIT;
  // Rounds of tiles on the SMs, times what a round takes against one of 256-column
  // pairs (per 256 of K at full load 0.40 us; 0.29, 0.31 and 0.23 for the others).
  auto cost = [&](int cg, int bn, double round) {
    const int64_t workers = sm_count / cg;
    return round * static_cast<double>((tile_count(cg, bn, M, N) + workers - 1) / workers);
  };
  const double pair256 = cost(2, 256, 1.0), pair128 = cost(2, 128, 0.7);
  const double one128 = cost(1, 128, 0.77), one64 = cost(1, 64, 0.58);
  const double pairs = pair256 < pair128 ? pair256 : pair128;
  const double ones = one128 < one64 ? one128 : one64;
  if (pairs <= ones) return pair256 <= pair128 ? AOTK_MXFP4_PAIR_256 : AOTK_MXFP4_PAIR_128;
  return one128 <= one64 ? AOTK_MXFP4_ONE_128 : AOTK_MXFP4_ONE_64;
}

template <typename T>
int dispatch(int path, void* c, const void* a, const void* as, const void* b, const void* bs, int M,
             int N, int K, cudaStream_t s, const DeviceInfo& info) {
  switch (path) {
    case AOTK_MXFP4_PAIR_256:
      return launch_tiles<T, 2, 256, 6, 1>(c, a, as, b, bs, M, N, K, s, info);
    case AOTK_MXFP4_PAIR_128:
      return launch_tiles<T, 2, 128, 8, 1>(c, a, as, b, bs, M, N, K, s, info);
    case AOTK_MXFP4_ONE_128:
      return launch_tiles<T, 1, 128, 6, 1>(c, a, as, b, bs, M, N, K, s, info);
    default: return launch_tiles<T, 1, 64, 4, 2>(c, a, as, b, bs, M, N, K, s, info);
  }
}

// Arguments that do not depend on memory or a device.
int check_sizes(const char* who, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0) return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (K % 32 != 0)
    return fail(AOTK_ERR_UNSUPPORTED, "%s: K = %lld is not a multiple of the block size 32", who,
                (long long)K);
  return AOTK_OK;
}

int check_limits(const char* who, int64_t M, int64_t N, int64_t K) {
  if (M > 0x7fffff00LL || N > 0x7fffff00LL)
    return fail(AOTK_ERR_UNSUPPORTED, "%s: extents above 2^31 - 256", who);
  if (K > kMaxK)
    return fail(AOTK_ERR_UNSUPPORTED, "%s: K = %lld is above 2^28", who, (long long)K);
  return AOTK_OK;
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
  if (int st = check_sizes(who, M, N, K)) return st;
  if (!valid_dtype(out_dtype))
    return fail(AOTK_ERR_UNSUPPORTED, "%s: unsupported output dtype %d", who, out_dtype);
  if (M == 0 || N == 0) return AOTK_OK;
  if (!c || (K > 0 && (!a || !a_scales || !b || !b_scales)))
    return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (int st = check_limits(who, M, N, K)) return st;
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
  const int path = path_of(m, n, k, info.sm_count);
  if (path == AOTK_MXFP4_SPLIT)
    return gemm_mxfp4_skinny(c, a, a_scales, b, b_scales, m, n, k, out_dtype, stream, info);
  switch (out_dtype) {
    case AOTK_FLOAT32: return dispatch<float>(path, c, a, a_scales, b, b_scales, m, n, k, s, info);
    case AOTK_FLOAT16: return dispatch<__half>(path, c, a, a_scales, b, b_scales, m, n, k, s, info);
    default: return dispatch<__nv_bfloat16>(path, c, a, a_scales, b, b_scales, m, n, k, s, info);
  }
}

extern "C" int aotk_mxfp4_gemm_path(int64_t M, int64_t N, int64_t K, int sm_count, int* path) {
  using namespace aotk;
  const char* who = "aotk_mxfp4_gemm_path";
  if (int st = check_sizes(who, M, N, K)) return st;
  if (!path || M == 0 || N == 0 || K == 0 || sm_count < 2)
    return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: bad arguments", who);
  if (int st = check_limits(who, M, N, K)) return st;
  *path = path_of((int)M, (int)N, (int)K, sm_count);
  return AOTK_OK;
}
