// The norms around a residual block in one pass ("sandwich" norm):
//   h   = alpha * residual + gate * (x * rsqrt(mean(x^2) + eps) * post_weight)
//   out = h * rsqrt(mean(h^2) + eps) * pre_weight
// x is the block's output, h the next residual and out what the next block
// reads.  fp32 math; h and out are each rounded once (the second norm sees the
// unrounded h, so no error of h's rounding enters out).
//
// The row lives in registers from its one read to its two writes, so 2 rows
// are read and 2 written per row of the problem, which bounds the kernel by
// HBM.  A row is owned by TPR threads with VPT accesses of E elements each
// (16-byte vectors, or single elements where the row length or a pointer is
// not a multiple of 16 bytes); the two sums meet through warp shuffles and
// shared memory.  Longer rows take a kernel that reads the row again.
//
// gate is [gate_rows, gate_cols]: gate_cols is the row length or 1, and row r
// of the problem uses gate row r / (rows / gate_rows) - one row for all
// (per channel), one for each sequence, or one for each token.
#include "common.h"
#include "gemm_internal.h"
#include "sm100.cuh"
#include "vec.cuh"

namespace aotk {
namespace {

struct Gate {
  const void* ptr;       // null: no gate
  int64_t rows_per;      // rows of the problem per gate row
  int64_t row_stride;
  int col_stride;        // 1, or 0 for one value per row
};

template <typename T>
struct Args {
  const T* x;
  const T* residual;
  const T* post;
  const T* pre;
  T* out;
  T* h_out;
  Gate gate;
  float alpha, eps;
  int64_t rows;
  int cols;
};

// Sum over the threads of a row; `buf` holds one value per warp of the block.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    constexpr int WPR = TPR / 32;
    const int warp = threadIdx.x / 32;
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    v = 0.f;
    const int first = warp / WPR * WPR;
#pragma unroll
    for (int k = 0; k < WPR; ++k) v += buf[first + k];
  }
  return v;
}

template <typename T, int E>
struct Access;  // one access of E consecutive elements

template <typename T>
struct Access<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void load_cached(const T* p) { v = *p; }
  __device__ __forceinline__ void get(float* f) const { f[0] = Elem<T>::to_f(v); }
  __device__ __forceinline__ static void store(T* p, const float* f) { *p = Elem<T>::from_f(f[0]); }
};

template <typename T, int E>
struct Access {
  static_assert(E == Elem<T>::kPerVec, "16-byte accesses");
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = ld_stream(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void load_cached(const T* p) {
    v = ld_cached(reinterpret_cast<const uint4*>(p));
  }
  __device__ __forceinline__ void get(float* f) const { Elem<T>::unpack(v, f); }
  __device__ __forceinline__ static void store(T* p, const float* f) {
    st_stream(reinterpret_cast<uint4*>(p), Elem<T>::pack(f));
  }
};

// Two fp32 operations per instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 w, x, y, z;\n\t"
      "mov.b64 w, {%2, %3};\n\tmov.b64 x, {%4, %5};\n\tmov.b64 y, {%6, %7};\n\t"
      "fma.rn.f32x2 z, w, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

constexpr int threads_for(int tpr) { return tpr > 256 ? tpr : 256; }

template <typename T, int E, int VPT, int TPR>
__global__ void __launch_bounds__(threads_for(TPR)) sandwich_kernel(const Args<T> a) {
  constexpr int kThreads = threads_for(TPR);
  constexpr int RPB = kThreads / TPR;
  __shared__ float buf[2][kThreads / 32];
  const int t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
  const bool live = row < a.rows;
  const int64_t off = (live ? row : 0) * static_cast<int64_t>(a.cols);

  sm100::pdl_launch_dependents();
  sm100::pdl_wait_prior();
  const T* gate = static_cast<const T*>(a.gate.ptr);
  if (gate != nullptr && live) gate += row / a.gate.rows_per * a.gate.row_stride;

  // Everything that the row needs is requested before the first sum.
  Access<T, E> x[VPT], res[VPT], post[VPT], pre[VPT], g[VPT];
  float g_row = 1.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * TPR) * E;
    if (live && c < a.cols) {
      x[i].load(a.x + off + c);
      res[i].load(a.residual + off + c);
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * TPR) * E;
    if (live && c < a.cols) {
      post[i].load_cached(a.post + c);
      pre[i].load_cached(a.pre + c);
      if (gate != nullptr && a.gate.col_stride) g[i].load_cached(gate + c);
    }
  }
  if (gate != nullptr && live && !a.gate.col_stride) g_row = Elem<T>::to_f(gate[0]);
  const bool gate_cols = gate != nullptr && a.gate.col_stride;

  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (live && (t + i * TPR) * E < a.cols) {
      float f[E];
      x[i].get(f);
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(f[e], f[e], ss);
    }
  }
  ss = row_sum<TPR>(ss, buf[0]);
  const float inv = rsqrtf(ss / static_cast<float>(a.cols) + a.eps);

  float h[VPT][E];
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * TPR) * E;
    if (live && c < a.cols) {
      float r[E], w[E];
      x[i].get(h[i]);
      res[i].get(r);
      post[i].get(w);
#pragma unroll
      for (int e = 0; e < E; ++e) h[i][e] = h[i][e] * inv * w[e];
      if (gate_cols) {
        float gf[E];
        g[i].get(gf);
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] *= gf[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] *= g_row;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        h[i][e] = fmaf(a.alpha, r[e], h[i][e]);
        ss = fmaf(h[i][e], h[i][e], ss);
      }
      Access<T, E>::store(a.h_out + off + c, h[i]);
    }
  }
  ss = row_sum<TPR>(ss, buf[1]);
  const float inv_h = rsqrtf(ss / static_cast<float>(a.cols) + a.eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * TPR) * E;
    if (live && c < a.cols) {
      float w[E];
      pre[i].get(w);
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] *= h[i][e] * inv_h;
      Access<T, E>::store(a.out + off + c, w);
    }
  }
}

// ---- many rows: a ring of rows in shared memory ----------------------------------
//
// One persistent block per SM; a group of TPR threads takes every k-th row.  Each
// group keeps STAGES rows of x and of the residual on their way into shared memory
// by bulk copies (about 190 KB per SM in flight, whatever the threads wait for),
// which is what the two sums per row cost a kernel that loads into registers: at
// 8192 x 4096 bf16 that one keeps 96 KB in flight and stops at each sum.

constexpr int kRingThreads = 512;
constexpr int kRingBytes = 196608;
constexpr int kMaxStages = 8;
#ifndef RMIN
#define RMIN 1024
#define RTOT (1<<20)
#endif
constexpr int64_t kRingMinRow = RMIN, kRingMinTotal = RTOT;

__device__ unsigned g_norm_watchdog;
enum : unsigned { kWdRow = 262144u };

// Sum over the group's threads, and whether any of them failed.
template <int TPR>
__device__ __forceinline__ float group_sum(float v, float* buf, int group, int t, bool& bad) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR == 32) {
    bad = __any_sync(0xffffffffu, bad);
  } else {
    if ((t & 31) == 0) buf[t / 32] = v;
    int any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.s32 p, %3, 0;\n\t"
        "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
        "selp.s32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(group + 1), "n"(TPR), "r"(bad ? 1 : 0)
        : "memory");
    bad = any != 0;
    v = 0.f;
#pragma unroll
    for (int k = 0; k < TPR / 32; ++k) v += buf[k];
  }
  return v;
}

template <typename T, int VPT, int TPR>
__global__ void __launch_bounds__(kRingThreads, 1)
    sandwich_ring_kernel(const Args<T> a, int stages, int pitch) {
  using namespace sm100;
  constexpr int E = Elem<T>::kPerVec;
  constexpr int P = E / 2;  // pairs per vector
  constexpr int G = kRingThreads / TPR;
  constexpr int WPR = TPR / 32;
  extern __shared__ __align__(16) uint8_t ring[];  // [G][stages][x, residual][pitch]
  __shared__ float partial[G][2][WPR];
  __shared__ __align__(8) uint64_t bars[G][kMaxStages];
  __shared__ int abort_flag;
  const int group = threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * G;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * G + group;
  uint8_t* mine = ring + static_cast<int64_t>(group) * stages * 2 * pitch;
  const uint32_t bar0 = smem_addr(bars[group]);

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int g = 0; g < G; ++g)
      for (int k = 0; k < kMaxStages; ++k) mbar_init(smem_addr(&bars[g][k]), 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait_prior();

  auto request = [&](int64_t row, int stage) {  // one thread
    const uint32_t bytes = static_cast<uint32_t>(a.cols) * sizeof(T);
    const uint32_t bar = bar0 + 8u * stage;
    const uint32_t dst = smem_addr(mine + static_cast<int64_t>(stage) * 2 * pitch);
    mbar_arrive_expect_tx(bar, 2 * bytes);
    bulk_load(dst, a.x + row * a.cols, bytes, bar);
    bulk_load(dst + pitch, a.residual + row * a.cols, bytes, bar);
  };
  if (t == 0)
    for (int k = 0; k < stages && first + k * step < a.rows; ++k) request(first + k * step, k);

  // A thread's columns are the same in every row, so their weights stay in
  // registers (from L2 they would be as many bytes per row as x and the
  // residual), and so does the gate until its row changes.
  const T* gate = static_cast<const T*>(a.gate.ptr);
  const bool gate_cols = gate != nullptr && a.gate.col_stride;
  uint4 post[VPT], pre[VPT], g[VPT];
  float g_row = 1.f;
  int64_t g_at = -1;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * TPR) * E;
    if (c < a.cols) {
      post[i] = ld_cached(reinterpret_cast<const uint4*>(a.post + c));
      pre[i] = ld_cached(reinterpret_cast<const uint4*>(a.pre + c));
    }
  }

  int stage = 0;
  uint32_t phase = 0;
  for (int64_t row = first; row < a.rows; row += step) {
    if (gate != nullptr) {
      const int64_t at = row / a.gate.rows_per;
      if (at != g_at) {
        g_at = at;
        const T* gr = gate + at * a.gate.row_stride;
        if (gate_cols) {
#pragma unroll
          for (int i = 0; i < VPT; ++i) {
            const int c = (t + i * TPR) * E;
            if (c < a.cols) g[i] = ld_cached(reinterpret_cast<const uint4*>(gr + c));
          }
        } else {
          g_row = Elem<T>::to_f(*gr);
        }
      }
    }
    const uint4* xs = reinterpret_cast<const uint4*>(mine + static_cast<int64_t>(stage) * 2 * pitch);
    const uint4* rs = reinterpret_cast<const uint4*>(mine + (static_cast<int64_t>(stage) * 2 + 1) * pitch);
    T* h_row = a.h_out + row * a.cols;
    T* o_row = a.out + row * a.cols;
    bool bad = !mbar_wait_bounded(bar0 + 8u * stage, phase, &abort_flag, &g_norm_watchdog, kWdRow);

    float2 h[VPT][P];  // x, then h
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if ((t + i * TPR) * E < a.cols) {
        Elem<T>::unpack(xs[t + i * TPR], &h[i][0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) ss = fma2(h[i][e], h[i][e], ss);
      }
    }
    const float sum = group_sum<TPR>(ss.x + ss.y, partial[group][0], group, t, bad);
    if (bad) break;  // the whole group
    const float inv = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);

    ss = make_float2(0.f, 0.f);
    const float scale = gate_cols ? inv : inv * g_row;
    const float2 scale2 = make_float2(scale, scale), alpha2 = make_float2(a.alpha, a.alpha);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * TPR) * E;
      if (c < a.cols) {
        float2 w[P];
        Elem<T>::unpack(post[i], &w[0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) h[i][e] = mul2(mul2(h[i][e], scale2), w[e]);
        if (gate_cols) {
          Elem<T>::unpack(g[i], &w[0].x);
#pragma unroll
          for (int e = 0; e < P; ++e) h[i][e] = mul2(h[i][e], w[e]);
        }
        Elem<T>::unpack(rs[t + i * TPR], &w[0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          h[i][e] = fma2(alpha2, w[e], h[i][e]);
          ss = fma2(h[i][e], h[i][e], ss);
        }
        st_stream(reinterpret_cast<uint4*>(h_row + c), Elem<T>::pack(&h[i][0].x));
      }
    }
    const float sum_h = group_sum<TPR>(ss.x + ss.y, partial[group][1], group, t, bad);
    // The whole group has read the stage.
    if (t == 0 && row + stages * step < a.rows) request(row + stages * step, stage);
    const float inv_h = rsqrtf(sum_h / static_cast<float>(a.cols) + a.eps);
    const float2 inv_h2 = make_float2(inv_h, inv_h);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (t + i * TPR) * E;
      if (c < a.cols) {
        float2 w[P];
        Elem<T>::unpack(pre[i], &w[0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) w[e] = mul2(mul2(h[i][e], inv_h2), w[e]);
        st_stream(reinterpret_cast<uint4*>(o_row + c), Elem<T>::pack(&w[0].x));
      }
    }
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  // After a wait that gave up, copies may still be in flight.
  if (t == 0 && abort_flag)
    for (int k = 0; k < stages; ++k) mbar_drain(bar0 + 8u * k, phase);
}

// Any row length: one block per row; h is computed again from its inputs for
// the output pass, so that it is never rounded in between.
template <typename T>
__global__ void __launch_bounds__(256) sandwich_long_kernel(const Args<T> a) {
  __shared__ float buf[2][8];
  const int64_t row = blockIdx.x;
  const int64_t off = row * a.cols;
  float ss = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float f = Elem<T>::to_f(a.x[off + c]);
    ss = fmaf(f, f, ss);
  }
  ss = row_sum<256>(ss, buf[0]);
  const float inv = rsqrtf(ss / static_cast<float>(a.cols) + a.eps);
  const T* gate = static_cast<const T*>(a.gate.ptr);
  if (gate != nullptr) gate += row / a.gate.rows_per * a.gate.row_stride;
  auto h_at = [&](int c) {
    float v = Elem<T>::to_f(a.x[off + c]) * inv * Elem<T>::to_f(a.post[c]);
    if (gate != nullptr) v *= Elem<T>::to_f(gate[static_cast<int64_t>(c) * a.gate.col_stride]);
    return fmaf(a.alpha, Elem<T>::to_f(a.residual[off + c]), v);
  };
  ss = 0.f;
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float h = h_at(c);
    ss = fmaf(h, h, ss);
  }
  ss = row_sum<256>(ss, buf[1]);
  const float inv_h = rsqrtf(ss / static_cast<float>(a.cols) + a.eps);
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float h = h_at(c);
    a.h_out[off + c] = Elem<T>::from_f(h);
    a.out[off + c] = Elem<T>::from_f(h * inv_h * Elem<T>::to_f(a.pre[c]));
  }
}

template <typename T, int E, int VPT, int TPR>
int launch_rows(const Args<T>& a, cudaStream_t s) {
  constexpr int kThreads = threads_for(TPR);
  const int64_t blocks = (a.rows + kThreads / TPR - 1) / (kThreads / TPR);
  if (blocks > 0x7fffffffLL)
    return fail(AOTK_ERR_INVALID_ARGUMENT, "aotk_sandwich_rmsnorm: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, sandwich_kernel<T, E, VPT, TPR>, a);
  if (e != cudaSuccess)
    return fail(AOTK_ERR_CUDA, "aotk_sandwich_rmsnorm launch: %s", cudaGetErrorString(e));
  return check_launch("aotk_sandwich_rmsnorm");
}

template <typename T, int E>
int launch_access(const Args<T>& a, cudaStream_t s) {
    constexpr int V = E == 1 ? 8 : 4;  // accesses per thread
  const int n = a.cols / E;
  if (n <= 32) return launch_rows<T, E, 1, 32>(a, s);
  if (n <= V * 32) return launch_rows<T, E, V, 32>(a, s);
  if (n <= V * 64) return launch_rows<T, E, V, 64>(a, s);
  if (n <= V * 128) return launch_rows<T, E, V, 128>(a, s);
  if (n <= V * 256) return launch_rows<T, E, V, 256>(a, s);
  if (n <= V * 512) return launch_rows<T, E, V, 512>(a, s);
  if (n <= V * 1024) return launch_rows<T, E, V, 1024>(a, s);
  if (a.rows > 0x7fffffffLL)
    return fail(AOTK_ERR_INVALID_ARGUMENT, "aotk_sandwich_rmsnorm: too many rows");
  sandwich_long_kernel<T><<<static_cast<unsigned>(a.rows), 256, 0, s>>>(a);
  return check_launch("aotk_sandwich_rmsnorm");
}

template <typename T, int VPT, int TPR>
int launch_ring(const Args<T>& a, cudaStream_t s, const DeviceInfo& info) {
  constexpr int G = kRingThreads / TPR;
  const int pitch = a.cols * static_cast<int>(sizeof(T));
  int stages = kRingBytes / (G * 2 * pitch);
  if (stages > kMaxStages) stages = kMaxStages;
  auto kernel = sandwich_ring_kernel<T, VPT, TPR>;
  if (int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kRingBytes, info)) return st;
  const int64_t groups = (a.rows + G - 1) / G;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(groups < info.sm_count ? groups : info.sm_count), 1, 1);
  cfg.blockDim = dim3(kRingThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(G) * stages * 2 * pitch;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a, stages, pitch);
  if (e != cudaSuccess)
    return fail(AOTK_ERR_CUDA, "aotk_sandwich_rmsnorm launch: %s", cudaGetErrorString(e));
  return check_launch("aotk_sandwich_rmsnorm");
}

// The smallest group that holds a row in at most four vectors per thread.
template <typename T>
int dispatch_ring(const Args<T>& a, cudaStream_t s, const DeviceInfo& info) {
  const int n = a.cols / Elem<T>::kPerVec;
  if (n <= 2 * 32) return launch_ring<T, 2, 32>(a, s, info);
  if (n <= 3 * 32) return launch_ring<T, 3, 32>(a, s, info);
  if (n <= 4 * 32) return launch_ring<T, 4, 32>(a, s, info);
  if (n <= 3 * 64) return launch_ring<T, 3, 64>(a, s, info);
  if (n <= 4 * 64) return launch_ring<T, 4, 64>(a, s, info);
  if (n <= 3 * 128) return launch_ring<T, 3, 128>(a, s, info);
  if (n <= 4 * 128) return launch_ring<T, 4, 128>(a, s, info);
  if (n <= 3 * 256) return launch_ring<T, 3, 256>(a, s, info);
  if (n <= 4 * 256) return launch_ring<T, 4, 256>(a, s, info);
  if (n <= 3 * 512) return launch_ring<T, 3, 512>(a, s, info);
  return launch_ring<T, 4, 512>(a, s, info);
}

template <typename T>
int launch(void* out, void* h_out, const void* x, const void* residual, const void* post,
           const void* pre, const Gate& gate, double alpha, int64_t rows, int64_t cols, double eps,
           cudaStream_t s) {
  const Args<T> a = {static_cast<const T*>(x),    static_cast<const T*>(residual),
                     static_cast<const T*>(post), static_cast<const T*>(pre),
                     static_cast<T*>(out),        static_cast<T*>(h_out),
                     gate,                        static_cast<float>(alpha),
                     static_cast<float>(eps),     rows,
                     static_cast<int>(cols)};
  constexpr int E = Elem<T>::kPerVec;
  const bool vec = cols % E == 0 && aligned16(x) && aligned16(residual) && aligned16(post) &&
                   aligned16(pre) && aligned16(out) && aligned16(h_out) && aligned16(gate.ptr);
  // Rows of 1 to 32 KB, enough of them to fill the ring: the ring kernel.
  DeviceInfo info;
  if (int st = current_device_info(&info)) return st;
  const int64_t row_bytes = cols * static_cast<int64_t>(sizeof(T));
  if (vec && row_bytes >= kRingMinRow && row_bytes <= 32768 && rows * row_bytes >= kRingMinTotal)
    return dispatch_ring<T>(a, s, info);
  return vec ? launch_access<T, E>(a, s) : launch_access<T, 1>(a, s);
}

}  // namespace

int norm_watchdog(uint32_t* status, bool clear) {
  unsigned v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_norm_watchdog, sizeof(v));
  if (e != cudaSuccess) return fail(AOTK_ERR_CUDA, "watchdog read: %s", cudaGetErrorString(e));
  if (clear) {
    const unsigned zero = 0;
    e = cudaMemcpyToSymbol(g_norm_watchdog, &zero, sizeof(zero));
    if (e != cudaSuccess) return fail(AOTK_ERR_CUDA, "watchdog clear: %s", cudaGetErrorString(e));
  }
  *status |= v;
  return AOTK_OK;
}

}  // namespace aotk

extern "C" int aotk_sandwich_rmsnorm(void* out, void* h_out, const void* x, const void* residual,
                                     const void* post_weight, const void* pre_weight,
                                     const void* gate, int64_t gate_rows, int64_t gate_cols,
                                     double residual_scale, int64_t rows, int64_t cols, double eps,
                                     int dtype, void* stream) {
  using namespace aotk;
  const char* who = "aotk_sandwich_rmsnorm";
  if (rows < 0 || cols < 0) return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (!valid_dtype(dtype)) return fail(AOTK_ERR_UNSUPPORTED, "%s: unsupported dtype %d", who, dtype);
  if (rows == 0 || cols == 0) return AOTK_OK;
  if (!out || !h_out || !x || !residual || !post_weight || !pre_weight)
    return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (cols > 0x3fffffffLL) return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: row too long", who);
  Gate g = {nullptr, 1, 0, 0};
  if (gate) {
    if (gate_rows < 1 || rows % gate_rows != 0 || (gate_cols != cols && gate_cols != 1))
      return fail(AOTK_ERR_INVALID_ARGUMENT,
                  "%s: gate [%lld, %lld] does not fit rows [%lld, %lld]", who, (long long)gate_rows,
                  (long long)gate_cols, (long long)rows, (long long)cols);
    g = {gate, rows / gate_rows, gate_cols, gate_cols == cols ? 1 : 0};
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case AOTK_FLOAT32:
      return launch<float>(out, h_out, x, residual, post_weight, pre_weight, g, residual_scale,
                           rows, cols, eps, s);
    case AOTK_FLOAT16:
      return launch<__half>(out, h_out, x, residual, post_weight, pre_weight, g, residual_scale,
                            rows, cols, eps, s);
    default:
      return launch<__nv_bfloat16>(out, h_out, x, residual, post_weight, pre_weight, g,
                                   residual_scale, rows, cols, eps, s);
  }
}
