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

  Access<T, E> x[VPT], res[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * TPR) * E;
    if (live && c < a.cols) {
      x[i].load(a.x + off + c);
      res[i].load(a.residual + off + c);
    }
  }
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

  const T* gate = static_cast<const T*>(a.gate.ptr);
  if (gate != nullptr && live) gate += row / a.gate.rows_per * a.gate.row_stride;
  float h[VPT][E];
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (t + i * TPR) * E;
    if (live && c < a.cols) {
      float r[E], w[E];
      x[i].get(h[i]);
      res[i].get(r);
      Access<T, E> wv;
      wv.load_cached(a.post + c);
      wv.get(w);
#pragma unroll
      for (int e = 0; e < E; ++e) h[i][e] = h[i][e] * inv * w[e];
      if (gate != nullptr) {
        float g[E];
        if (a.gate.col_stride) {
          Access<T, E> gv;
          gv.load_cached(gate + c);
          gv.get(g);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) g[e] = Elem<T>::to_f(gate[0]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) h[i][e] *= g[e];
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
      Access<T, E> wv;
      wv.load_cached(a.pre + c);
      wv.get(w);
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] *= h[i][e] * inv_h;
      Access<T, E>::store(a.out + off + c, w);
    }
  }
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
  sandwich_kernel<T, E, VPT, TPR><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(a);
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
  return vec ? launch_access<T, E>(a, s) : launch_access<T, 1>(a, s);
}

}  // namespace
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
