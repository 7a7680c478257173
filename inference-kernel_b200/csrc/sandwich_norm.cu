// The norms around a residual block in one pass ("sandwich" norm):
//   h   = alpha * residual + gate * (x * rsqrt(mean(x^2) + eps) * post_weight)
//   out = h * rsqrt(mean(h^2) + eps) * pre_weight
// x is the block's output, h the next residual and out what the next block
// reads.  fp32 math; h and out are each rounded once (the second norm sees the
// unrounded h, so no error of h's rounding enters out).
//
// Two rows are read and two written per row of the problem, which bounds it by
// HBM: the row lives in registers from its one read to its two writes, and the
// two sums meet through warp shuffles and shared memory.  Three kernels:
//   * sandwich_kernel: TPR threads per row hold it in registers, everything
//     requested before the first sum: rows below 1 KB, few rows (less than 1 MB in
//     all), and rows of up to 64 KB that are too long for the next;
//   * sandwich_ring_kernel: 1 MB or more of rows of 1 to 48 KB (32 KB where they do not
//     start on 16 bytes), streamed through shared memory;
//   * sandwich_long_kernel: rows above 64 KB, or tensors that do not start on 16
//     bytes: the row is read three times.
//
// Squares of bf16's and fp32's largest numbers (from about 1.8e19 on) and, with a
// small eps, of their smallest leave fp32's range, where rms(v) itself is of order 1.
// Rows whose mean square shows that are computed again (row_out_of_range), which takes
// about 17 times as long; the others pay a few comparisons.
//
// gate is [gate_rows, gate_cols]: gate_cols is the row length or 1, and row r
// of the problem uses gate row r / (rows / gate_rows) - one row for all
// (per channel), one for each sequence, or one for each token.
#include <type_traits>

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
  int64_t total;         // elements
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
  for (int o = TPR < 32 ? TPR / 2 : 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
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

// The lanes of this thread's row in its warp.
template <int TPR>
__device__ __forceinline__ unsigned row_lanes() {
  if constexpr (TPR >= 32) return 0xffffffffu;
  return ((1u << (TPR & 31)) - 1) << (threadIdx.x & 31 & ~(TPR - 1));
}

// Waits for the threads of a row; `group` numbers the rows of a block.
template <int TPR>
__device__ __forceinline__ void group_sync(int group) {
  if constexpr (TPR <= 32)
    __syncwarp(row_lanes<TPR>());
  else
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(group + 1), "n"(TPR) : "memory");
}

// m = mean(v^2) + eps of a row.  Below 2^-100 squares may have been lost (one that is
// keeps an error of 2^-150 at most, 2^-50 of such a mean); infinity says that the sum
// overflowed, unless v holds one.  NaN is in range: squares and their sum are NaN only
// if v holds one, and then so is the row by the formula.
__device__ __forceinline__ bool out_of_range(float m) {
  return m < 0x1p-100f || m > 3.402823466e38f;
}

// A row with such a mean square, of x or of h, once more, element by element from its
// inputs: v is multiplied by f = 2^96 or 2^-96 before it is squared, so that |f v| <= 2^32,
// or |f v| < 2^62 (a mean below 2^-100 leaves |v| < 2^-50 sqrt(cols)) with no number below
// 2^-53, and what counts fits.  v / rms is (v f) inv for small numbers and (v inv) f for
// large ones, so that neither step takes bits from a number that is small beside its row.
// Called by the TPR threads of the row, `t` of them, with `buf` for their warps' sums;
// writes after what they wrote before.
template <typename T, int TPR>
__device__ __forceinline__ void row_out_of_range(const Args<T>& a, int64_t row, int t, int group,
                                                 float* buf) {
  const int n = a.cols;
  const int64_t off = row * n;
  group_sync<TPR>(group);
  auto row_sum_of = [&](auto v_at, float f) {
    float s = 0.f;
#pragma unroll 1
    for (int c = t; c < n; c += TPR) {
      const float v = v_at(c) * f;
      s = fmaf(v, v, s);
    }
#pragma unroll
    for (int o = TPR < 32 ? TPR / 2 : 16; o > 0; o >>= 1) s += __shfl_xor_sync(row_lanes<TPR>(), s, o);
    if constexpr (TPR > 32) {
      group_sync<TPR>(group);  // all have read buf
      if ((t & 31) == 0) buf[t / 32] = s;
      group_sync<TPR>(group);
      s = 0.f;
#pragma unroll 1
      for (int k = 0; k < TPR / 32; ++k) s += buf[k];
    }
    return s;
  };
  struct TwoSteps {
    float first, second;
  };
  auto inverse = [&](auto v_at) {
    const float cols = static_cast<float>(a.cols);
    const float m = row_sum_of(v_at, 1.f) / cols + a.eps;
    const float f = !out_of_range(m) ? 1.f : m < 1.f ? 0x1p96f : 0x1p-96f;
    const float inv = rsqrtf(row_sum_of(v_at, f) / cols + a.eps * f * f);
    return m < 1.f ? TwoSteps{f, inv} : TwoSteps{inv, f};
  };
  const T* gate = static_cast<const T*>(a.gate.ptr);
  if (gate != nullptr) gate += row / a.gate.rows_per * a.gate.row_stride;
  auto x_at = [&](int c) { return Elem<T>::to_f(a.x[off + c]); };
  const TwoSteps by_x = inverse(x_at);
  auto h_at = [&](int c) {
    float v = x_at(c) * by_x.first * by_x.second * Elem<T>::to_f(a.post[c]);
    if (gate != nullptr) v *= Elem<T>::to_f(gate[a.gate.col_stride ? c : 0]);
    return fmaf(a.alpha, Elem<T>::to_f(a.residual[off + c]), v);
  };
  const TwoSteps by_h = inverse(h_at);
#pragma unroll 1
  for (int c = t; c < n; c += TPR) {
    const float h = h_at(c);
    a.h_out[off + c] = Elem<T>::from_f(h);
    a.out[off + c] = Elem<T>::from_f(h * by_h.first * by_h.second * Elem<T>::to_f(a.pre[c]));
  }
}

// The same out of line, for rows of a warp or less, of which there may be many at a time:
// inlined it costs their kernels registers, and with them blocks per SM (16384 x 256 bf16
// 7.3 us; inline 9.9).
template <typename T, int TPR>
__device__ __noinline__ void row_out_of_range_call(const Args<T>& a) {
  const int group = threadIdx.x / TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / TPR) + group;
  row_out_of_range<T, TPR>(a, row, threadIdx.x % TPR, group, nullptr);
}

// Elements [pos + lo, pos + hi) of `base` in their places of a vector, one by one.
template <typename T>
__device__ __forceinline__ uint4 gather(const T* base, int64_t pos, int lo, int hi) {
  constexpr int E = Elem<T>::kPerVec;
  float f[E];
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = e >= lo && e < hi ? Elem<T>::to_f(base[pos + e]) : 0.f;
  return Elem<T>::pack(f);
}

// Bits of a vector's elements [lo, hi).
template <typename T>
__device__ __forceinline__ uint4 element_mask(int lo, int hi) {
  constexpr int E = Elem<T>::kPerVec;
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (E == 4) {
      w[k] = k >= lo && k < hi ? 0xFFFFFFFFu : 0u;
    } else {
      w[k] = (2 * k >= lo && 2 * k < hi ? 0x0000FFFFu : 0u) |
             (2 * k + 1 >= lo && 2 * k + 1 < hi ? 0xFFFF0000u : 0u);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 operator&(const uint4& a, const uint4& b) {
  return make_uint4(a.x & b.x, a.y & b.y, a.z & b.z, a.w & b.w);
}

// Elements [shift, shift + E) of the vectors a and b.
template <typename T>
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int shift) {
  uint32_t r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const int words = shift * static_cast<int>(sizeof(T)) / 4;
#pragma unroll
  for (int i = 0; i < 6; ++i) r[i] = words & 2 ? r[i + 2] : r[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) r[i] = words & 1 ? r[i + 1] : r[i];
  if constexpr (sizeof(T) == 2) {
    const uint32_t bits = (shift & 1) * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __funnelshift_r(r[i], r[i + 1], bits);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Elements [pos, pos + E) of `base` [total], which starts on 16 bytes, for any
// pos > -E.  Only those in [lo, hi) are wanted; where a vector would reach behind
// the last element they are taken one by one.
template <typename T>
__device__ __forceinline__ uint4 load_shifted(const T* base, int64_t pos, int64_t total, int lo,
                                              int hi) {
  constexpr int E = Elem<T>::kPerVec;
  const int shift = static_cast<int>(pos & (E - 1));
  const int64_t q = (pos - shift) / E;
  if ((q + (shift ? 2 : 1)) * E > total) return gather(base, pos, lo, hi);
  const uint4* v = reinterpret_cast<const uint4*>(base) + q;
  uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
  if (q >= 0) a = ld_cached(v);
  if (shift) b = ld_cached(v + 1);
  return shifted<T>(a, b, shift);
}

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

// A weight [cols], which starts on 16 bytes, at the places of a row that starts at
// element `skip` of its first vector.  The weight's own last vector, if it is not
// whole, is gathered once.
template <typename T>
struct ShiftedWeight {
  static constexpr int E = Elem<T>::kPerVec;
  const T* w;
  int full, skip;
  uint4 tail;
  __device__ __forceinline__ ShiftedWeight(const T* weight, int cols, int skip_)
      : w(weight), full(cols / E), skip(skip_), tail(gather(weight, cols / E * E, 0, cols % E)) {}
  __device__ __forceinline__ uint4 vec(int v) const {
    if (v >= 0 && v < full) return ld_cached(reinterpret_cast<const uint4*>(w) + v);
    return v == full ? tail : make_uint4(0u, 0u, 0u, 0u);
  }
  // For vector j of the row: elements j E - skip on.
  __device__ __forceinline__ uint4 at(int j) const {
    return skip ? shifted<T>(vec(j - 1), vec(j), E - skip) : vec(j);
  }
};

constexpr int threads_for(int tpr) { return tpr > 256 ? tpr : 256; }

// Blocks per SM that rows of a warp or less are compiled for, one of which the registers
// of the call behind them would cost (65536 x 128 bf16 13.1 us; 16.9 with three blocks).
// Unaligned 16-bit rows of two vectors keep theirs, and lose if held to it (30000 x 99 fp16
// 11.3 -> 12.0).
template <typename T, bool kShift, int VPT, int TPR>
constexpr int blocks_for() {
  constexpr bool kWide = kShift && std::is_same_v<T, __nv_bfloat16>;
  if (TPR > 32) return 1;
  if (VPT == 1) return kWide ? 4 : 5;
  return kShift && sizeof(T) == 2 ? 1 : 4;
}

// kShift: rows need not start on 16 bytes (the tensors do).  A thread's vectors
// are those of the tensors, so the row's first and last may hold elements of its
// neighbours, which count as zeros and are not written; the weights' elements are
// shifted into the places of the row's.
template <typename T, bool kShift, int VPT, int TPR>
__global__ void __launch_bounds__(threads_for(TPR), blocks_for<T, kShift, VPT, TPR>())
    sandwich_kernel(const __grid_constant__ Args<T> a) {
  constexpr int E = Elem<T>::kPerVec;
  constexpr int P = E / 2;  // pairs per vector
  constexpr int kThreads = threads_for(TPR);
  constexpr int RPB = kThreads / TPR;
  // With 1024 threads the registers hold the row, but not its weights too.
  constexpr bool kEarly = TPR < 1024;
  // Nor do those that leave room for three to five blocks per SM: there the second weight
  // of 16-bit rows comes before the second sum (16384 x 256 bf16 7.3 us, 65536 x 128 13.1;
  // 9.9 and 16.6 with spills).
  constexpr bool kPreLate = TPR <= 32 && sizeof(T) == 2;
  __shared__ float buf[2][kThreads / 32];
  const int t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR;
  const bool live = row < a.rows;
  const int64_t off = (live ? row : 0) * static_cast<int64_t>(a.cols);
  const int64_t total = a.rows * static_cast<int64_t>(a.cols);
  const int skip = kShift ? static_cast<int>(off & (E - 1)) : 0;
  const int nv = live ? (skip + a.cols + E - 1) / E : 0;
  const T* gate = static_cast<const T*>(a.gate.ptr);
  const bool gate_cols = gate != nullptr && a.gate.col_stride;

  sm100::pdl_launch_dependents();
  sm100::pdl_wait_prior();
  const int64_t gate_at =
      live && gate != nullptr ? row / a.gate.rows_per * a.gate.row_stride : 0;
  const float g_row = gate != nullptr && !gate_cols ? Elem<T>::to_f(gate[gate_at]) : 1.f;

  auto column = [&](int i) { return (t + i * TPR) * E - skip; };  // of element 0
  auto used = [&](int i) { return t + i * TPR < nv; };
  auto first = [&](int c) { return kShift && c < 0 ? -c : 0; };
  auto last = [&](int c) { return kShift && a.cols - c < E ? a.cols - c : E; };
  auto row_vec = [&](const T* p, int c) {
    int64_t at = off + c;
    if constexpr (kShift) {
      if (total < E) return make_uint4(0u, 0u, 0u, 0u);
      at = min(at, (total & ~static_cast<int64_t>(E - 1)) - E);
    }
    return ld_stream(reinterpret_cast<const uint4*>(p + at));
  };
  auto gate_vec = [&](int c) {
    if constexpr (kShift) return load_shifted(gate, gate_at + c, a.gate.total, first(c), last(c));
    return ld_cached(reinterpret_cast<const uint4*>(gate + gate_at + c));
  };
  auto write = [&](T* p, int c, const float2* f) {
    const uint4 v = Elem<T>::pack(&f[0].x);
    const int lo = first(c), hi = last(c);
    if (!kShift || (lo == 0 && hi == E)) {
      st_stream(reinterpret_cast<uint4*>(p + off + c), v);
    } else {
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (k >= lo && k < hi) p[off + c + k] = e[k];
    }
  };
  auto mask = [&](int c, float2* f) {  // zeros where the row is not
    if constexpr (kShift) {
      const int lo = first(c), hi = last(c);
      if (lo > 0 || hi < E) {
#pragma unroll
        for (int k = 0; k < P; ++k) {
          if (2 * k < lo || 2 * k >= hi) f[k].x = 0.f;
          if (2 * k + 1 < lo || 2 * k + 1 >= hi) f[k].y = 0.f;
        }
      }
    }
  };

  uint4 x[VPT], res[VPT], post[VPT], pre[VPT], g[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (used(i)) {
      x[i] = row_vec(a.x, column(i));
      res[i] = row_vec(a.residual, column(i));
    }
  }
  // The tensor's last elements, if they lie behind its last whole vector (not where the
  // row is loaded: behind a branch each vector there waits for its own load, 61 x 2047
  // bf16 4.4 -> 5.3 us with four vectors per thread).
  auto load_rest = [&]() {
    if constexpr (kShift) {
      if (off + a.cols > (total & ~static_cast<int64_t>(E - 1))) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int c = column(i);
          if (used(i) && off + c + E > total) {
            x[i] = gather(a.x, off + c, first(c), last(c));
            res[i] = gather(a.residual, off + c, first(c), last(c));
          }
        }
      }
    }
  };
  const ShiftedWeight<T> post_w(a.post, a.cols, skip), pre_w(a.pre, a.cols, skip);
  auto weight_vec = [&](const ShiftedWeight<T>& w, int i) {
    if constexpr (kShift) return w.at(t + i * TPR);
    return ld_cached(reinterpret_cast<const uint4*>(w.w) + t + i * TPR);
  };
  auto load_post = [&](int i) {
    post[i] = weight_vec(post_w, i);
    if (gate_cols) g[i] = gate_vec(column(i));
  };
  auto load_pre = [&](int i) { pre[i] = weight_vec(pre_w, i); };
  if constexpr (kEarly) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (used(i)) {
        load_post(i);
        if constexpr (!kPreLate) load_pre(i);
      }
    }
  }

  load_rest();
  float2 h[VPT][P];  // x, then h
  float2 ss = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (used(i)) {
      Elem<T>::unpack(x[i], &h[i][0].x);
      mask(column(i), h[i]);
#pragma unroll
      for (int e = 0; e < P; ++e) ss = fma2(h[i][e], h[i][e], ss);
    }
  }
  const float sum = row_sum<TPR>(ss.x + ss.y, buf[0]);
  const float mean = sum / static_cast<float>(a.cols) + a.eps;
  const float inv = rsqrtf(mean);
  bool again = live && out_of_range(mean);

  ss = make_float2(0.f, 0.f);
  const float scale = inv * g_row;
  const float2 scale2 = make_float2(scale, scale), alpha2 = make_float2(a.alpha, a.alpha);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (used(i)) {
      if constexpr (!kEarly) load_post(i);
      float2 w[P];
      Elem<T>::unpack(post[i], &w[0].x);
#pragma unroll
      for (int e = 0; e < P; ++e) h[i][e] = mul2(mul2(h[i][e], scale2), w[e]);
      if (gate_cols) {
        Elem<T>::unpack(g[i], &w[0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) h[i][e] = mul2(h[i][e], w[e]);
      }
      Elem<T>::unpack(res[i], &w[0].x);
#pragma unroll
      for (int e = 0; e < P; ++e) h[i][e] = fma2(alpha2, w[e], h[i][e]);
      mask(column(i), h[i]);
#pragma unroll
      for (int e = 0; e < P; ++e) ss = fma2(h[i][e], h[i][e], ss);
      write(a.h_out, column(i), h[i]);
    }
  }
  if constexpr (kPreLate) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (used(i)) load_pre(i);
  }
  const float sum_h = row_sum<TPR>(ss.x + ss.y, buf[1]);
  const float mean_h = sum_h / static_cast<float>(a.cols) + a.eps;
  const float inv_h = rsqrtf(mean_h);
  again |= live && out_of_range(mean_h);
  const float2 inv_h2 = make_float2(inv_h, inv_h);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (used(i)) {
      if constexpr (!kEarly) load_pre(i);
      float2 w[P];
      Elem<T>::unpack(pre[i], &w[0].x);
#pragma unroll
      for (int e = 0; e < P; ++e) w[e] = mul2(mul2(h[i][e], inv_h2), w[e]);
      write(a.out, column(i), w);
    }
  }
  // The row's threads have the same sums.
  if (again) {
    const int group = threadIdx.x / TPR;
    if constexpr (TPR <= 32)
      row_out_of_range_call<T, TPR>(a);
    else
      row_out_of_range<T, TPR>(a, row, t, group, buf[0] + group * (TPR / 32));
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
constexpr int64_t kRingMinRow = 1024, kRingMinTotal = 1 << 20;  // bytes
// Vectors of a row: as many as two stages hold, or as a thread holds with its weights.
template <bool kShift>
constexpr int64_t kRingMaxVectors = (kShift ? 4 : 6) * kRingThreads;

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

// kShift: rows need not start on 16 bytes (the tensors do).  The copies take the
// vectors around a row, a thread works on those, and the row's first and last are
// written element by element.  The grid makes a group's rows `step` apart with step
// a multiple of E, so they all start at the same element of a vector, and weights
// shifted to it once stay in registers like those of aligned rows.
template <typename T, bool kShift, int VPT, int TPR>
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
  __shared__ __align__(16) uint4 ends[kShift ? G : 1][2][2];  // [h, out][first, last vector]
  __shared__ int abort_flag;
  const int group = threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  const int64_t step = static_cast<int64_t>(gridDim.x) * G;
  const int64_t first_row = static_cast<int64_t>(blockIdx.x) * G + group;
  const int64_t total = a.rows * static_cast<int64_t>(a.cols);
  uint8_t* mine = ring + static_cast<int64_t>(group) * stages * 2 * pitch;
  const uint32_t bar0 = smem_addr(bars[group]);
  const T* gate = static_cast<const T*>(a.gate.ptr);
  const bool gate_cols = gate != nullptr && a.gate.col_stride;
  // Of every row of this group (step is a multiple of E).
  const int skip = kShift ? static_cast<int>(first_row * a.cols & (E - 1)) : 0;
  const int nv = (skip + a.cols + E - 1) / E;
  auto column = [&](int i) { return (t + i * TPR) * E - skip; };  // of element 0
  auto used = [&](int i) { return t + i * TPR < nv; };
  const int last_i = (nv - 1) / TPR;
  uint4 head, foot;  // of the thread's vectors 0 and last_i
  bool head_cut = false, foot_cut = false;
  T* end_to = nullptr;
  const T* end_from = nullptr;
  if constexpr (kShift) {
    const int c = column(0), d = column(last_i);
    head = element_mask<T>(c < 0 ? -c : 0, E);
    foot = element_mask<T>(0, a.cols - d < E ? a.cols - d : E);
    head_cut = c < 0;
    foot_cut = d < a.cols && d + E > a.cols;
    // One thread per element of the shared vectors: [h, out][first, last][element].
    const int which = t / (2 * E), end = t / E % 2, e = t % E;
    const int at = (end ? nv - 1 : 0) * E - skip + e;
    if (t < 4 * E && at >= 0 && at < a.cols && (end ? (nv * E - skip) > a.cols : skip > 0)) {
      end_to = (which ? a.out : a.h_out) + at;
      end_from = reinterpret_cast<const T*>(&ends[kShift ? group : 0][which][end]) + e;
    }
  }

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int g = 0; g < G; ++g)
      for (int k = 0; k < kMaxStages; ++k) mbar_init(smem_addr(&bars[g][k]), 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  // The row's vectors: from the one that its first element is in to the one that
  // its last is in, or the tensor's last whole one.
  auto row_bytes = [&](int64_t row) {
    uint32_t vectors = static_cast<uint32_t>(a.cols / E);
    if constexpr (kShift) {
      int64_t v1 = (row + 1) * a.cols / E;
      if (v1 * E < (row + 1) * a.cols && (v1 + 1) * E <= total) ++v1;
      vectors = static_cast<uint32_t>(v1 - row * a.cols / E);
    }
    return vectors * 16u;
  };
  // The residual is older than the previous kernel's output, as a rule: its first rows
  // are asked for in L2 before that kernel is done (1024 x 4096 bf16 9.8 -> 8.5 us,
  // 8192 x 4096 45.5 -> 43.1, 1001 x 2047 8.5 -> 8.1 in graph replays).
  if (t == 0)
    for (int k = 0; k < stages && first_row + k * step < a.rows; ++k) {
      const int64_t row = first_row + k * step;
      bulk_prefetch(a.residual + row * a.cols / E * E, row_bytes(row));
    }
  __syncthreads();
  pdl_wait_prior();

  auto request = [&](int64_t row, int stage) {  // one thread
    const int64_t at = row * a.cols / E * E;
    const uint32_t bytes = row_bytes(row);
    const uint32_t bar = bar0 + 8u * stage;
    const uint32_t dst = smem_addr(mine + static_cast<int64_t>(stage) * 2 * pitch);
    mbar_arrive_expect_tx(bar, 2 * bytes);
    bulk_load(dst, a.x + at, bytes, bar);
    bulk_load(dst + pitch, a.residual + at, bytes, bar);
  };
  if (t == 0)
    for (int k = 0; k < stages && first_row + k * step < a.rows; ++k)
      request(first_row + k * step, k);

  // A thread's columns are the same in every row, so their weights stay in
  // registers (from L2 they would be as many bytes per row as x and the residual),
  // and so does the gate until its row changes.  Weights of more than four vectors do
  // not fit there and are read again for every row, ahead of the sum before their use,
  // which is still better than a row at a time in the registers of 1024 threads
  // (1024 x 20480 bf16 56 -> 28 us).
  constexpr bool kKeep = VPT <= 4;
  static_assert(kKeep || !kShift, "shifted once");
  uint4 post[kKeep ? VPT : 1], pre[kKeep ? VPT : 1], g[VPT], reread[kKeep ? 1 : VPT];
  auto weight = [&](const uint4* kept, int i) { return kKeep ? kept[i] : reread[kKeep ? 0 : i]; };
  auto read_weight = [&](const T* w) {
    if constexpr (!kKeep) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (used(i)) reread[i] = ld_cached(reinterpret_cast<const uint4*>(w) + t + i * TPR);
    }
  };
  float g_row = 1.f;
  int64_t g_at = 0, g_end = 0;  // the gate row in use, the first row beyond it
  if constexpr (kKeep) {
    const ShiftedWeight<T> post_w(a.post, a.cols, skip), pre_w(a.pre, a.cols, skip);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = t + i * TPR;
      if (j < nv) {
        post[i] = kShift ? post_w.at(j) : ld_cached(reinterpret_cast<const uint4*>(a.post) + j);
        pre[i] = kShift ? pre_w.at(j) : ld_cached(reinterpret_cast<const uint4*>(a.pre) + j);
      }
    }
  }

  // Rows out of range are written as NaN, and again once the group has no more rows to
  // stream: what that needs is not held meanwhile.
  bool again = false;
  auto inverse = [&](float sum) {
    const float mean = sum / static_cast<float>(a.cols) + a.eps;
    const bool out = out_of_range(mean);
    again |= out;
    return out ? __int_as_float(0x7fc00000) : rsqrtf(mean);
  };
  int stage = 0;
  uint32_t phase = 0;
  for (int64_t row = first_row; row < a.rows; row += step) {
    const int64_t off = row * a.cols;
    // Zeros where a vector is not the row's; only the first and the last are shared.
    auto own = [&](const uint4& v, int i) {
      if constexpr (kShift) {
        if (i == 0 && last_i == 0) return v & head & foot;
        if (i == 0) return v & head;
        if (i == last_i) return v & foot;
      }
      return v;
    };
    // A whole vector goes to its place, one that the row shares to `ends`.
    auto write = [&](T* p, int which, int i, const float2* f) {
      const uint4 v = Elem<T>::pack(&f[0].x);
      if (kShift && i == 0 && head_cut)
        ends[kShift ? group : 0][which][0] = v;
      else if (kShift && i == last_i && foot_cut)
        ends[kShift ? group : 0][which][1] = v;
      else
        st_stream(reinterpret_cast<uint4*>(p + off + column(i)), v);
    };
    if (gate != nullptr && row >= g_end) {  // the next gate row (a division only here)
      g_at = row / a.gate.rows_per;
      g_end = (g_at + 1) * a.gate.rows_per;
      const int64_t at = g_at * a.gate.row_stride;
      if (gate_cols) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
          if (used(i)) {
            const int c = column(i);
            if constexpr (kShift) {
              const int left = a.cols - c;
              g[i] = own(load_shifted(gate, at + c, a.gate.total, c < 0 ? -c : 0, left < E ? left : E), i);
            } else {
              g[i] = ld_cached(reinterpret_cast<const uint4*>(gate + at + c));
            }
          }
      } else {
        g_row = Elem<T>::to_f(gate[at]);
      }
    }
    const uint4* xs = reinterpret_cast<const uint4*>(mine + static_cast<int64_t>(stage) * 2 * pitch);
    const uint4* rs = reinterpret_cast<const uint4*>(mine + (static_cast<int64_t>(stage) * 2 + 1) * pitch);
    bool bad = !mbar_wait_bounded(bar0 + 8u * stage, phase, &abort_flag, &g_norm_watchdog, kWdRow);
    if constexpr (kShift) {
      // The tensor's last elements, if they lie behind its last whole vector.
      const int rest = static_cast<int>(total & (E - 1));
      if (rest > 0 && off + a.cols == total) {
        if (t < rest) {
          uint8_t* at = mine + static_cast<int64_t>(stage) * 2 * pitch + ((nv - 1) * E + t) * sizeof(T);
          *reinterpret_cast<T*>(at) = a.x[total - rest + t];
          *reinterpret_cast<T*>(at + pitch) = a.residual[total - rest + t];
        }
        group_sync<TPR>(group);
      }
    }

    float2 h[VPT][P];  // x, then h
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (used(i)) {
        Elem<T>::unpack(own(xs[t + i * TPR], i), &h[i][0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) ss = fma2(h[i][e], h[i][e], ss);
      }
    }
    read_weight(a.post);
    const float sum = group_sum<TPR>(ss.x + ss.y, partial[group][0], group, t, bad);
    if (bad) {  // the whole group, once what it has requested has arrived
      for (int k = 0; t == 0 && k < stages && row + k * step < a.rows; ++k) {
        const bool wraps = stage + k >= stages;
        mbar_drain(bar0 + 8u * (stage + k - (wraps ? stages : 0)), phase ^ (wraps ? 1u : 0u));
      }
      return;
    }
    const float inv = inverse(sum);

    ss = make_float2(0.f, 0.f);
    const float scale = gate_cols ? inv : inv * g_row;
    const float2 scale2 = make_float2(scale, scale), alpha2 = make_float2(a.alpha, a.alpha);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (used(i)) {
        float2 w[P];
        Elem<T>::unpack(weight(post, i), &w[0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) h[i][e] = mul2(mul2(h[i][e], scale2), w[e]);
        if (gate_cols) {
          Elem<T>::unpack(g[i], &w[0].x);
#pragma unroll
          for (int e = 0; e < P; ++e) h[i][e] = mul2(h[i][e], w[e]);
        }
        Elem<T>::unpack(own(rs[t + i * TPR], i), &w[0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          h[i][e] = fma2(alpha2, w[e], h[i][e]);
          ss = fma2(h[i][e], h[i][e], ss);
        }
        write(a.h_out, 0, i, h[i]);
      }
    }
    read_weight(a.pre);
    const float sum_h = group_sum<TPR>(ss.x + ss.y, partial[group][1], group, t, bad);
    // The whole group has read the stage.
    if (t == 0 && row + stages * step < a.rows) request(row + stages * step, stage);
    const float inv_h = inverse(sum_h);
    const float2 inv_h2 = make_float2(inv_h, inv_h);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (used(i)) {
        float2 w[P];
        Elem<T>::unpack(weight(pre, i), &w[0].x);
#pragma unroll
        for (int e = 0; e < P; ++e) w[e] = mul2(mul2(h[i][e], inv_h2), w[e]);
        write(a.out, 1, i, w);
      }
    }
    if constexpr (kShift) {
      // One lane per element of the first and the last vector, if they are shared.
      group_sync<TPR>(group);
      if (end_to != nullptr) end_to[off] = *end_from;
      group_sync<TPR>(group);
    }
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  if (again) {  // the whole group: its threads have the same sums
    group_sync<TPR>(group);
    for (int64_t row = first_row; row < a.rows; row += step) {
      const T* first = a.out + row * a.cols;
      if (isnan(Elem<T>::to_f(*first)))  // what the group wrote, or NaN by the formula
        row_out_of_range<T, TPR>(a, row, t, group, partial[group][0]);
    }
  }
}

// Any row length and alignment: one block per row; h is computed again from its
// inputs for the output pass, so that it is never rounded in between.
constexpr int kLongThreads = 1024;

template <typename T, int E>
__global__ void __launch_bounds__(kLongThreads) sandwich_long_kernel(const Args<T> a) {
  __shared__ float buf[2][kLongThreads / 32];
  const int64_t row = blockIdx.x;
  const int64_t off = row * a.cols;
  sm100::pdl_launch_dependents();
  sm100::pdl_wait_prior();
  auto load = [](const T* p, float* f) {
    if constexpr (E == 1)
      f[0] = Elem<T>::to_f(*p);
    else
      Elem<T>::unpack(ld_cached(reinterpret_cast<const uint4*>(p)), f);
  };
  auto store = [](T* p, const float* f) {
    if constexpr (E == 1)
      *p = Elem<T>::from_f(f[0]);
    else
      st_stream(reinterpret_cast<uint4*>(p), Elem<T>::pack(f));
  };
  const int step = kLongThreads * E;
  float ss = 0.f;
  for (int64_t c = threadIdx.x * E; c < a.cols; c += step) {
    float f[E];
    load(a.x + off + c, f);
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(f[e], f[e], ss);
  }
  ss = row_sum<kLongThreads>(ss, buf[0]);
  const float mean = ss / static_cast<float>(a.cols) + a.eps;
  const float inv = rsqrtf(mean);
  const T* gate = static_cast<const T*>(a.gate.ptr);
  if (gate != nullptr) gate += row / a.gate.rows_per * a.gate.row_stride;
  const bool gate_cols = gate != nullptr && a.gate.col_stride;
  const float scale = gate != nullptr && !gate_cols ? inv * Elem<T>::to_f(*gate) : inv;
  auto h_at = [&](int64_t c, float* h) {
    float w[E];
    load(a.x + off + c, h);
    load(a.post + c, w);
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = h[e] * scale * w[e];
    if (gate_cols) {
      load(gate + c, w);
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] *= w[e];
    }
    load(a.residual + off + c, w);
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = fmaf(a.alpha, w[e], h[e]);
  };
  ss = 0.f;
  for (int64_t c = threadIdx.x * E; c < a.cols; c += step) {
    float h[E];
    h_at(c, h);
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(h[e], h[e], ss);
  }
  ss = row_sum<kLongThreads>(ss, buf[1]);
  const float mean_h = ss / static_cast<float>(a.cols) + a.eps;
  if (out_of_range(mean) || out_of_range(mean_h)) {
    row_out_of_range<T, kLongThreads>(a, row, threadIdx.x, 0, buf[0]);
    return;
  }
  const float inv_h = rsqrtf(mean_h);
  for (int64_t c = threadIdx.x * E; c < a.cols; c += step) {
    float h[E], w[E];
    h_at(c, h);
    store(a.h_out + off + c, h);
    load(a.pre + c, w);
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] *= h[e] * inv_h;
    store(a.out + off + c, w);
  }
}

template <typename T>
int launch_kernel(void (*kernel)(const Args<T>), const Args<T>& a, int64_t blocks, int threads,
                  cudaStream_t s) {
  if (blocks > 0x7fffffffLL)
    return fail(AOTK_ERR_INVALID_ARGUMENT, "aotk_sandwich_rmsnorm: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess)
    return fail(AOTK_ERR_CUDA, "aotk_sandwich_rmsnorm launch: %s", cudaGetErrorString(e));
  return check_launch("aotk_sandwich_rmsnorm");
}

template <typename T, bool kShift, int VPT, int TPR>
int launch_rows(const Args<T>& a, cudaStream_t s) {
  constexpr int kThreads = threads_for(TPR);
  const int64_t blocks = (a.rows + kThreads / TPR - 1) / (kThreads / TPR);
  return launch_kernel<T>(sandwich_kernel<T, kShift, VPT, TPR>, a, blocks, kThreads, s);
}

template <typename T, int E>
int launch_long(const Args<T>& a, cudaStream_t s) {
  return launch_kernel<T>(sandwich_long_kernel<T, E>, a, a.rows, kLongThreads, s);
}

// The smallest group of threads that holds a row in at most two vectors each: with
// four there was more to do behind every wait (16 x 4096 bf16 2.7 -> 2.1 us, 100 x 2048
// 2.8 -> 2.1, 61 x 2047 4.6 -> 3.4, 16384 x 256 7.9 -> 6.9).  Rows of 8 to 16 vectors
// stay with 8 threads, which many rows want (32768 x 128 6.6 us, 16 threads 7.5).  Of
// the longest, 16-bit rows take 1024 threads (1 x 16384 8.6 -> 4.1) and fp32 rows
// 512 with four vectors (1 x 8192 3.2, 3.8 with 1024).
template <typename T, bool kShift>
int dispatch_rows(const Args<T>& a, cudaStream_t s) {
  constexpr int E = Elem<T>::kPerVec;
  const int64_t n = (static_cast<int64_t>(a.cols) + (kShift ? 2 * (E - 1) : 0)) / E;  // at most
  if (n <= 8) return launch_rows<T, kShift, 1, 8>(a, s);
  if (n <= 16) return launch_rows<T, kShift, 2, 8>(a, s);
  if (n <= 32) return launch_rows<T, kShift, 2, 16>(a, s);
  if (n <= 64) return launch_rows<T, kShift, 2, 32>(a, s);
  if (n <= 128) return launch_rows<T, kShift, 2, 64>(a, s);
  if (n <= 256) return launch_rows<T, kShift, 2, 128>(a, s);
  if (n <= 512) return launch_rows<T, kShift, 2, 256>(a, s);
  if (n <= 1024) return launch_rows<T, kShift, 2, 512>(a, s);
  if constexpr (sizeof(T) == 2) {
    if (n <= 2048) return launch_rows<T, kShift, 2, 1024>(a, s);
  } else {
    if (n <= 2048) return launch_rows<T, kShift, 4, 512>(a, s);
  }
  if (n <= 4096) return launch_rows<T, kShift, 4, 1024>(a, s);
  return kShift ? launch_long<T, 1>(a, s) : launch_long<T, E>(a, s);
}

template <typename T, bool kShift, int VPT, int TPR>
int launch_ring(const Args<T>& a, cudaStream_t s, const DeviceInfo& info) {
  constexpr int G = kRingThreads / TPR;
  constexpr int E = Elem<T>::kPerVec;
  const int pitch = ((a.cols + E - 1) / E + (kShift ? 1 : 0)) * 16;
  int stages = kRingBytes / (G * 2 * pitch);
  if (stages > kMaxStages) stages = kMaxStages;
  auto kernel = sandwich_ring_kernel<T, kShift, VPT, TPR>;
  if (int st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), kRingBytes, info)) return st;
  int64_t blocks = (a.rows + G - 1) / G;
  if (blocks > info.sm_count) {
    // Groups that take several rows: blocks x G, the rows between them, a multiple of E.
    constexpr int unit = E > G ? E / G : 1;
    blocks = kShift ? info.sm_count / unit * unit : info.sm_count;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
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

// The smallest group that holds a row in few vectors per thread: four of fp32, three
// of 16-bit types, whose four would not fit the registers beside their weights
// (20000 x 1001 bf16 45.0 -> 33.9 us, 8192 x 4096 48.0 -> 45.1; fp32 8192 x 4096 is
// 89.5 with four and 95.2 with two).  Three of unaligned fp16 rows spill 36 to 44 bytes
// all the same, and run as fast as those of bf16, which do not (20000 x 1001 30.6 us;
// 32.6).
template <typename T, bool kShift, int TPR>
int dispatch_group(const Args<T>& a, int n, cudaStream_t s, const DeviceInfo& info) {
  if (n <= 2 * TPR) return launch_ring<T, kShift, 2, TPR>(a, s, info);
  if (n <= 3 * TPR) return launch_ring<T, kShift, 3, TPR>(a, s, info);
  if constexpr (sizeof(T) == 4 || TPR == kRingThreads)
    if (n <= 4 * TPR) return launch_ring<T, kShift, 4, TPR>(a, s, info);
  if constexpr (TPR == kRingThreads && !kShift)
    if (n <= 6 * TPR) return launch_ring<T, kShift, 6, TPR>(a, s, info);
  if constexpr (TPR < kRingThreads) return dispatch_group<T, kShift, TPR * 2>(a, n, s, info);
  return fail(AOTK_ERR_UNSUPPORTED, "aotk_sandwich_rmsnorm: row of %d vectors", n);
}

template <typename T, bool kShift>
int dispatch_ring(const Args<T>& a, cudaStream_t s, const DeviceInfo& info) {
  constexpr int E = Elem<T>::kPerVec;
  const int n = (a.cols + (kShift ? 2 * (E - 1) : 0)) / E;  // at most
  return dispatch_group<T, kShift, 32>(a, n, s, info);
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
  if (!(aligned16(x) && aligned16(residual) && aligned16(post) && aligned16(pre) &&
        aligned16(out) && aligned16(h_out) && aligned16(gate.ptr)))
    return launch_long<T, 1>(a, s);
  DeviceInfo info;
  if (int st = current_device_info(&info)) return st;
  const bool shift = cols % E != 0;
  const int64_t row_bytes = cols * static_cast<int64_t>(sizeof(T));
  const int64_t vectors = (cols + (shift ? 2 * (E - 1) : 0)) / E;
  const int64_t most = shift ? kRingMaxVectors<true> : kRingMaxVectors<false>;
  if (row_bytes >= kRingMinRow && vectors <= most && rows * row_bytes >= kRingMinTotal)
    return shift ? dispatch_ring<T, true>(a, s, info) : dispatch_ring<T, false>(a, s, info);
  return shift ? dispatch_rows<T, true>(a, s) : dispatch_rows<T, false>(a, s);
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
  Gate g = {nullptr, 1, 0, 0, 0};
  if (gate) {
    if (gate_rows < 1 || rows % gate_rows != 0 || (gate_cols != cols && gate_cols != 1))
      return fail(AOTK_ERR_INVALID_ARGUMENT,
                  "%s: gate [%lld, %lld] does not fit rows [%lld, %lld]", who, (long long)gate_rows,
                  (long long)gate_cols, (long long)rows, (long long)cols);
    g = {gate, rows / gate_rows, gate_cols, gate_rows * gate_cols, gate_cols == cols ? 1 : 0};
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
