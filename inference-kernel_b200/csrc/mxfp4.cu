// Microscaled 4-bit floating point (MX: blocks of 32 along the row share a
// power-of-two scale byte, elements are e2m1): quantisation and reading back.
//
//   e = floor(log2(max |x| over the block)),  S = 2^clamp(e - 2, -127, 127)
//   q = x / S rounded to the nearest of {0, .5, 1, 1.5, 2, 3, 4, 6}, ties to the
//       even code, larger magnitudes to 6;   value read back = q * S
//
// 2^(e-2) puts the block's largest magnitude into [4, 8), the top binade of
// e2m1.  The scale byte is the exponent field of max |x| less 2 (0 stands for
// 2^-127), so no logarithm is taken and x / S is an exact multiplication by a
// power of two: the one rounding is that to e2m1.  A block that holds a NaN or
// an infinity has no such scale: its byte is 255 (NaN), its codes are 0, and
// all 32 values read back as NaN.
//
// Layout: codes [rows, cols / 2], the even column in the low nibble; scales in
// tiles of 128 rows x 4 blocks, [ceil(rows/128)][ceil(cols/128)][512], byte
// (r % 32) * 16 + (r % 128 / 32) * 4 + block % 4 of its tile - the order in
// which the tensor cores' scale loads take them.  Bytes of a tile that belong
// to no row or block are written as 0.
//
// Both kernels stream HBM, and what has to be kept down for that is the
// arithmetic per element.  In the quantiser a lane owns a whole block of 32
// elements, so that the index arithmetic, the maximum and the scale are paid once
// per block and no lane waits for another, apart from two shuffles that make one
// 4-byte word of the scales of four neighbours.  (With four lanes to a block it
// issued 132 instructions per 8 elements and ran at 0.58 of the copy rate.)  A
// lane's 64 or 128 bytes are read as 32-byte accesses, whole sectors each, or, where
// rows do not start on 32 bytes, as the vectors around the block, shifted (4096 x 8192
// bf16 14.2 -> 16.1 us).  Reading back, a lane's item is 32 bytes of output.
#include <type_traits>

#include "common.h"
#include "mxfp4.cuh"
#include "sm100.cuh"
#include "vec.cuh"

namespace aotk {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = kThreads;  // blocks of 32 per thread block and step

// Item t of the padded problem is item t % items_k of row t / items_k; a thread's
// items are kLanes apart.
struct Walk {
  int items_k;
  int step_rows, step_items;  // kLanes / items_k and the remainder
};

// This thread's first item: one division by a uniform value and one of small
// numbers, and none from item to item.
template <int U>
__device__ __forceinline__ void first_item(const Walk& w, int64_t& row, int& kb) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kLanes * U);
  const int64_t row0 = t / w.items_k;
  const unsigned in_row = static_cast<unsigned>(t - row0 * w.items_k) + threadIdx.x;
  const unsigned more = in_row / static_cast<unsigned>(w.items_k);
  row = row0 + more;
  kb = static_cast<int>(in_row - more * w.items_k);
}

__device__ __forceinline__ void next_item(const Walk& w, int64_t& row, int& kb) {
  row += w.step_rows;
  kb += w.step_items;
  if (kb >= w.items_k) {
    kb -= w.items_k;
    ++row;
  }
}

// Offset of the scale byte of block kb of a row.
__device__ __forceinline__ int64_t scale_byte(int64_t row, int kb, int blocks_k) {
  const int r = static_cast<int>(row & 127);
  return ((row >> 7) * (blocks_k >> 2) + (kb >> 2)) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (kb & 3);
}

// The larger magnitude of each pair, NaN if either is; the sign is of no use.
template <typename T>
__device__ __forceinline__ uint32_t max_abs(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (sizeof(T) == 4)
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else if constexpr (std::is_same_v<T, __half>)
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// One block of 32 elements in registers.
template <typename T>
struct Block {
  static constexpr int kWords = 8 * sizeof(T);  // 32-bit words
  uint32_t w[kWords];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // p aligned to 32 bytes
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; i += 8) {
      uint4 a, b;
      ld_stream32(reinterpret_cast<const uint32_t*>(p) + i, a, b);
      w[i] = a.x, w[i + 1] = a.y, w[i + 2] = a.z, w[i + 3] = a.w;
      w[i + 4] = b.x, w[i + 5] = b.y, w[i + 6] = b.z, w[i + 7] = b.w;
    }
  }
  // Any p: the aligned 16-byte vectors around the block, through L1 since
  // neighbours share them, shifted into place - or, where such a vector would
  // reach out of [begin, end), element by element.
  __device__ __forceinline__ void load_any(const T* p, const T* begin, const T* end) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uintptr_t lo = at & ~static_cast<uintptr_t>(15);
    const uintptr_t hi = lo + (kWords * 4 + 16);
    if (lo >= reinterpret_cast<uintptr_t>(begin) && hi <= reinterpret_cast<uintptr_t>(end)) {
      const uint4* v = reinterpret_cast<const uint4*>(lo);
      uint32_t r[kWords + 4];
#pragma unroll
      for (int i = 0; i < kWords / 4 + 1; ++i) {
        const uint4 q = ld_cached(v + i);
        r[4 * i] = q.x, r[4 * i + 1] = q.y, r[4 * i + 2] = q.z, r[4 * i + 3] = q.w;
      }
      const bool two = at & 8, one = at & 4;
#pragma unroll
      for (int i = 0; i < kWords + 2; ++i) r[i] = two ? r[i + 2] : r[i];
#pragma unroll
      for (int i = 0; i < kWords + 1; ++i) r[i] = one ? r[i + 1] : r[i];
      const uint32_t bits = (at & 3) * 8;
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(r[i], r[i + 1], bits);
    } else {
      T e[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) e[i] = p[i];
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (sizeof(T) == 4)
          w[i] = __float_as_uint(e[i]);
        else
          w[i] = Elem<T>::pack2(Elem<T>::to_f(e[2 * i]), Elem<T>::to_f(e[2 * i + 1]));
      }
    }
  }
  // Exponent field of the largest magnitude as fp32: 255 for a NaN or an infinity.
  __device__ __forceinline__ uint32_t top_exponent() const {
    uint32_t m = w[0];
#pragma unroll
    for (int i = 1; i < kWords; ++i) m = max_abs<T>(m, w[i]);
    if constexpr (sizeof(T) == 4) {
      return (m >> 23) & 255u;
    } else {
      m = max_abs<T>(m, m >> 16 | m << 16);
      const uint16_t h = static_cast<uint16_t>(m);
      return (__float_as_uint(Elem<T>::to_f(*reinterpret_cast<const T*>(&h))) >> 23) & 255u;
    }
  }
  // Elements [8 i, 8 i + 8)
  __device__ __forceinline__ void get8(int i, float* f) const {
    constexpr int n = 2 * sizeof(T);
#pragma unroll
    for (int j = 0; j < n; ++j) {
      if constexpr (sizeof(T) == 4) {
        f[j] = __uint_as_float(w[n * i + j]);
      } else {
        const float2 t = Elem<T>::unpack2(w[n * i + j]);
        f[2 * j] = t.x;
        f[2 * j + 1] = t.y;
      }
    }
  }
};

// One block per thread: the next ones come with the SM's other thread blocks, and a
// problem of few waves ends evenly (two per thread, 16-bit types: 1024 x 4096 3.7 ->
// 4.8 us, 4096 x 8192 14.1 -> 14.7, 1 x 4096 1.4 -> 1.7).
template <typename T, bool kAligned>
__global__ void __launch_bounds__(kThreads)
    quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                    const T* x, int64_t stride, int64_t rows, int64_t rows_padded, int cols,
                    const Walk walk) {
  sm100::pdl_launch_dependents();
  sm100::pdl_wait_prior();
  int64_t row;
  int kb;
  first_item<1>(walk, row, kb);
  const bool live = row < rows && kb * 32 < cols;
  Block<T> in;
  if (live) {
    const T* p = x + row * stride + kb * 32;
    if constexpr (kAligned)
      in.load(p);
    else
      in.load_any(p, x, x + (rows - 1) * stride + cols);
  } else {
    in.zero();
  }
  const uint32_t e = in.top_exponent();
  const bool bad = e == 255;
  const uint32_t byte = bad ? 255u : e > 2 ? e - 2 : 0u;
  const float inv = __uint_as_float((254u - (bad ? 0u : byte)) << 23);
  uint32_t word[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f[8];
    in.get8(i, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= inv;
    word[i] = bad ? 0u : mx::encode_e2m1x8(f);
  }
  // Four neighbours are a row's four blocks of one scale tile.
  uint32_t four = byte << ((threadIdx.x & 3) * 8);
  four |= __shfl_xor_sync(0xffffffffu, four, 1);
  four |= __shfl_xor_sync(0xffffffffu, four, 2);
  if (live)
    *reinterpret_cast<uint4*>(codes + row * (cols / 2) + kb * 16) =
        make_uint4(word[0], word[1], word[2], word[3]);
  if ((threadIdx.x & 3) == 0 && row < rows_padded)
    *reinterpret_cast<uint32_t*>(scales + scale_byte(row, kb, walk.items_k)) = four;
}

// Elements per item when reading back: 32 bytes of output, so that a warp's
// stores are one run (whole blocks per lane gave 42.4 -> 46.8 us for 14336 x 4096
// fp32, and too few threads where there is little to do).
template <typename T>
constexpr int kOutItem = 32 / sizeof(T);
// Items per thread (1024 x 4096 bf16 with 1 / 2 / 4: 3.3 / 3.8 / 4.8 us, 4096 x 8192
// 14.2 / 12.3 / 12.1, 14336 x 4096 fp32 46.2 / 42.1 / 42.9).
constexpr int kOutUnroll = 2;

template <typename T, bool kAligned>
__global__ void __launch_bounds__(kThreads)
    dequantize_kernel(T* __restrict__ out, const uint8_t* codes, const uint8_t* scales,
                      int64_t rows, int cols, const Walk walk) {
  constexpr int E = kOutItem<T>, U = kOutUnroll;
  sm100::pdl_launch_dependents();
  sm100::pdl_wait_prior();
  uint32_t word[U][E / 8], byte[U];
  int64_t at[U], row;
  int item;
  first_item<U>(walk, row, item);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u > 0) next_item(walk, row, item);
    const int col = item * E;
    at[u] = row < rows && col < cols ? row * cols + col : -1;
    if (at[u] >= 0) {
      if constexpr (E == 16) {
        const uint2 w = *reinterpret_cast<const uint2*>(codes + at[u] / 2);
        word[u][0] = w.x;
        word[u][1] = w.y;
      } else {
        word[u][0] = *reinterpret_cast<const uint32_t*>(codes + at[u] / 2);
      }
      byte[u] = scales[scale_byte(row, col / 32, walk.items_k / (32 / E))];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] < 0) continue;
    float f[E];
#pragma unroll
    for (int j = 0; j < E; j += 8) mx::decode_e2m1x8(word[u][j / 8], f + j);
    const float s = mx::scale_value(byte[u]);
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] *= s;
    if constexpr (kAligned) {
      st_stream32(out + at[u], Elem<T>::pack(f), Elem<T>::pack(f + E / 2));
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) out[at[u] + j] = Elem<T>::from_f(f[j]);
    }
  }
}

int check(const char* who, const void* values, const void* codes, const void* scales, int64_t rows,
          int64_t cols, int dtype) {
  if (rows < 0 || cols < 0) return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: negative size", who);
  if (!valid_dtype(dtype)) return fail(AOTK_ERR_UNSUPPORTED, "%s: unsupported dtype %d", who, dtype);
  if (cols % 32 != 0)
    return fail(AOTK_ERR_UNSUPPORTED, "%s: cols = %lld is not a multiple of the block size 32", who,
                (long long)cols);
  if (rows == 0 || cols == 0) return AOTK_OK;
  if (!values || !codes || !scales)
    return fail(AOTK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(codes) || !aligned16(scales))
    return fail(AOTK_ERR_UNSUPPORTED, "%s: codes and scales must be 16-byte aligned", who);
  if (cols > 0x7fffff00LL || rows > 0x7fffff00LL)
    return fail(AOTK_ERR_UNSUPPORTED, "%s: extents above 2^31 - 256", who);
  return AOTK_OK;
}

template <typename... P, typename... A>
int launch(const char* who, void (*kernel)(P...), int64_t items, int per_thread, cudaStream_t s,
           A... args) {
  const int64_t per_block = static_cast<int64_t>(kLanes) * per_thread;
  const int64_t n = (items + per_block - 1) / per_block;
  if (n > 0x7fffffffLL) return fail(AOTK_ERR_UNSUPPORTED, "%s: too many elements", who);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(n), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(AOTK_ERR_CUDA, "%s launch: %s", who, cudaGetErrorString(e));
  return check_launch(who);
}

// Rows of whole 128-column scale tiles in items of `elements`.
Walk walk_of(int64_t cols, int elements) {
  const int items_k = static_cast<int>((cols + 127) / 128) * (128 / elements);
  return Walk{items_k, kLanes / items_k, kLanes % items_k};
}

bool aligned32(const void* p, int64_t row_bytes) {
  return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(row_bytes)) % 32 == 0;
}

template <typename T>
int quantize(void* codes, void* scales, const void* x, int64_t stride, int64_t rows, int64_t cols,
             cudaStream_t s) {
  const Walk walk = walk_of(cols, 32);
  const int64_t padded = (rows + 127) / 128 * 128;
  auto run = [&](auto kernel) {
    return launch("aotk_mxfp4_quantize", kernel, padded * walk.items_k, 1, s,
                  static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales),
                  static_cast<const T*>(x), stride, rows, padded, static_cast<int>(cols), walk);
  };
  return aligned32(x, rows > 1 ? stride * static_cast<int64_t>(sizeof(T)) : 0)
             ? run(quantize_kernel<T, true>)
             : run(quantize_kernel<T, false>);
}

template <typename T>
int dequantize(void* out, const void* codes, const void* scales, int64_t rows, int64_t cols,
               cudaStream_t s) {
  const Walk walk = walk_of(cols, kOutItem<T>);
  auto run = [&](auto kernel) {
    return launch("aotk_mxfp4_dequantize", kernel, rows * walk.items_k, kOutUnroll, s, static_cast<T*>(out),
                  static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows,
                  static_cast<int>(cols), walk);
  };
  return aligned32(out, 0) ? run(dequantize_kernel<T, true>) : run(dequantize_kernel<T, false>);
}

}  // namespace
}  // namespace aotk

extern "C" int aotk_mxfp4_quantize(void* codes, void* scales, const void* x, int64_t x_stride,
                                   int64_t rows, int64_t cols, int dtype, void* stream) {
  using namespace aotk;
  if (int st = check("aotk_mxfp4_quantize", x, codes, scales, rows, cols, dtype)) return st;
  if (rows == 0 || cols == 0) return AOTK_OK;
  if (rows > 1 && x_stride < cols)
    return fail(AOTK_ERR_INVALID_ARGUMENT, "aotk_mxfp4_quantize: row stride %lld < cols %lld",
                (long long)x_stride, (long long)cols);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case AOTK_FLOAT32: return quantize<float>(codes, scales, x, x_stride, rows, cols, s);
    case AOTK_FLOAT16: return quantize<__half>(codes, scales, x, x_stride, rows, cols, s);
    default: return quantize<__nv_bfloat16>(codes, scales, x, x_stride, rows, cols, s);
  }
}

extern "C" int aotk_mxfp4_dequantize(void* out, const void* codes, const void* scales, int64_t rows,
                                     int64_t cols, int dtype, void* stream) {
  using namespace aotk;
  if (int st = check("aotk_mxfp4_dequantize", out, codes, scales, rows, cols, dtype)) return st;
  if (rows == 0 || cols == 0) return AOTK_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case AOTK_FLOAT32: return dequantize<float>(out, codes, scales, rows, cols, s);
    case AOTK_FLOAT16: return dequantize<__half>(out, codes, scales, rows, cols, s);
    default: return dequantize<__nv_bfloat16>(out, codes, scales, rows, cols, s);
  }
}
