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
// Both kernels are bound by HBM.  A half-warp owns one 128-column tile of one
// row: a lane 8 elements (one 16-byte or 32-byte load), which make one 4-byte word
// of codes; four lanes a block, two shuffles for its maximum; 16 lanes one 4-byte
// word of scales, two more.  Each lane has kUnroll loads in flight.
#include "common.h"
#include "mxfp4.cuh"
#include "sm100.cuh"
#include "vec.cuh"

namespace aotk {
namespace {

constexpr int kThreads = 256;
constexpr int kRowTiles = kThreads / 16;  // 128-column row tiles per block at a time
constexpr int kUnroll = 4;                // of each half-warp, kRowTiles apart

// Row tile t of the problem is columns [128 (t % tiles_k), +128) of row t / tiles_k.
// A block's tiles are consecutive; step = kRowTiles tiles on.
struct Walk {
  int tiles_k;
  int step_rows, step_tiles;  // kRowTiles / tiles_k and the remainder
};

// This half-warp's first tile: one division by a uniform value and one of small
// numbers per thread, and none from tile to tile.
__device__ __forceinline__ void first_tile(const Walk& w, int64_t& row, int& kt) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kRowTiles * kUnroll);
  const int64_t row0 = t / w.tiles_k;
  const unsigned in_row = static_cast<unsigned>(t - row0 * w.tiles_k) + threadIdx.x / 16;
  const unsigned more = in_row / static_cast<unsigned>(w.tiles_k);
  row = row0 + more;
  kt = static_cast<int>(in_row - more * w.tiles_k);
}

__device__ __forceinline__ void next_tile(const Walk& w, int64_t& row, int& kt) {
  row += w.step_rows;
  kt += w.step_tiles;
  if (kt >= w.tiles_k) {
    kt -= w.tiles_k;
    ++row;
  }
}

__device__ __forceinline__ int64_t scale_word(int64_t row, int kt, int tiles_k) {
  const int r = static_cast<int>(row & 127);
  return ((row >> 7) * tiles_k + kt) * 512 + (r & 31) * 16 + (r >> 5) * 4;
}

enum : int { kElements = 0, kVectors = 1, kWide = 2 };  // accesses of 1, 16 / sizeof, 32 / sizeof

// Eight consecutive elements of a lane.
template <typename T, int kAccess>
struct Eight {
  static constexpr int kWords = sizeof(T) / 2;  // 16-byte vectors
  uint4 raw[kWords];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kAccess == kWide) {
      ld_stream32(p, raw[0], raw[1]);
    } else if constexpr (kAccess == kVectors) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) raw[i] = ld_stream(reinterpret_cast<const uint4*>(p) + i);
    } else {
      T* e = reinterpret_cast<T*>(raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) Elem<T>::unpack(raw[i], f + i * Elem<T>::kPerVec);
  }
  // Bits of the largest magnitude as fp32.  Magnitudes order like their bits,
  // with infinity above all numbers and NaN above it; 16-bit ones are compared
  // in pairs.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        m = max(m, max(max(raw[i].x & 0x7FFFFFFFu, raw[i].y & 0x7FFFFFFFu),
                       max(raw[i].z & 0x7FFFFFFFu, raw[i].w & 0x7FFFFFFFu)));
      return m;
    } else {
      const uint32_t m = __vmaxu2(__vmaxu2(raw[0].x & 0x7FFF7FFFu, raw[0].y & 0x7FFF7FFFu),
                                  __vmaxu2(raw[0].z & 0x7FFF7FFFu, raw[0].w & 0x7FFF7FFFu));
      const uint16_t h = static_cast<uint16_t>(max(m & 0xFFFFu, m >> 16));
      return __float_as_uint(Elem<T>::to_f(*reinterpret_cast<const T*>(&h)));
    }
  }
};

template <typename T, int kAccess>
__global__ void __launch_bounds__(kThreads)
    quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                    const T* __restrict__ x, int64_t stride, int64_t rows, int64_t rows_padded,
                    int cols, const Walk walk) {
  const int lane16 = threadIdx.x & 15;
  sm100::pdl_launch_dependents();
  sm100::pdl_wait_prior();
  Eight<T, kAccess> in[kUnroll];
  int64_t row[kUnroll];
  int kt[kUnroll];
  first_tile(walk, row[0], kt[0]);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (u > 0) {
      row[u] = row[u - 1];
      kt[u] = kt[u - 1];
      next_tile(walk, row[u], kt[u]);
    }
    const int col = kt[u] * 128 + lane16 * 8;
    if (row[u] < rows && col < cols)
      in[u].load(x + row[u] * stride + col);
    else
      in[u].zero();
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    uint32_t top = in[u].top();
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t biased = top >> 23;
    const bool bad = biased == 255;
    const uint32_t byte = bad ? 255u : biased > 2 ? biased - 2 : 0u;
    float f[8];
    in[u].get(f);
    const float inv = __uint_as_float((254u - (bad ? 0u : byte)) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= inv;
    const uint32_t word = bad ? 0u : mx::encode_e2m1x8(f);
    uint32_t four = byte << (lane16 / 4 * 8);
    four |= __shfl_xor_sync(0xffffffffu, four, 4);
    four |= __shfl_xor_sync(0xffffffffu, four, 8);
    const int col = kt[u] * 128 + lane16 * 8;
    if (row[u] < rows && col < cols)
      *reinterpret_cast<uint32_t*>(codes + row[u] * (cols / 2) + col / 2) = word;
    if (lane16 == 0 && row[u] < rows_padded)
      *reinterpret_cast<uint32_t*>(scales + scale_word(row[u], kt[u], walk.tiles_k)) = four;
  }
}

template <typename T, int kAccess>
__global__ void __launch_bounds__(kThreads)
    dequantize_kernel(T* __restrict__ out, const uint8_t* __restrict__ codes,
                      const uint8_t* __restrict__ scales, int64_t rows, int cols, const Walk walk) {
  const int lane16 = threadIdx.x & 15;
  sm100::pdl_launch_dependents();
  sm100::pdl_wait_prior();
  uint32_t word[kUnroll], byte[kUnroll];
  int64_t at[kUnroll], row;
  int kt;
  first_tile(walk, row, kt);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (u > 0) next_tile(walk, row, kt);
    const int col = kt * 128 + lane16 * 8;
    at[u] = row < rows && col < cols ? row * cols + col : -1;
    if (at[u] >= 0) {
      word[u] = *reinterpret_cast<const uint32_t*>(codes + at[u] / 2);
      byte[u] = scales[scale_word(row, kt, walk.tiles_k) + lane16 / 4];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (at[u] < 0) continue;
    float f[8];
    mx::decode_e2m1x8(word[u], f);
    const float s = mx::scale_value(byte[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= s;
    T* o = out + at[u];
    if constexpr (kAccess == kWide) {
      st_stream32(o, Elem<T>::pack(f), Elem<T>::pack(f + 4));
    } else if constexpr (kAccess == kVectors) {
#pragma unroll
      for (int i = 0; i < 8 / Elem<T>::kPerVec; ++i)
        st_stream(reinterpret_cast<uint4*>(o) + i, Elem<T>::pack(f + i * Elem<T>::kPerVec));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = Elem<T>::from_f(f[i]);
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
  if (cols > 0x7fffffffLL || rows > 0x7fffffffLL)
    return fail(AOTK_ERR_UNSUPPORTED, "%s: extents above 2^31 - 1", who);
  return AOTK_OK;
}

template <typename... P, typename... A>
int launch(const char* who, void (*kernel)(P...), int64_t row_tiles, cudaStream_t s, A... args) {
  const int64_t n = (row_tiles + kRowTiles * kUnroll - 1) / (kRowTiles * kUnroll);
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

Walk walk_of(int64_t cols) {
  const int tiles_k = static_cast<int>((cols + 127) / 128);
  return Walk{tiles_k, kRowTiles / tiles_k, kRowTiles % tiles_k};
}

// Rows of 32 columns are 64 or 128 bytes, so the base and the row stride decide.
template <typename T>
int access_of(const void* p, int64_t stride) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride * sizeof(T));
  if (sizeof(T) == 4 && bits % 32 == 0) return kWide;
  return bits % 16 == 0 ? kVectors : kElements;
}

template <typename T>
int quantize(void* codes, void* scales, const void* x, int64_t stride, int64_t rows, int64_t cols,
             cudaStream_t s) {
  const char* who = "aotk_mxfp4_quantize";
  const Walk walk = walk_of(cols);
  const int64_t padded = (rows + 127) / 128 * 128;
  auto run = [&](auto kernel) {
    return launch(who, kernel, padded * walk.tiles_k, s, static_cast<uint8_t*>(codes),
                  static_cast<uint8_t*>(scales), static_cast<const T*>(x), stride, rows, padded,
                  static_cast<int>(cols), walk);
  };
  const int access = access_of<T>(x, rows > 1 ? stride : 0);
  if constexpr (sizeof(T) == 4)
    if (access == kWide) return run(quantize_kernel<T, kWide>);
  return access == kVectors ? run(quantize_kernel<T, kVectors>) : run(quantize_kernel<T, kElements>);
}

template <typename T>
int dequantize(void* out, const void* codes, const void* scales, int64_t rows, int64_t cols,
               cudaStream_t s) {
  const char* who = "aotk_mxfp4_dequantize";
  const Walk walk = walk_of(cols);
  auto run = [&](auto kernel) {
    return launch(who, kernel, rows * walk.tiles_k, s, static_cast<T*>(out),
                  static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows,
                  static_cast<int>(cols), walk);
  };
  const int access = access_of<T>(out, 0);
  if constexpr (sizeof(T) == 4)
    if (access == kWide) return run(dequantize_kernel<T, kWide>);
  return access == kVectors ? run(dequantize_kernel<T, kVectors>)
                            : run(dequantize_kernel<T, kElements>);
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
