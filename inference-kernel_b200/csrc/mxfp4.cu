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
// row (a lane 8 elements: one or two 16-byte loads, one 4-byte word of codes;
// four lanes a block, one shuffle pair for its maximum; 16 lanes one 4-byte
// word of scales), and each lane has kUnroll such loads in flight.
#include "common.h"
#include "mxfp4.cuh"
#include "vec.cuh"

namespace aotk {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;                              // tiles in flight per half-warp
constexpr int kTilesPerBlock = kThreads / 16 * kUnroll;  // 128-column row tiles

// Eight consecutive elements as 16-byte vectors (kVec) or one by one.
template <typename T, bool kVec>
struct Eight {
  static constexpr int kWords = 8 / Elem<T>::kPerVec;
  uint4 raw[kWords];
  T one[kVec ? 1 : 8];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (!kVec) {
#pragma unroll
      for (int i = 0; i < 8; ++i) one[i] = Elem<T>::from_f(0.f);
    }
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) raw[i] = ld_stream(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) one[i] = p[i];
    }
  }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) Elem<T>::unpack(raw[i], f + i * Elem<T>::kPerVec);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = Elem<T>::to_f(one[i]);
    }
  }
};

// Row tile t of the padded problem: row t / tiles_k, columns [128 (t % tiles_k), +128).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
    quantize_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                    const T* __restrict__ x, int64_t stride, int64_t rows, int64_t cols,
                    int tiles_k, int64_t tiles) {
  const int lane16 = threadIdx.x & 15;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTilesPerBlock + threadIdx.x / 16;
  Eight<T, kVec> in[kUnroll];
  int64_t row[kUnroll], col[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t t = t0 + u * (kThreads / 16);
    row[u] = t / tiles_k;
    col[u] = (t - row[u] * tiles_k) * 128 + lane16 * 8;
    if (row[u] < rows && col[u] < cols)
      in[u].load(x + row[u] * stride + col[u]);
    else
      in[u].zero();
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    float f[8];
    in[u].get(f);
    // Magnitudes as integers: they order like the values, and a NaN is above
    // an infinity, which is above all else.
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t biased = top >> 23;
    const uint32_t byte = biased == 255 ? 255u : biased > 2 ? biased - 2 : 0u;
    const float inv = __uint_as_float((254u - (byte == 255 ? 254u : byte)) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= inv;
    uint32_t word = mx::encode_e2m1x8(f);
    if (byte == 255) word = 0;
    const int base = threadIdx.x & 16;
    const uint32_t b0 = __shfl_sync(0xffffffffu, byte, base);
    const uint32_t b1 = __shfl_sync(0xffffffffu, byte, base + 4);
    const uint32_t b2 = __shfl_sync(0xffffffffu, byte, base + 8);
    const uint32_t b3 = __shfl_sync(0xffffffffu, byte, base + 12);
    const int64_t t = t0 + u * (kThreads / 16);
    if (t < tiles) {
      if (row[u] < rows && col[u] < cols)
        *reinterpret_cast<uint32_t*>(codes + (row[u] * cols + col[u]) / 2) = word;
      if (lane16 == 0) {
        const int64_t tile = (row[u] / 128) * tiles_k + (t - row[u] * tiles_k);
        const int r = static_cast<int>(row[u] % 128);
        *reinterpret_cast<uint32_t*>(scales + tile * 512 + (r % 32) * 16 + r / 32 * 4) =
            b0 | b1 << 8 | b2 << 16 | b3 << 24;
      }
    }
  }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
    dequantize_kernel(T* __restrict__ out, const uint8_t* __restrict__ codes,
                      const uint8_t* __restrict__ scales, int64_t rows, int64_t cols, int tiles_k,
                      int64_t tiles) {
  const int lane16 = threadIdx.x & 15;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTilesPerBlock + threadIdx.x / 16;
  uint32_t word[kUnroll], byte[kUnroll];
  int64_t at[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t t = t0 + u * (kThreads / 16);
    const int64_t row = t / tiles_k;
    const int64_t kt = t - row * tiles_k;
    const int64_t col = kt * 128 + lane16 * 8;
    at[u] = t < tiles && col < cols ? row * cols + col : -1;
    if (at[u] >= 0) {
      word[u] = *reinterpret_cast<const uint32_t*>(codes + at[u] / 2);
      const int r = static_cast<int>(row % 128);
      byte[u] = scales[((row / 128) * tiles_k + kt) * 512 + (r % 32) * 16 + r / 32 * 4 + lane16 / 4];
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
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < 8 / Elem<T>::kPerVec; ++i)
        st_stream(reinterpret_cast<uint4*>(out + at[u]) + i,
                  Elem<T>::pack(f + i * Elem<T>::kPerVec));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) out[at[u] + i] = Elem<T>::from_f(f[i]);
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

int blocks_for(const char* who, int64_t tiles, unsigned* blocks) {
  const int64_t n = (tiles + kTilesPerBlock - 1) / kTilesPerBlock;
  if (n > 0x7fffffffLL) return fail(AOTK_ERR_UNSUPPORTED, "%s: too many elements", who);
  *blocks = static_cast<unsigned>(n);
  return AOTK_OK;
}

template <typename T>
int quantize(void* codes, void* scales, const void* x, int64_t stride, int64_t rows, int64_t cols,
             cudaStream_t s) {
  const int tiles_k = static_cast<int>((cols + 127) / 128);
  const int64_t tiles = (rows + 127) / 128 * 128 * tiles_k;
  unsigned blocks;
  if (int st = blocks_for("aotk_mxfp4_quantize", tiles, &blocks)) return st;
  const bool vec = aligned16(x) && stride * static_cast<int64_t>(sizeof(T)) % 16 == 0;
  auto* c = static_cast<uint8_t*>(codes);
  auto* sc = static_cast<uint8_t*>(scales);
  auto* xt = static_cast<const T*>(x);
  if (vec)
    quantize_kernel<T, true><<<blocks, kThreads, 0, s>>>(c, sc, xt, stride, rows, cols, tiles_k, tiles);
  else
    quantize_kernel<T, false><<<blocks, kThreads, 0, s>>>(c, sc, xt, stride, rows, cols, tiles_k, tiles);
  return check_launch("aotk_mxfp4_quantize");
}

template <typename T>
int dequantize(void* out, const void* codes, const void* scales, int64_t rows, int64_t cols,
               cudaStream_t s) {
  const int tiles_k = static_cast<int>((cols + 127) / 128);
  const int64_t tiles = rows * tiles_k;
  unsigned blocks;
  if (int st = blocks_for("aotk_mxfp4_dequantize", tiles, &blocks)) return st;
  auto* o = static_cast<T*>(out);
  auto* c = static_cast<const uint8_t*>(codes);
  auto* sc = static_cast<const uint8_t*>(scales);
  if (aligned16(out))
    dequantize_kernel<T, true><<<blocks, kThreads, 0, s>>>(o, c, sc, rows, cols, tiles_k, tiles);
  else
    dequantize_kernel<T, false><<<blocks, kThreads, 0, s>>>(o, c, sc, rows, cols, tiles_k, tiles);
  return check_launch("aotk_mxfp4_dequantize");
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
