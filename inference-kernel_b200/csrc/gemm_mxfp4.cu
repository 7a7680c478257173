// Product of two microscaled 4-bit matrices: C[m, n] = sum_k A[m, k] B[n, k],
// A [M, K / 2] and B [N, K / 2] codes with scale tiles as in mxfp4.cu, fp32
// accumulation, one rounding to the output type.
//
// 64 x 64 tile per block, 4 x 4 outputs per thread, K in steps of one block of
// 32, decoded into shared memory as fp32 once per tile.  A block's sum of
// products of elements is exact (multiples of 1/4 up to 1152) and takes both
// scales at once, so that no factor leaves fp32's range before the product does.
#include "common.h"
#include "mxfp4.cuh"
#include "vec.cuh"

namespace aotk {
namespace {

constexpr int kTile = 64;

// Row r, block j of a scale array.
__device__ __forceinline__ uint32_t scale_at(const uint8_t* s, int64_t r, int64_t j, int tiles_k) {
  return s[((r / 128) * tiles_k + j / 4) * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + j % 4];
}

template <typename T>
__global__ void __launch_bounds__(256)
    gemm_mxfp4_simt_kernel(T* __restrict__ c, const uint8_t* __restrict__ a,
                           const uint8_t* __restrict__ as, const uint8_t* __restrict__ b,
                           const uint8_t* __restrict__ bs, int64_t M, int64_t N, int64_t K,
                           int tiles_k) {
  __shared__ float sa[kTile][33], sb[kTile][33];
  __shared__ int ea[kTile], eb[kTile];  // exponents of the block's scales
  constexpr int kNan = 1 << 20;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kTile;
  const int r = threadIdx.x / 4, q = threadIdx.x % 4;  // row and 8-element word of a block
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += 32) {
    float va[8] = {}, vb[8] = {};
    uint32_t xa = 127, xb = 127;
    if (m0 + r < M) {
      mx::decode_e2m1x8(*reinterpret_cast<const uint32_t*>(a + ((m0 + r) * K + k0) / 2 + q * 4), va);
      xa = scale_at(as, m0 + r, k0 / 32, tiles_k);
    }
    if (n0 + r < N) {
      mx::decode_e2m1x8(*reinterpret_cast<const uint32_t*>(b + ((n0 + r) * K + k0) / 2 + q * 4), vb);
      xb = scale_at(bs, n0 + r, k0 / 32, tiles_k);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sa[r][q * 8 + i] = va[i];
      sb[r][q * 8 + i] = vb[i];
    }
    if (q == 0) {
      ea[r] = xa == 255 ? kNan : static_cast<int>(xa) - 127;
      eb[r] = xb == 255 ? kNan : static_cast<int>(xb) - 127;
    }
    __syncthreads();
    float sum[4][4] = {};
#pragma unroll 8
    for (int k = 0; k < 32; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sum[i][j] = fmaf(sa[ty + 16 * i][k], sb[tx + 16 * j][k], sum[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = ea[ty + 16 * i] + eb[tx + 16 * j];
        acc[i][j] += e >= kNan / 2 ? __int_as_float(0x7FC00000) : ldexpf(sum[i][j], e);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < M && n < N) c[m * N + n] = Elem<T>::from_f(acc[i][j]);
    }
}

template <typename T>
int launch(void* c, const void* a, const void* as, const void* b, const void* bs, int64_t M,
           int64_t N, int64_t K, cudaStream_t s) {
  const int64_t gy = (M + kTile - 1) / kTile;
  if (gy > 65535) return fail(AOTK_ERR_UNSUPPORTED, "aotk_mxfp4_gemm: M = %lld", (long long)M);
  const dim3 grid(static_cast<unsigned>((N + kTile - 1) / kTile), static_cast<unsigned>(gy));
  gemm_mxfp4_simt_kernel<T><<<grid, 256, 0, s>>>(
      static_cast<T*>(c), static_cast<const uint8_t*>(a), static_cast<const uint8_t*>(as),
      static_cast<const uint8_t*>(b), static_cast<const uint8_t*>(bs), M, N, K,
      static_cast<int>((K + 127) / 128));
  return check_launch("aotk_mxfp4_gemm");
}

}  // namespace
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
  switch (out_dtype) {
    case AOTK_FLOAT32: return launch<float>(c, a, a_scales, b, b_scales, M, N, K, s);
    case AOTK_FLOAT16: return launch<__half>(c, a, a_scales, b, b_scales, M, N, K, s);
    default: return launch<__nv_bfloat16>(c, a, a_scales, b, b_scales, M, N, K, s);
  }
}
