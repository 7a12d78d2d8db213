// Microscaled 4-bit floating point (OCP MX: E2M1 values in blocks of 32 along
// K, one E8M0 power of two each): quantisation, its inverse, and the products
// of two quantised operands, dense and grouped by expert.
//
// A quantised operand of `rows` x K:
//   data    rows x ldq bytes, two values a byte (the even one in the low half),
//           K padded to a multiple of 32 with zeros, ldq a multiple of 16;
//   scales  [ceil(K / 128)][rows] words of four E8M0 bytes (zero past K): one
//           word is what a row needs for K = 128, and words of neighbouring
//           rows are neighbours, so a tile may start at any row.
#include <cuda_fp4.h>

#include <algorithm>

#include "experts_host.hpp"

namespace tb {
namespace {

template <typename T>
__device__ __forceinline__ void load8(const T* src, int valid, bool vec, float (&x)[8]) {
  if (valid <= 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    return;
  }
  if (vec && valid >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(src));
      const float4 b = __ldg(reinterpret_cast<const float4*>(src) + 1);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          x[2 * i] = __uint_as_float(w[i] << 16);
          x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = i < valid ? static_cast<float>(src[i]) : 0.0f;
}

// Four lanes hold a block of 32 (8 values each). The block's unit is 2^(s - 127)
// with s = max(E, 2) - 2, E the biased exponent of the block's largest
// magnitude: the largest power of two not above it, divided by 4 (E2M1's
// largest power of two). Scaling by it is exact; the conversion rounds to the
// nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to even, and saturates (a block's
// largest magnitude is below 8 units). A block that holds an infinity or a NaN
// gets the NaN scale 255.
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], uint32_t& s) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const uint32_t E = m >> 23;
  if (E == 255) {
    s = 255;
    return 0;
  }
  s = max(E, 2u) - 2u;
  const float inv = __uint_as_float((254u - s) << 23);  // 2^(127 - s), normal
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(make_float2(x[2 * i] * inv, x[2 * i + 1] * inv),
                                                        __NV_E2M1, cudaRoundNearest))
         << (8 * i);
  return w;
}

// A warp takes 4 rows x 256 values, its lanes 8 neighbouring values of a row
// each: 16-byte loads and 128-byte stores, four of them in flight. Eight warps
// of a block take 32 neighbouring rows, so the scale words of a K block leave
// as 128 contiguous bytes. Bounded by the read of X.
template <typename T>
__global__ void __launch_bounds__(256)
    mxfp4_quantize_kernel(const T* __restrict__ X, long long ldx, int rows, int K, int vec,
                          uint8_t* __restrict__ data, long long ldq, uint32_t* __restrict__ scales) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = blockIdx.x * 32 + warp * 4;
  const int k = blockIdx.y * 256 + lane * 8;
  const int kwords = (K + 127) >> 7;
  float x[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    load8(X + (r0 + i < rows ? static_cast<long long>(r0 + i) * ldx + k : 0), r0 + i < rows ? K - k : 0, vec, x[i]);
  uint32_t word[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t s;
    const uint32_t w = quantize8(x[i], s);
    if (r0 + i < rows && (k >> 1) < ldq)
      *reinterpret_cast<uint32_t*>(data + static_cast<long long>(r0 + i) * ldq + (k >> 1)) = w;
    // the four scale bytes of 16 lanes; past K's last block zero
    if ((k & ~31) >= K) s = 0;
    uint32_t b = s << (8 * ((lane >> 2) & 3));
    b |= __shfl_xor_sync(0xffffffffu, b, 4);
    b |= __shfl_xor_sync(0xffffffffu, b, 8);
    word[i] = b;
  }
  const int kw = k >> 7;
  if ((lane & 15) == 0 && kw < kwords) {
    uint32_t* dst = scales + static_cast<long long>(kw) * rows + r0;
    if (r0 + 4 <= rows && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(word[0], word[1], word[2], word[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + i < rows) dst[i] = word[i];
    }
  }
}

template <typename T>
__device__ __forceinline__ T to_out(float v);
template <>
__device__ __forceinline__ float to_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half to_out<__half>(float v) { return __float2half_rn(v); }

// The values: 8 a lane, 4 rows a warp as above. An E2M1 code s ee m is the
// fp16 number with these bits at the sign, the low exponent and the top
// mantissa places, times 2^14 (subnormals included), so no table is read. The
// unit 2^(s - 127) is subnormal for s = 0 and NaN for s = 255; the product of
// a 2-bit mantissa and a power of two is exact, and rounds once to T.
template <typename T>
__global__ void __launch_bounds__(256)
    mxfp4_dequantize_kernel(const uint8_t* __restrict__ data, long long ldq,
                            const uint32_t* __restrict__ scales, int rows, int K, int vec,
                            T* __restrict__ Y, long long ldy) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r0 = blockIdx.x * 32 + warp * 4;
  const int k = blockIdx.y * 256 + lane * 8;
  if (k >= K) return;
  uint32_t w[4], sw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool ok = r0 + i < rows;
    w[i] = ok ? __ldg(reinterpret_cast<const uint32_t*>(data + static_cast<long long>(r0 + i) * ldq + (k >> 1))) : 0;
    sw[i] = ok ? __ldg(scales + static_cast<long long>(k >> 7) * rows + r0 + i) : 0;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r0 + i >= rows) break;
    const uint32_t s = (sw[i] >> (8 * ((k >> 5) & 3))) & 0xFFu;
    const float unit = s == 255 ? __uint_as_float(0x7FC00000u)
                                : (s == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23));
    T out[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t c = (w[i] >> (4 * j)) & 0xFu;
      const float v = __half2float(__ushort_as_half(static_cast<unsigned short>(((c & 8u) << 12) | ((c & 7u) << 9))));
      out[j] = to_out<T>(v * 16384.0f * unit);
    }
    T* dst = Y + static_cast<long long>(r0 + i) * ldy + k;
    if (vec && k + 8 <= K) {
#pragma unroll
      for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h)
        reinterpret_cast<uint4*>(dst)[h] = reinterpret_cast<const uint4*>(out)[h];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < K) dst[j] = out[j];
    }
  }
}

int check_mx(const char* what, int64_t rows, int64_t K, int64_t ldq) {
  const int64_t lim = (1ll << 31) - 512;
  if (rows < 0 || K < 0 || rows > lim || K > lim) {
    set_error(std::string(what) + ": sizes must be in [0, 2^31 - 512]");
    return TRNBLAS_ERR_ARG;
  }
  if (ldq < round_up(K, 32) / 2 || ldq % 16) {
    set_error(std::string(what) + ": a row of packed values takes round_up(K, 32) / 2 bytes at a stride of a multiple of 16");
    return TRNBLAS_ERR_ARG;
  }
  if (ceil_div(K, 256) > 65535) {
    set_error(std::string(what) + ": K above 65535 * 256");
    return TRNBLAS_ERR_ARG;
  }
  return TRNBLAS_OK;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" {

int trnblas_mxfp4_quantize(int dtype, int64_t rows, int64_t K, const void* X, int64_t ldx, void* data,
                           int64_t ldq, void* scales, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (dtype != TRNBLAS_F32 && dtype != TRNBLAS_BF16 && dtype != TRNBLAS_F16) {
    set_error("trnblas_mxfp4_quantize: dtype must be F32, BF16 or F16");
    return TRNBLAS_ERR_ARG;
  }
  if (int rc = check_mx("trnblas_mxfp4_quantize", rows, K, ldq)) return rc;
  if (rows == 0 || K == 0) return TRNBLAS_OK;
  if (!X || !data || !scales || ldx < K || !al16(data) || (reinterpret_cast<uintptr_t>(scales) & 3)) {
    set_error("trnblas_mxfp4_quantize: NULL or unaligned operand, or ldx smaller than K");
    return TRNBLAS_ERR_ARG;
  }
  const dim3 grid(static_cast<unsigned>(ceil_div(rows, 32)), static_cast<unsigned>(ceil_div(K, 256)));
  const int es = dtype == TRNBLAS_F32 ? 4 : 2;
  const int vec = al16(X) && (ldx * es) % 16 == 0;
  uint8_t* q = static_cast<uint8_t*>(data);
  uint32_t* s = static_cast<uint32_t*>(scales);
  const int r = static_cast<int>(rows), k = static_cast<int>(K);
  if (dtype == TRNBLAS_F32)
    mxfp4_quantize_kernel<float><<<grid, 256, 0, stream>>>(static_cast<const float*>(X), ldx, r, k, vec, q, ldq, s);
  else if (dtype == TRNBLAS_BF16)
    mxfp4_quantize_kernel<__nv_bfloat16>
        <<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(X), ldx, r, k, vec, q, ldq, s);
  else
    mxfp4_quantize_kernel<__half><<<grid, 256, 0, stream>>>(static_cast<const __half*>(X), ldx, r, k, vec, q, ldq, s);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "mxfp4 quantise kernel launch");
}

int trnblas_mxfp4_dequantize(int dtype, int64_t rows, int64_t K, const void* data, int64_t ldq,
                             const void* scales, void* Y, int64_t ldy, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (dtype != TRNBLAS_F32 && dtype != TRNBLAS_BF16 && dtype != TRNBLAS_F16) {
    set_error("trnblas_mxfp4_dequantize: dtype must be F32, BF16 or F16");
    return TRNBLAS_ERR_ARG;
  }
  if (int rc = check_mx("trnblas_mxfp4_dequantize", rows, K, ldq)) return rc;
  if (rows == 0 || K == 0) return TRNBLAS_OK;
  if (!Y || !data || !scales || ldy < K || !al16(data) || (reinterpret_cast<uintptr_t>(scales) & 3)) {
    set_error("trnblas_mxfp4_dequantize: NULL or unaligned operand, or ldy smaller than K");
    return TRNBLAS_ERR_ARG;
  }
  const dim3 grid(static_cast<unsigned>(ceil_div(rows, 32)), static_cast<unsigned>(ceil_div(K, 256)));
  const int es = dtype == TRNBLAS_F32 ? 4 : 2;
  const int vec = al16(Y) && (ldy * es) % 16 == 0;
  const uint8_t* q = static_cast<const uint8_t*>(data);
  const uint32_t* s = static_cast<const uint32_t*>(scales);
  const int r = static_cast<int>(rows), k = static_cast<int>(K);
  if (dtype == TRNBLAS_F32)
    mxfp4_dequantize_kernel<float><<<grid, 256, 0, stream>>>(q, ldq, s, r, k, vec, static_cast<float*>(Y), ldy);
  else if (dtype == TRNBLAS_BF16)
    mxfp4_dequantize_kernel<__nv_bfloat16>
        <<<grid, 256, 0, stream>>>(q, ldq, s, r, k, vec, static_cast<__nv_bfloat16*>(Y), ldy);
  else
    mxfp4_dequantize_kernel<__half><<<grid, 256, 0, stream>>>(q, ldq, s, r, k, vec, static_cast<__half*>(Y), ldy);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "mxfp4 dequantise kernel launch");
}

int trnblas_mxfp4_gemm(int out_dtype, int64_t rows, int64_t groups, int64_t N, int64_t K, float alpha,
                       const void* A, int64_t lda, const void* scalesA, const void* B, int64_t ldb,
                       const void* scalesB, const void* group_sizes, int sizes_64, float beta, const void* C,
                       int64_t ldc, void* D, int64_t ldd, void* stream) {
  if (out_dtype != TRNBLAS_F32 && out_dtype != TRNBLAS_BF16 && out_dtype != TRNBLAS_F16) {
    set_error("trnblas_mxfp4_gemm: out_dtype must be F32, BF16 or F16");
    return TRNBLAS_ERR_ARG;
  }
  if (int rc = check_group_dims("trnblas_mxfp4_gemm", rows, groups, N, K)) return rc;
  if (!group_sizes && groups != 1 && rows > 0 && groups > 0) {
    set_error("trnblas_mxfp4_gemm: several groups need group sizes");
    return TRNBLAS_ERR_ARG;
  }
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  if (!D || ldd < N || (C && beta != 0.0f && ldc < N)) {
    set_error("trnblas_mxfp4_gemm: NULL output, or ldc/ldd smaller than N");
    return TRNBLAS_ERR_ARG;
  }
  if (K == 0 || groups == 0)
    return trnblas_gemm(out_dtype, 1, rows, N, 0, alpha, nullptr, 1, 0, 0, nullptr, N, 0, 0, beta, C, ldc, 0,
                        D, ldd, 0, nullptr, 0, stream);
  if (int rc = check_mx("trnblas_mxfp4_gemm (A)", rows, K, lda)) return rc;
  if (int rc = check_mx("trnblas_mxfp4_gemm (B)", N, K, ldb)) return rc;
  if (!A || !B || !scalesA || !scalesB || (reinterpret_cast<uintptr_t>(scalesA) & 3) ||
      (reinterpret_cast<uintptr_t>(scalesB) & 3)) {
    set_error("trnblas_mxfp4_gemm: NULL operand, or scales not on 4 bytes");
    return TRNBLAS_ERR_ARG;
  }
  const auto dt = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const uint64_t kb = static_cast<uint64_t>(round_up(K, 32) / 2);
  // as for 16 bits: short row tiles and a deep pipeline where a group has at
  // most 64 rows on average
  const bool small = rows <= 64 * groups;
  CUtensorMap mw, mx, mx64;
  if (!encode_map_3d(&mw, dt, 1, B, kb, N, groups, ldb, ldb * N, 128, 128) ||
      !encode_map_3d(&mx, dt, 1, A, kb, rows, 1, lda, lda * rows, 128, small ? 64 : 192) ||
      !encode_map_3d(&mx64, dt, 1, A, kb, rows, 1, lda, lda * rows, 128, 64))
    return TRNBLAS_ERR_ALIGN;
  ExpertsParams p{};
  if (int rc = fill_experts(p, out_dtype, rows, groups, N, K, alpha, group_sizes, sizes_64, beta, C, ldc, D, ldd))
    return rc;
  p.xs = static_cast<const uint32_t*>(scalesA);
  p.xs_rows = rows;
  p.ws = static_cast<const uint32_t*>(scalesB);
  p.ws_rows = groups * N;
  return small ? launch_experts<kExpMx4, 64>(mw, mx, mx64, p, static_cast<cudaStream_t>(stream))
               : launch_experts<kExpMx4, 192>(mw, mx, mx64, p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
