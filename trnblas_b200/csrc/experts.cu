// C-ABI entry points of the products grouped by expert, 16-bit: the forward
// product (and with op(B) flipped the gradient of its rows) and the gradient
// of the weights.
#include <algorithm>

#include "experts_host.hpp"
#include "experts_wgrad_sm100.cuh"

namespace tb {
namespace {

// ---------------------------------------------------------------------------
// Operands that TMA cannot read (a base off 16 bytes, or a row or matrix stride
// that is no multiple of 8 elements) are copied to rows of round_up(cols, 8),
// both operands of a product in one launch. A thread writes 16 bytes; it reads
// in the widest pieces that every row of the source allows.
// ---------------------------------------------------------------------------
struct PadJob {
  const unsigned short* src;  // nullptr: none
  long long rows;             // all matrices
  int rows_per_matrix, cols;
  long long ld, stride;
  unsigned short* dst;
  int ldp;
  int piece;  // elements a load takes: 1, 2 or 4
};

__device__ __forceinline__ void pad_copy(const PadJob& j, long long first, long long step) {
  const int cq = j.ldp >> 3;
  const long long total = j.rows * cq;
  for (long long i = first; i < total; i += step) {
    const long long r = i / cq;
    const int c = static_cast<int>(i - r * cq) * 8;
    const long long m = r / j.rows_per_matrix;
    const unsigned short* s = j.src + m * j.stride + (r - m * j.rows_per_matrix) * j.ld + c;
    uint32_t w[4] = {0, 0, 0, 0};
    if (c + 8 <= j.cols && j.piece == 4) {
      const uint2 a = __ldg(reinterpret_cast<const uint2*>(s)), b = __ldg(reinterpret_cast<const uint2*>(s) + 1);
      w[0] = a.x, w[1] = a.y, w[2] = b.x, w[3] = b.y;
    } else if (c + 8 <= j.cols && j.piece == 2) {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = __ldg(reinterpret_cast<const uint32_t*>(s) + k);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < j.cols) w[k / 2] |= static_cast<uint32_t>(__ldg(s + k)) << (16 * (k & 1));
    }
    *reinterpret_cast<uint4*>(j.dst + r * j.ldp + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__global__ void __launch_bounds__(256) pad_rows_kernel(const PadJob a, const PadJob b) {
  const long long first = blockIdx.x * 256ll + threadIdx.x, step = gridDim.x * 256ll;
  if (a.src) pad_copy(a, first, step);
  if (b.src) pad_copy(b, first, step);
}

bool tma_readable(const void* X, int64_t ld, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(X) & 15) == 0 && ld % 8 == 0 && stride % 8 == 0;
}

size_t pad_bytes(const void* X, int64_t matrices, int64_t rows, int64_t cols, int64_t ld, int64_t stride) {
  return tma_readable(X, ld, stride) ? 0 : static_cast<size_t>(round_up(matrices * rows * round_up(cols, 8) * 2, 256));
}

// Redirects X / ld / stride to a padded copy in `ws` where TMA needs one.
PadJob pad_job(const void*& X, int64_t matrices, int64_t rows, int64_t cols, int64_t& ld, int64_t& stride,
               uint8_t*& ws) {
  PadJob j{};
  const size_t bytes = pad_bytes(X, matrices, rows, cols, ld, stride);
  if (!bytes) return j;
  j.src = static_cast<const unsigned short*>(X);
  j.rows = matrices * rows;
  j.rows_per_matrix = static_cast<int>(rows);
  j.cols = static_cast<int>(cols);
  j.ld = ld;
  j.stride = stride;
  j.dst = reinterpret_cast<unsigned short*>(ws);
  j.ldp = static_cast<int>(round_up(cols, 8));
  const uintptr_t al = reinterpret_cast<uintptr_t>(X) | static_cast<uintptr_t>(ld * 2) | static_cast<uintptr_t>(stride * 2);
  j.piece = al % 8 == 0 ? 4 : al % 4 == 0 ? 2 : 1;
  X = ws;
  ld = j.ldp;
  stride = rows * ld;
  ws += bytes;
  return j;
}

int launch_pad(const PadJob& a, const PadJob& b, cudaStream_t stream) {
  if (!a.src && !b.src) return TRNBLAS_OK;
  const long long n = (a.src ? a.rows * (a.ldp / 8) : 0) + (b.src ? b.rows * (b.ldp / 8) : 0);
  const int grid = static_cast<int>(std::min<long long>(ceil_div(n, 256), 16ll * num_sms()));
  pad_rows_kernel<<<grid, 256, 0, stream>>>(a, b);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "row padding kernel launch");
}

int check_workspace(const char* what, const void* ws, size_t have, size_t need) {
  if (need == 0 || (ws && have >= need && (reinterpret_cast<uintptr_t>(ws) & 15) == 0)) return TRNBLAS_OK;
  set_error(std::string(what) + ": operands off 16 bytes need " + std::to_string(need) +
            " workspace bytes, 16-byte aligned");
  return TRNBLAS_ERR_WORKSPACE;
}

int check_grouped(const char* what, int dtype, int out_dtype, int64_t rows, int64_t groups, int64_t N,
                  int64_t K, const void* sizes) {
  const std::string w(what);
  if (dtype != TRNBLAS_BF16 && dtype != TRNBLAS_F16) {
    set_error(w + ": dtype must be BF16 or F16");
    return TRNBLAS_ERR_ARG;
  }
  if (out_dtype != dtype && out_dtype != TRNBLAS_F32) {
    set_error(w + ": the output is of the operands' dtype or F32");
    return TRNBLAS_ERR_ARG;
  }
  if (int rc = check_group_dims(what, rows, groups, N, K)) return rc;
  if (groups > 0 && rows > 0 && !sizes) {
    set_error(w + ": NULL group sizes");
    return TRNBLAS_ERR_ARG;
  }
  return TRNBLAS_OK;
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" {

size_t trnblas_grouped_gemm_workspace_size(int64_t rows, int64_t groups, int64_t N, int64_t K, const void* A,
                                           int64_t lda, const void* B, int64_t ldb, int64_t strideB, int transB) {
  if (rows <= 0 || groups <= 0 || N <= 0 || K <= 0) return 0;
  const int64_t nb = groups == 1 || strideB == 0 ? 1 : groups;
  return pad_bytes(A, 1, rows, K, lda, 0) +
         pad_bytes(B, nb, transB ? N : K, transB ? K : N, ldb, nb > 1 ? strideB : 0);
}

size_t trnblas_grouped_gemm_wgrad_workspace_size(int64_t rows, int64_t M, int64_t N, const void* A, int64_t lda,
                                                 const void* B, int64_t ldb) {
  if (rows <= 0 || M <= 0 || N <= 0) return 0;
  return pad_bytes(A, 1, rows, M, lda, 0) + pad_bytes(B, 1, rows, N, ldb, 0);
}

int trnblas_grouped_gemm(int dtype, int out_dtype, int64_t rows, int64_t groups, int64_t N, int64_t K,
                         float alpha, const void* A, int64_t lda, const void* B, int64_t ldb,
                         int64_t strideB, int transB, const void* group_sizes, int sizes_64, float beta,
                         const void* C, int64_t ldc, void* D, int64_t ldd, void* workspace, size_t workspace_bytes,
                         void* stream) {
  if (int rc = check_grouped("trnblas_grouped_gemm", dtype, out_dtype, rows, groups, N, K, group_sizes))
    return rc;
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  if (!D || ldd < N || (C && beta != 0.0f && ldc < N)) {
    set_error("trnblas_grouped_gemm: NULL output, or ldc/ldd smaller than N");
    return TRNBLAS_ERR_ARG;
  }
  // no products at all: D = beta * C
  if (K == 0 || groups == 0)
    return trnblas_gemm(out_dtype, 1, rows, N, 0, alpha, nullptr, 1, 0, 0, nullptr, N, 0, 0, beta, C, ldc, 0,
                        D, ldd, 0, nullptr, 0, stream);
  const int64_t b_rows = transB ? N : K, b_cols = transB ? K : N;
  if (!A || !B || lda < K || ldb < b_cols || strideB < 0) {
    set_error("trnblas_grouped_gemm: NULL operand, or a stride smaller than the row length");
    return TRNBLAS_ERR_ARG;
  }
  const auto dt = dtype == TRNBLAS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const bool shared = groups == 1 || strideB == 0;  // one matrix
  const int64_t nb = shared ? 1 : groups;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int rc = check_workspace("trnblas_grouped_gemm", workspace, workspace_bytes,
                               trnblas_grouped_gemm_workspace_size(rows, groups, N, K, A, lda, B, ldb, strideB, transB)))
    return rc;
  {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    int64_t none = 0, sb0 = shared ? 0 : strideB;
    const PadJob ja = pad_job(A, 1, rows, K, lda, none, ws);
    const PadJob jb = pad_job(B, nb, b_rows, b_cols, ldb, sb0, ws);
    strideB = sb0;
    if (int rc = launch_pad(ja, jb, st)) return rc;
  }
  const int64_t sb = shared ? round_up(ldb * b_rows, 8) : strideB;
  const int64_t sa = round_up(lda * rows, 8);
  // Longer groups go to CTA pairs when there are weight columns for both.
  const bool small = small_tiles(rows, groups, N, true);
  const bool pair = !small && N > 128;
  const bool wide = !transB && N % 64 == 0;  // both 64-column blocks in one copy
  CUtensorMap mw, mx, mxs;
  bool ok;
  if (transB) {
    ok = encode_map_3d(&mw, dt, 2, B, K, N, nb, ldb, sb, 64, 128);
  } else if (wide) {
    const uint64_t dims[4] = {64, static_cast<uint64_t>(K), static_cast<uint64_t>(N / 64), static_cast<uint64_t>(nb)};
    const uint64_t strides[3] = {static_cast<uint64_t>(ldb), 64, static_cast<uint64_t>(sb)};
    const uint32_t box[4] = {64, 64, 2, 1};
    ok = encode_map(&mw, dt, 2, B, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    ok = encode_map_3d(&mw, dt, 2, B, N, K, nb, ldb, sb, 64, 64);
  }
  ok = ok && encode_map_3d(&mx, dt, 2, A, K, rows, 1, lda, sa, 64, pair ? 128 : small ? 64 : 256) &&
       encode_map_3d(&mxs, dt, 2, A, K, rows, 1, lda, sa, 64, pair ? 32 : small ? 16 : 64);
  if (!ok) return TRNBLAS_ERR_ALIGN;
  ExpertsParams p{};
  if (int rc = fill_experts(p, out_dtype, rows, groups, N, K, alpha, group_sizes, sizes_64, beta, C, ldc, D, ldd))
    return rc;
  p.in_fmt = dtype == TRNBLAS_BF16 ? kFmtBF16 : kFmtF16;
  p.w_mn = transB ? 0 : wide ? 2 : 1;
  p.w_shared = shared;
  if (small) return launch_experts<kExpF16, 64>(mw, mx, mxs, mw, mw, p, st);
  if (pair) return launch_experts_pair<kExpF16, 256, 2>(mw, mx, mxs, mw, mw, p, st);
  return launch_experts<kExpF16, 256>(mw, mx, mxs, mw, mw, p, st);
}

int trnblas_grouped_gemm_wgrad(int dtype, int out_dtype, int64_t rows, int64_t groups, int64_t M, int64_t N,
                               float alpha, const void* A, int64_t lda, const void* B, int64_t ldb,
                               const void* group_sizes, int sizes_64, float beta, const void* C, int64_t ldc,
                               int64_t strideC, void* D, int64_t ldd, int64_t strideD, void* workspace,
                               size_t workspace_bytes, void* stream_) {
  if (int rc = check_grouped("trnblas_grouped_gemm_wgrad", dtype, out_dtype, rows, groups, N, M, group_sizes))
    return rc;
  if (groups == 0 || M == 0 || N == 0) return TRNBLAS_OK;
  const bool has_c = C && beta != 0.0f;
  if (!D || ldd < N || (has_c && ldc < N) ||
      (groups > 1 && (strideD < ldd * M || (has_c && strideC < 0)))) {
    set_error("trnblas_grouped_gemm_wgrad: NULL output, or a C / D stride smaller than what it steps over");
    return TRNBLAS_ERR_ARG;
  }
  if (rows == 0)
    return trnblas_gemm(out_dtype, groups, M, N, 0, alpha, nullptr, 1, 0, 0, nullptr, N, 0, 0, beta, C, ldc,
                        strideC, D, ldd, strideD, nullptr, 0, stream_);
  if (!A || !B || lda < M || ldb < N) {
    set_error("trnblas_grouped_gemm_wgrad: NULL operand, or lda/ldb smaller than the row length");
    return TRNBLAS_ERR_ARG;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (int rc = check_workspace("trnblas_grouped_gemm_wgrad", workspace, workspace_bytes,
                               trnblas_grouped_gemm_wgrad_workspace_size(rows, M, N, A, lda, B, ldb)))
    return rc;
  {
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    int64_t none = 0;
    const PadJob ja = pad_job(A, 1, rows, M, lda, none, ws);
    none = 0;
    const PadJob jb = pad_job(B, 1, rows, N, ldb, none, ws);
    if (int rc = launch_pad(ja, jb, stream)) return rc;
  }
  const auto dt = dtype == TRNBLAS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  // CTA pairs (256 x 256 tiles) where both sides have columns for two CTAs
  const bool pair = M > 128 && N > 128;
  const int bm = pair ? WgradPairCfg::BM : WgradCfg::BM, bn = pair ? WgradPairCfg::BN : WgradCfg::BN;
  WgradParams w{};
  w.p.tiles_m = static_cast<int>(ceil_div(M, bm));
  w.p.tiles_n = static_cast<int>(ceil_div(N, bn));
  const long long tiles = groups * static_cast<long long>(w.p.tiles_m) * w.p.tiles_n;
  if (tiles > (1ll << 30)) {
    set_error("trnblas_grouped_gemm_wgrad: too many tiles");
    return TRNBLAS_ERR_ARG;
  }
  w.p.M = static_cast<int>(M);
  w.p.N = static_cast<int>(N);
  w.p.out_kind = out_kind_of(out_dtype);
  w.p.c_mode = has_c ? kCRow : kCNone;
  w.p.alpha = alpha;
  w.p.beta = beta;
  w.p.C = C;
  w.p.ldc = ldc;
  w.p.strideC = strideC;
  w.p.D = D;
  w.p.ldd = ldd;
  w.p.strideD = strideD;
  w.p.num_tiles = static_cast<int>(tiles);
  w.p.status = status_word();
  if (!w.p.status) return TRNBLAS_ERR_CUDA;
  w.p.timeout_ns = wait_timeout_ns();
  w.rows = static_cast<int>(rows);
  w.groups = static_cast<int>(groups);
  w.sizes = group_sizes;
  w.sizes64 = sizes_64;
  w.in_fmt = dtype == TRNBLAS_BF16 ? kFmtBF16 : kFmtF16;
  // whole blocks of 64 columns: a map of 64 columns x rows x blocks, so that one
  // copy brings 128 columns
  w.wide = pair && M % 64 == 0 && N % 64 == 0;
  CUtensorMap ma, mb, md;
  auto rows_map = [&](CUtensorMap* m, const void* X, int64_t cols, int64_t ld) {
    if (!w.wide) return encode_map_3d(m, dt, 2, X, cols, rows, 1, ld, round_up(ld * rows, 8), 64, 64);
    const uint64_t dims[3] = {64, static_cast<uint64_t>(rows), static_cast<uint64_t>(cols / 64)};
    const uint64_t strides[2] = {static_cast<uint64_t>(ld), 64};
    const uint32_t box[3] = {64, 64, 2};
    return encode_map(m, dt, 2, X, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  if (!rows_map(&ma, A, M, lda) || !rows_map(&mb, B, N, ldb)) return TRNBLAS_ERR_ALIGN;
  static bool attr_set[64] = {}, pair_attr_set[64] = {};
  if (!pair) {
    if (int rc = smem_attribute(reinterpret_cast<const void*>(&wgrad_kernel), WgradCfg::SMEM, attr_set)) return rc;
    const int grid = static_cast<int>(std::min<long long>(tiles, num_sms()));
    wgrad_kernel<<<grid, WgradCfg::THREADS, WgradCfg::SMEM, stream>>>(ma, mb, w);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "weight gradient kernel launch");
  }
  // stores by TMA where D's rows lie on 16 bytes and no C is added
  const int oes = out_dtype == TRNBLAS_F32 ? 4 : 2;
  const int64_t sd = groups > 1 ? strideD : round_up(ldd * M, 8);
  w.tma_d = !has_c && (reinterpret_cast<uintptr_t>(D) & 15) == 0 && (ldd * oes) % 16 == 0 && (sd * oes) % 16 == 0;
  md = ma;
  const uint64_t ddims[3] = {static_cast<uint64_t>(N), static_cast<uint64_t>(M), static_cast<uint64_t>(groups)};
  const uint64_t dstrides[2] = {static_cast<uint64_t>(ldd), static_cast<uint64_t>(sd)};
  const uint32_t dbox[3] = {static_cast<uint32_t>(64 / oes), 32, 1};
  if (w.tma_d && !encode_map(&md,
                             out_dtype == TRNBLAS_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                             : out_dtype == TRNBLAS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                             oes, D, 3, ddims, dstrides, dbox, CU_TENSOR_MAP_SWIZZLE_64B))
    return TRNBLAS_ERR_ALIGN;
  if (int rc = smem_attribute(reinterpret_cast<const void*>(&wgrad_pair_kernel), WgradPairCfg::SMEM, pair_attr_set))
    return rc;
  static int max_pairs[64] = {};
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pair_config(attr, WgradPairCfg::THREADS, WgradPairCfg::SMEM, stream);
  int pairs = 0;
  if (int rc = resident_pairs(wgrad_pair_kernel, cfg, max_pairs, pairs)) return rc;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<long long>(tiles, pairs)), 1, 1);
  cudaError_t e = cudaLaunchKernelEx(&cfg, wgrad_pair_kernel, ma, mb, md, static_cast<const WgradParams>(w));
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "weight gradient pair kernel launch");
}

}  // extern "C"
