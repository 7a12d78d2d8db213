// Host helpers of the products grouped by expert, shared by their 16-bit and
// 4-bit entry points.
#pragma once

#include <algorithm>
#include <string>

#include "experts_sm100.cuh"
#include "runtime.hpp"

namespace tb {

inline int out_kind_of(int dtype) {
  return dtype == TRNBLAS_F32 ? kOutF32 : dtype == TRNBLAS_BF16 ? kOutBF16 : kOutF16;
}

inline int check_group_dims(const char* what, int64_t rows, int64_t groups, int64_t N, int64_t K) {
  const int64_t lim = (1ll << 31) - 512;  // tile and box ends stay within an int
  if (rows < 0 || groups < 0 || N < 0 || K < 0 || rows > lim || N > lim || K > lim) {
    set_error(std::string(what) + ": sizes must be in [0, 2^31 - 512]");
    return TRNBLAS_ERR_ARG;
  }
  if (groups > kMaxGroups) {
    set_error(std::string(what) + ": at most " + std::to_string(kMaxGroups) + " groups");
    return TRNBLAS_ERR_ARG;
  }
  return TRNBLAS_OK;
}

// Dynamic shared memory above 48 KB, once per kernel and device (`done`: the
// kernel's flags).
inline int smem_attribute(const void* kernel, int bytes, bool (&done)[64]) {
  const int dev = current_device();
  if (dev >= 0 && dev < 64 && done[dev]) return TRNBLAS_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute(shared memory)");
  if (dev >= 0 && dev < 64) done[dev] = true;
  return TRNBLAS_OK;
}

inline int fill_experts(ExpertsParams& p, int out_dtype, int64_t rows, int64_t groups, int64_t N, int64_t K,
                        float alpha, const void* sizes, int sizes_64, float beta, const void* C, int64_t ldc,
                        void* D, int64_t ldd) {
  p.rows = static_cast<int>(rows);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.groups = static_cast<int>(groups);
  p.sizes = sizes;
  p.sizes64 = sizes_64;
  p.out_kind = out_kind_of(out_dtype);
  p.alpha = alpha;
  p.beta = beta;
  p.C = C;
  p.ldc = ldc;
  p.D = D;
  p.ldd = ldd;
  p.tiles_w = static_cast<int>(ceil_div(N, 128));
  p.status = status_word();
  if (!p.status) return TRNBLAS_ERR_CUDA;
  p.timeout_ns = wait_timeout_ns();
  return TRNBLAS_OK;
}

template <int KIND, int BN>
int launch_experts(const CUtensorMap& mw, const CUtensorMap& mx, const CUtensorMap& mx64,
                   const ExpertsParams& p, cudaStream_t stream) {
  using Cfg = ExpCfg<KIND, BN>;
  // at most one partly filled row tile a group, and the rows behind the last
  const long long tiles =
      (ceil_div(p.rows, BN) + std::min<long long>(p.groups, p.rows) + 1) * static_cast<long long>(p.tiles_w);
  if (tiles > (1ll << 30)) {
    set_error("grouped product: too many tiles");
    return TRNBLAS_ERR_ARG;
  }
  auto kern = experts_kernel<KIND, BN>;
  static bool attr_set[64] = {};
  if (int rc = smem_attribute(reinterpret_cast<const void*>(kern), Cfg::SMEM, attr_set)) return rc;
  const int grid = static_cast<int>(std::min<long long>(tiles, num_sms()));
  kern<<<grid, Cfg::THREADS, Cfg::SMEM, stream>>>(mw, mx, mx64, p);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "grouped product kernel launch");
}

}  // namespace tb
