// Host helpers of the products grouped by expert, shared by their 16-bit and
// 4-bit entry points.
#pragma once

#include <algorithm>
#include <string>

#include "experts_pair_sm100.cuh"
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

inline cudaLaunchConfig_t pair_config(cudaLaunchAttribute (&attr)[2], int threads, int smem,
                                      cudaStream_t stream, bool dependent = false) {
  cudaLaunchConfig_t cfg{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * (num_sms() / 2)), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  return cfg;
}

// CTA pairs that fit on the device at once, asked once per kernel and device.
template <typename Kernel>
int resident_pairs(Kernel kern, const cudaLaunchConfig_t& cfg, int (&cache)[64], int& pairs) {
  const int dev = current_device();
  if (dev >= 0 && dev < 64 && cache[dev]) {
    pairs = cache[dev];
    return TRNBLAS_OK;
  }
  cudaError_t e = cudaOccupancyMaxActiveClusters(&pairs, kern, &cfg);
  if (e != cudaSuccess) return cuda_fail(e, "cudaOccupancyMaxActiveClusters");
  if (pairs < 1) {
    set_error("no CTA pair fits on this device");
    return TRNBLAS_ERR_CUDA;
  }
  if (dev >= 0 && dev < 64) cache[dev] = pairs;
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
  p.status = status_word();
  if (!p.status) return TRNBLAS_ERR_CUDA;
  p.timeout_ns = wait_timeout_ns();
  return TRNBLAS_OK;
}

// Row tiles of 64 on single CTAs: where a group has at most 64 rows on average
// (eight pipeline stages keep more weight bytes in flight, which is what bounds
// a few rows a group), or where even these tiles make at most one wave. Pairs
// otherwise. Measured with weights from DRAM, small against pair, 16 groups of m
// rows, K 2048, N 4096: bf16 m = 16 47.7 / 50.5 us, 64 49.4 / 52.9, 96 66.9 /
// 54.6; MXFP4 m = 16 18.2 / 19.3, 64 22.3 / 23.2, 96 28.6 / 25.5; dense MXFP4, N =
// K = 4096, 192 rows (96 small tiles) 8.8 / 11.2.
inline bool small_tiles(int64_t rows, int64_t groups, int64_t N, bool grouped) {
  const int64_t bound = (ceil_div(rows, 64) + (grouped ? std::min(groups, rows) : 0)) * ceil_div(N, 128);
  return rows <= 64 * groups || bound <= num_sms();
}

// Sets p.tiles_w for weight tiles of `wt` columns and gives an upper bound of
// the tiles (at most one partly filled row tile a group, and the rows behind
// the last), or 0 with the error set.
inline long long bound_tiles(ExpertsParams& p, int bn, int wt) {
  p.tiles_w = static_cast<int>(ceil_div(p.N, wt));
  const long long tiles =
      (ceil_div(p.rows, bn) + std::min<long long>(p.groups, p.rows) + 1) * static_cast<long long>(p.tiles_w);
  if (tiles <= (1ll << 30)) return tiles;
  set_error("grouped product: too many tiles");
  return 0;
}

template <int KIND, int BN>
int launch_experts(const CUtensorMap& mw, const CUtensorMap& mx, const CUtensorMap& mx64,
                   const CUtensorMap& msw, const CUtensorMap& msx, ExpertsParams& p, cudaStream_t stream) {
  using Cfg = ExpCfg<KIND, BN>;
  const long long tiles = bound_tiles(p, BN, 128);
  if (!tiles) return TRNBLAS_ERR_ARG;
  auto kern = experts_kernel<KIND, BN>;
  static bool attr_set[64] = {};
  if (int rc = smem_attribute(reinterpret_cast<const void*>(kern), Cfg::SMEM, attr_set)) return rc;
  const int grid = static_cast<int>(std::min<long long>(tiles, num_sms()));
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = p.after_quantise ? 1 : 0;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaError_t e =
      cudaLaunchKernelEx(&cfg, kern, mw, mx, mx64, msw, msx, static_cast<const ExpertsParams>(p));
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "grouped product kernel launch");
}

// Clusters of two CTAs, as many as can be resident at once (a cluster's CTAs
// wait for one another only).
template <int KIND, int BN, int NBUF>
int launch_experts_pair(const CUtensorMap& mw, const CUtensorMap& mx, const CUtensorMap& mx32,
                        const CUtensorMap& msw, const CUtensorMap& msx, ExpertsParams& p,
                        cudaStream_t stream) {
  using Cfg = ExpPairCfg<KIND, BN, NBUF>;
  const long long tiles = bound_tiles(p, BN, 256);
  if (!tiles) return TRNBLAS_ERR_ARG;
  auto kern = experts_pair_kernel<KIND, BN, NBUF>;
  static bool attr_set[64] = {};
  static int max_pairs[64] = {};
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pair_config(attr, Cfg::THREADS, Cfg::SMEM, stream, p.after_quantise != 0);
  if (int rc = smem_attribute(reinterpret_cast<const void*>(kern), Cfg::SMEM, attr_set)) return rc;
  int pairs = 0;
  if (int rc = resident_pairs(kern, cfg, max_pairs, pairs)) return rc;
  cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<long long>(tiles, pairs)), 1, 1);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mw, mx, mx32, msw, msx, static_cast<const ExpertsParams>(p));
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "grouped product pair kernel launch");
}

}  // namespace tb
