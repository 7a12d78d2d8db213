// Microscaled 4-bit floating point (OCP MX: E2M1 values in blocks of 32 along
// K, one E8M0 power of two each): quantisation, its inverse, and the products
// of two quantised operands, dense and grouped by expert.
//
// A quantised operand of `rows` x K:
//   data    rows x ldq bytes, two values a byte (the even one in the low half),
//           K padded to a multiple of 32 with zeros, ldq a multiple of 16;
//   scales  blocks of 128 rows x 128 K, [row block][ceil(K / 128)][512 bytes]:
//           the word of a row's four E8M0 bytes (zero past K) at 16 * (r % 32)
//           + 4 * (r / 32 % 4), as the tensor core's copy wants them. Every
//           matrix of a stack starts a block of its own.
#include <algorithm>

#include "experts_host.hpp"
#include "mxfp4_convert.cuh"
#include "mxfp4_token_sm100.cuh"

namespace tb {
namespace {

// Which rows a scale block holds: local rows 0 .. limit - 1 at `base` + local.
struct BlockRows {
  long long base;
  int local0, limit;
};

__device__ __forceinline__ BlockRows stack_block(int blk, int rows, int per_matrix) {
  const int m = blk / per_matrix;
  return {static_cast<long long>(m) * rows, (blk - m * per_matrix) * 128, rows};
}

// Groups' blocks (group table in shared memory); limit 0 behind the last one.
__device__ __forceinline__ BlockRows group_block(const GroupTable& tb, int groups, int blk) {
  if (blk >= tb.blk0[groups]) return {0, 0, 0};
  int lo = 0, hi = groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tb.blk0[mid] <= blk) lo = mid;
    else hi = mid;
  }
  return {tb.row0[lo], (blk - tb.blk0[lo]) * 128, tb.row0[lo + 1] - tb.row0[lo]};
}

struct GroupArgs {
  const void* sizes;  // nullptr: a stack of matrices of `rows` rows
  int sizes64, groups, rows;
  int* status;
};

// The group table of a quantising or regrouping block (all threads).
__device__ __forceinline__ GroupTable block_table(int* mem, const GroupArgs& ga) {
  GroupTable tb{mem, nullptr, mem + kMaxGroups + 2};
  if (threadIdx.x < 32) build_groups(tb, ga.sizes, ga.sizes64, ga.groups, ga.rows, 0, 0, ga.status);
  __syncthreads();
  return tb;
}

// A warp takes 4 rows x 256 values, its lanes 8 neighbouring values of a row
// each: 16-byte loads, four in flight and the next chunk's behind them, and
// 128-byte stores. Blocks walk K with stride gridDim.y. Bounded by the read of X.
//
// A stack's rows lie 32 apart in a warp: their scale words are neighbours, and
// the eight warps of a block hold neighbouring ones, so a K block's words leave
// as 128 contiguous bytes. Rows grouped by expert (GROUPED) are taken in their
// own order, 32 to a block, and each word goes to its group's blocks: the first
// loads do not wait for the scan of the sizes, and short groups make no empty
// blocks (64 rows of 32 groups x 4096: 14 us by blocks of the groups, 5 so).
template <typename T, bool GROUPED>
__global__ void __launch_bounds__(256)
    mxfp4_quantize_kernel(const T* __restrict__ X, long long ldx, GroupArgs ga, int per_matrix, int K, int vec,
                          uint8_t* __restrict__ data, long long ldq, uint32_t* __restrict__ scales) {
  __shared__ int mem[GROUPED ? 2 * (kMaxGroups + 2) : 1];
  launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kwords = (K + 127) >> 7;
  const int blk = blockIdx.x >> 2;
  const int l32 = (blockIdx.x & 3) * 8 + warp;  // a stack's row % 32
  bool ok[4];
  long long row[4];
  if constexpr (GROUPED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long r = static_cast<long long>(blockIdx.x) * 32 + warp * 4 + i;
      ok[i] = r < ga.rows;
      row[i] = ok[i] ? r : 0;
    }
  } else {
    const BlockRows br = stack_block(blk, ga.rows, per_matrix);
    const int l0 = br.local0 + l32;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ok[i] = l0 + 32 * i < br.limit;
      row[i] = ok[i] ? br.base + l0 + 32 * i : br.base;
    }
  }
  const int kstep = gridDim.y * 256;
  int k = blockIdx.y * 256 + lane * 8;
  Raw8<T> cur[4], nxt[4];
  auto fetch = [&](Raw8<T> (&dst)[4], int at) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      dst[i] = load8(X + row[i] * ldx + (at < K ? at : 0), ok[i] ? K - at : 0, vec);
  };
  fetch(cur, k);
  long long word_at[4];  // GROUPED: each row's first word (K block 0), -1 behind the last group
  if constexpr (GROUPED) {
    const GroupTable tb = block_table(mem, ga);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = static_cast<int>(row[i]);
      int lo = 0, hi = ga.groups;  // row0[lo] <= r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tb.row0[mid] <= r) lo = mid;
        else hi = mid;
      }
      const int l = r - tb.row0[lo];
      word_at[i] = ok[i] && r < tb.row0[ga.groups]
                       ? static_cast<long long>(tb.blk0[lo] + (l >> 7)) * kwords * 128 + (l & 31) * 4 + ((l >> 5) & 3)
                       : -1;
    }
  }
  for (; k - lane * 8 < K; k += kstep) {
    if (k - lane * 8 + kstep < K) fetch(nxt, k + kstep);  // in flight while this chunk is converted
    uint32_t word[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t s;
      const uint32_t w = quantize8<T>(cur[i], s);
      // up to K's last block: what follows in a longer row stride is not the row's
      if (ok[i] && (k & ~31) < K) *reinterpret_cast<uint32_t*>(data + row[i] * ldq + (k >> 1)) = w;
      // the four scale bytes of 16 lanes; zero past K's last block
      if ((k & ~31) >= K || !ok[i]) s = 0;
      uint32_t b = s << (8 * ((lane >> 2) & 3));
      b |= __shfl_xor_sync(0xffffffffu, b, 4);
      b |= __shfl_xor_sync(0xffffffffu, b, 8);
      word[i] = b;
    }
    const int kw = k >> 7;
    if ((lane & 15) == 0 && kw < kwords) {
      if constexpr (GROUPED) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (word_at[i] >= 0) scales[word_at[i] + static_cast<long long>(kw) * 128] = word[i];
      } else {
        reinterpret_cast<uint4*>(scales)[(static_cast<long long>(blk) * kwords + kw) * 32 + l32] =
            make_uint4(word[0], word[1], word[2], word[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) cur[i] = nxt[i];
  }
}

// The scales of rows held as one matrix, in blocks that start with the groups.
// One thread per 16 bytes of the result.
__global__ void __launch_bounds__(256)
    mxfp4_regroup_kernel(const uint32_t* __restrict__ src, GroupArgs ga, int kwords, uint4* __restrict__ dst) {
  __shared__ int mem[2 * (kMaxGroups + 2)];
  const GroupTable tb = block_table(mem, ga);
  const int blk = blockIdx.x;
  const BlockRows br = group_block(tb, ga.groups, blk);
  if (br.limit == 0) return;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < kwords * 32; i += gridDim.y * 256) {
    const int kw = i >> 5, l32 = i & 31;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int l = br.local0 + l32 + 32 * j;
      const long long r = br.base + l;
      w[j] = l < br.limit ? __ldg(src + ((r >> 7) * kwords + kw) * 128 + (r & 31) * 4 + ((r >> 5) & 3)) : 0u;
    }
    dst[(static_cast<long long>(blk) * kwords + kw) * 32 + l32] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Two E2M1 codes (the low byte of c, the earlier in its low half) as bf16 bits:
// a code s ee m is the bf16 number with these bits at the sign, the low
// exponent and the top mantissa places, times 2^126 (subnormals included), so no
// table is read.
__device__ __forceinline__ uint32_t e2m1x2_bits(uint32_t c) {
  const uint32_t y = (c & 0xFu) | ((c & 0xF0u) << 12);
  return ((y & 0x00070007u) << 6) | ((y & 0x00080008u) << 12);
}

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }

// 8 values of codes w in units of 2^(s - 127). bf16 holds every product of a
// 2-bit mantissa and a power of two down to 2^-133 exactly, so the two
// multiplications (by 2^126, by the unit: subnormal for s = 0, NaN for s = 255)
// are exact in pairs of bf16; fp32 and fp16 are taken from there, fp16 with its
// own rounding. (Units above 2^125 overflow to infinities where fp32 does.)
template <typename T>
__device__ __forceinline__ void dequantize8(uint32_t w, uint32_t s, T (&out)[8]) {
  const uint32_t ub = s == 255 ? 0x7FC0u : (s == 0 ? 0x0040u : s << 7);
  const __nv_bfloat162 unit = as_bf162(ub | (ub << 16)), big = as_bf162(0x7E807E80u);  // 2^126
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 v = __hmul2(__hmul2(as_bf162(e2m1x2_bits((w >> (8 * j)) & 0xFFu)), big), unit);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      reinterpret_cast<__nv_bfloat162*>(out)[j] = v;
    } else {
      const float2 f = __bfloat1622float2(v);
      if constexpr (std::is_same<T, float>::value) {
        out[2 * j] = f.x;
        out[2 * j + 1] = f.y;
      } else {
        out[2 * j] = __float2half_rn(f.x);
        out[2 * j + 1] = __float2half_rn(f.y);
      }
    }
  }
}

// 8 values a lane, 4 rows a warp as in the quantiser. Bounded by the write.
template <typename T>
__global__ void __launch_bounds__(256)
    mxfp4_dequantize_kernel(const uint8_t* __restrict__ data, long long ldq,
                            const uint4* __restrict__ scales, int rows, int per_matrix, int K, int vec,
                            T* __restrict__ Y, long long ldy) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blk = blockIdx.x >> 2;
  const BlockRows br = stack_block(blk, rows, per_matrix);
  const int l32 = (blockIdx.x & 3) * 8 + warp;
  const int l0 = br.local0 + l32;
  const int kwords = (K + 127) >> 7;
  if (l0 >= br.limit) return;
  for (int k = blockIdx.y * 256 + lane * 8; k < K; k += gridDim.y * 256) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = l0 + 32 * i < br.limit
                 ? __ldg(reinterpret_cast<const uint32_t*>(data + (br.base + l0 + 32 * i) * ldq + (k >> 1)))
                 : 0;
    const uint4 s4 = __ldg(scales + (static_cast<long long>(blk) * kwords + (k >> 7)) * 32 + l32);
    const uint32_t sw[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (l0 + 32 * i >= br.limit) break;
      const uint32_t s = (sw[i] >> (8 * ((k >> 5) & 3))) & 0xFFu;
      alignas(16) T out[8];
      dequantize8<T>(w[i], s, out);
      T* dst = Y + (br.base + l0 + 32 * i) * ldy + k;
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
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_mx(const char* what, int64_t rows, int64_t K, int64_t ldq) {
  // (a thread's place along K stays an int one stride past the end)
  if (rows < 0 || K < 0 || rows > (1ll << 31) - 512 || K > (1ll << 30)) {
    set_error(std::string(what) + ": rows must be in [0, 2^31 - 512], K in [0, 2^30]");
    return TRNBLAS_ERR_ARG;
  }
  if (ldq < round_up(K, 32) / 2 || ldq % 16) {
    set_error(std::string(what) + ": a row of packed values takes round_up(K, 32) / 2 bytes at a stride of a multiple of 16");
    return TRNBLAS_ERR_ARG;
  }
  return TRNBLAS_OK;
}

int check_mx_gemm(int out_dtype, int64_t rows, int64_t groups, int64_t N, int64_t K, const void* A, int64_t lda,
                  const void* scalesA, const void* B, int64_t ldb, const void* scalesB, const void* group_sizes,
                  float beta, const void* C, int64_t ldc, const void* D, int64_t ldd) {
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
  if (K == 0 || groups == 0) return TRNBLAS_OK;
  if (int rc = check_mx("trnblas_mxfp4_gemm (A)", rows, K, lda)) return rc;
  if (int rc = check_mx("trnblas_mxfp4_gemm (B)", N, K, ldb)) return rc;
  if (!A || !B || !scalesA || !scalesB || !al16(scalesA) || !al16(scalesB)) {
    set_error("trnblas_mxfp4_gemm: NULL operand, or scales not on 16 bytes");
    return TRNBLAS_ERR_ARG;
  }
  return TRNBLAS_OK;
}

// Thread blocks along K: about four chunks of 256 each, so that a block has the
// next chunk in flight behind the one it converts; one each where that leaves
// less than two blocks an SM.
unsigned k_blocks(long long xblocks, long long K) {
  const long long chunks = ceil_div(K, 256), y = ceil_div(chunks, 4);
  return static_cast<unsigned>(std::min<long long>(xblocks * y < 2ll * num_sms() ? chunks : y, 65535));
}

template <bool GROUPED>
int launch_quantize(int dtype, const GroupArgs& ga, long long xblocks, int per_matrix, int64_t K, const void* X,
                    int64_t ldx, void* data, int64_t ldq, void* scales, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(xblocks), k_blocks(xblocks, K));
  const int vec = al16(X) && (ldx * (dtype == TRNBLAS_F32 ? 4 : 2)) % 16 == 0;
  uint8_t* q = static_cast<uint8_t*>(data);
  uint32_t* s = static_cast<uint32_t*>(scales);
  const int k = static_cast<int>(K);
  if (dtype == TRNBLAS_F32)
    mxfp4_quantize_kernel<float, GROUPED>
        <<<grid, 256, 0, stream>>>(static_cast<const float*>(X), ldx, ga, per_matrix, k, vec, q, ldq, s);
  else if (dtype == TRNBLAS_BF16)
    mxfp4_quantize_kernel<__nv_bfloat16, GROUPED>
        <<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16*>(X), ldx, ga, per_matrix, k, vec, q, ldq, s);
  else
    mxfp4_quantize_kernel<__half, GROUPED>
        <<<grid, 256, 0, stream>>>(static_cast<const __half*>(X), ldx, ga, per_matrix, k, vec, q, ldq, s);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "mxfp4 quantise kernel launch");
}

bool kernel_dtype(int dtype) { return dtype == TRNBLAS_F32 || dtype == TRNBLAS_BF16 || dtype == TRNBLAS_F16; }

int check_quantize(const char* what, int dtype, int64_t matrices, int64_t rows, int64_t K, const void* X, int64_t ldx,
                   const void* data, int64_t ldq, const void* scales) {
  const std::string w(what);
  if (!kernel_dtype(dtype)) {
    set_error(w + ": dtype must be F32, BF16 or F16");
    return TRNBLAS_ERR_ARG;
  }
  if (int rc = check_mx(what, rows, K, ldq)) return rc;
  if (matrices < 0 || (matrices > 0 && matrices * ceil_div(rows, 128) > (1ll << 28))) {
    set_error(w + ": too many rows");
    return TRNBLAS_ERR_ARG;
  }
  if (matrices == 0 || rows == 0 || K == 0) return TRNBLAS_OK;
  if (!X || !data || !scales || ldx < K || !al16(data) || !al16(scales)) {
    set_error(w + ": NULL or unaligned operand (16 bytes for data and scales), or a row stride smaller than K");
    return TRNBLAS_ERR_ARG;
  }
  return TRNBLAS_OK;
}

size_t scale_bytes(int64_t rows, int64_t groups, int64_t K) {
  return static_cast<size_t>(ceil_div(rows, 128) + groups) * ceil_div(K, 128) * 512;
}

// A few rows of a dense product go to the kernel that quantises them itself.
bool token_path(int64_t rows, int64_t K, bool grouped) {
  return !grouped && rows <= TokenCfg::ROWS && ceil_div(K, 256) <= TokenCfg::MAX_KB * TokenCfg::MAX_SPLIT;
}

int launch_token(int a_dtype, int out_dtype, int64_t rows, int64_t N, int64_t K, float alpha, const void* X,
                 int64_t ldx, const void* B, int64_t ldb, const void* scalesB, float beta, const void* C,
                 int64_t ldc, void* D, int64_t ldd, cudaStream_t stream) {
  using Cfg = TokenCfg;
  const int64_t kw = ceil_div(K, 128), kb = ceil_div(K, 256), tiles = ceil_div(N, 128);
  CUtensorMap mw, msw;
  const uint64_t dims[3] = {128, static_cast<uint64_t>(kw), static_cast<uint64_t>(tiles)};
  const uint64_t strides[2] = {128, 128 * static_cast<uint64_t>(kw)};
  const uint32_t box[3] = {128, 2, 1};
  if (!encode_map_3d(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, B, round_up(K, 32) / 2, N, 1, ldb, ldb * N, 128, 128) ||
      !encode_map(&msw, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, scalesB, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE))
    return TRNBLAS_ERR_ALIGN;
  // K over enough CTAs to occupy the SMs once, at least two blocks of it each,
  // and at most what a CTA holds
  int split = 1;
  while (split < Cfg::MAX_SPLIT &&
         (ceil_div(kb, split) > Cfg::MAX_KB || (tiles * split * 2 <= num_sms() && kb >= 4 * split)))
    split *= 2;
  TokenParams p{};
  p.X = X;
  p.ldx = ldx;
  p.vec = al16(X) && (ldx * (a_dtype == TRNBLAS_F32 ? 4 : 2)) % 16 == 0;
  p.rows = static_cast<int>(rows);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.kb_per_cta = static_cast<int>(ceil_div(kb, split));
  p.alpha = alpha;
  p.beta = beta;
  p.out_kind = out_kind_of(out_dtype);
  p.C = C;
  p.ldc = ldc;
  p.D = D;
  p.ldd = ldd;
  p.status = status_word();
  if (!p.status) return TRNBLAS_ERR_CUDA;
  p.timeout_ns = wait_timeout_ns();
  const int smem = Cfg::smem(p.kb_per_cta, split);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(split);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * split), 1, 1);
  cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto launch = [&](auto kern, bool (&done)[64]) {
    if (int rc = smem_attribute(reinterpret_cast<const void*>(kern), Cfg::smem(Cfg::MAX_KB, Cfg::MAX_SPLIT), done))
      return rc;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mw, msw, static_cast<const TokenParams>(p));
    return e == cudaSuccess ? static_cast<int>(TRNBLAS_OK) : cuda_fail(e, "mxfp4 token kernel launch");
  };
  static bool done[3][64] = {};
  if (a_dtype == TRNBLAS_F32) return launch(mxfp4_token_kernel<float>, done[0]);
  if (a_dtype == TRNBLAS_BF16) return launch(mxfp4_token_kernel<__nv_bfloat16>, done[1]);
  return launch(mxfp4_token_kernel<__half>, done[2]);
}

// The product on data and scales in place (with group sizes the rows' scales
// start a block with every group). `after_quantise`: the launch before it in the
// stream is the quantiser, which lets this kernel set up while it runs.
int launch_mx_gemm(int out_dtype, int64_t rows, int64_t groups, int64_t N, int64_t K, float alpha, const void* A,
                   int64_t lda, const void* scalesA, const void* B, int64_t ldb, const void* scalesB,
                   const void* group_sizes, int sizes_64, float beta, const void* C, int64_t ldc, void* D,
                   int64_t ldd, bool after_quantise, cudaStream_t stream) {
  const auto dt = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const uint64_t kb = static_cast<uint64_t>(round_up(K, 32) / 2);
  const bool small = small_tiles(rows, groups, N, group_sizes != nullptr);
  const bool pair = !small && N > 128;
  // Pair tiles of 192 rows: two accumulators and the scales of five stages fill
  // TMEM. Where those need a second wave of pairs and tiles of 256 with one
  // accumulator do not, take these (dense: 777 rows x 4096 x 4010, 80 tiles of
  // 192 against 64 of 256 on 74 pairs: 16.6 against 13.4 us).
  const int64_t wt = ceil_div(N, 256), pairs = num_sms() / 2;
  const bool one_wave = pair && !group_sizes && ceil_div(rows, 192) * wt > pairs && ceil_div(rows, 256) * wt <= pairs;
  const uint32_t xbox = small ? 64 : !pair ? 192 : one_wave ? 128 : 96;
  const uint64_t kw = static_cast<uint64_t>(ceil_div(K, 128));
  const uint64_t wb = static_cast<uint64_t>(ceil_div(N, 128));
  auto scale_map = [&](CUtensorMap* m, const void* base, uint64_t blocks, uint32_t box_blocks) {
    const uint64_t dims[3] = {128, kw, blocks};
    const uint64_t strides[2] = {128, 128 * kw};
    const uint32_t box[3] = {128, 2, box_blocks};
    return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, base, 3, dims, strides, box,
                      CU_TENSOR_MAP_SWIZZLE_NONE);
  };
  CUtensorMap mw, mx, mxs, msw, msx;
  if (!encode_map_3d(&mw, dt, 1, B, kb, N, groups, ldb, ldb * N, 128, 128) ||
      !encode_map_3d(&mx, dt, 1, A, kb, rows, 1, lda, lda * rows, 128, xbox) ||
      !encode_map_3d(&mxs, dt, 1, A, kb, rows, 1, lda, lda * rows, 128, pair ? 32 : small ? 16 : 64) ||
      !scale_map(&msw, scalesB, wb * groups, 1) ||
      !scale_map(&msx, scalesA, ceil_div(rows, 128) + (group_sizes ? groups : 0), small ? 1 : 2))
    return TRNBLAS_ERR_ALIGN;
  ExpertsParams p{};
  if (int rc = fill_experts(p, out_dtype, rows, groups, N, K, alpha, group_sizes, sizes_64, beta, C, ldc, D, ldd))
    return rc;
  p.w_blocks = static_cast<int>(wb);
  p.after_quantise = after_quantise;
  if (small) return launch_experts<kExpMx4, 64>(mw, mx, mxs, msw, msx, p, stream);
  if (one_wave) return launch_experts_pair<kExpMx4, 256, 1>(mw, mx, mxs, msw, msx, p, stream);
  if (pair) return launch_experts_pair<kExpMx4, 192, 2>(mw, mx, mxs, msw, msx, p, stream);
  return launch_experts<kExpMx4, 192>(mw, mx, mxs, msw, msx, p, stream);
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" {

int trnblas_mxfp4_quantize(int dtype, int64_t matrices, int64_t rows, int64_t K, const void* X, int64_t ldx,
                           void* data, int64_t ldq, void* scales, void* stream) {
  if (int rc = check_quantize("trnblas_mxfp4_quantize", dtype, matrices, rows, K, X, ldx, data, ldq, scales)) return rc;
  if (matrices == 0 || rows == 0 || K == 0) return TRNBLAS_OK;
  GroupArgs ga{};
  ga.rows = static_cast<int>(rows);
  const int per = static_cast<int>(ceil_div(rows, 128));
  return launch_quantize<false>(dtype, ga, matrices * per * 4, per, K, X, ldx, data, ldq, scales,
                                static_cast<cudaStream_t>(stream));
}

int trnblas_mxfp4_dequantize(int dtype, int64_t matrices, int64_t rows, int64_t K, const void* data, int64_t ldq,
                             const void* scales, void* Y, int64_t ldy, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (int rc = check_quantize("trnblas_mxfp4_dequantize", dtype, matrices, rows, K, Y, ldy, data, ldq, scales))
    return rc;
  if (matrices == 0 || rows == 0 || K == 0) return TRNBLAS_OK;
  const int per = static_cast<int>(ceil_div(rows, 128));
  const long long blocks = matrices * per * 4;
  const dim3 grid(static_cast<unsigned>(blocks), k_blocks(blocks, K));
  const int vec = al16(Y) && (ldy * (dtype == TRNBLAS_F32 ? 4 : 2)) % 16 == 0;
  const uint8_t* q = static_cast<const uint8_t*>(data);
  const uint4* s = static_cast<const uint4*>(scales);
  const int r = static_cast<int>(rows), k = static_cast<int>(K);
  if (dtype == TRNBLAS_F32)
    mxfp4_dequantize_kernel<float><<<grid, 256, 0, stream>>>(q, ldq, s, r, per, k, vec, static_cast<float*>(Y), ldy);
  else if (dtype == TRNBLAS_BF16)
    mxfp4_dequantize_kernel<__nv_bfloat16>
        <<<grid, 256, 0, stream>>>(q, ldq, s, r, per, k, vec, static_cast<__nv_bfloat16*>(Y), ldy);
  else
    mxfp4_dequantize_kernel<__half><<<grid, 256, 0, stream>>>(q, ldq, s, r, per, k, vec, static_cast<__half*>(Y), ldy);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TRNBLAS_OK : cuda_fail(e, "mxfp4 dequantise kernel launch");
}

size_t trnblas_mxfp4_gemm_workspace_size(int64_t rows, int64_t groups, int64_t K, int grouped) {
  if (rows <= 0 || groups <= 0 || K <= 0 || !grouped) return 0;
  return scale_bytes(rows, groups, K);
}

int trnblas_mxfp4_gemm(int out_dtype, int64_t rows, int64_t groups, int64_t N, int64_t K, float alpha,
                       const void* A, int64_t lda, const void* scalesA, const void* B, int64_t ldb,
                       const void* scalesB, const void* group_sizes, int sizes_64, float beta, const void* C,
                       int64_t ldc, void* D, int64_t ldd, void* workspace, size_t workspace_bytes,
                       void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (int rc = check_mx_gemm(out_dtype, rows, groups, N, K, A, lda, scalesA, B, ldb, scalesB, group_sizes, beta, C,
                             ldc, D, ldd))
    return rc;
  if (rows == 0 || N == 0) return TRNBLAS_OK;
  if (K == 0 || groups == 0)
    return trnblas_gemm(out_dtype, 1, rows, N, 0, alpha, nullptr, 1, 0, 0, nullptr, N, 0, 0, beta, C, ldc, 0,
                        D, ldd, 0, nullptr, 0, stream_);
  if (group_sizes) {
    if (!workspace || !al16(workspace) || workspace_bytes < scale_bytes(rows, groups, K)) {
      set_error("trnblas_mxfp4_gemm: grouped needs " + std::to_string(scale_bytes(rows, groups, K)) +
                " workspace bytes, 16-byte aligned");
      return TRNBLAS_ERR_WORKSPACE;
    }
    GroupArgs ga{group_sizes, sizes_64, static_cast<int>(groups), static_cast<int>(rows), status_word()};
    if (!ga.status) return TRNBLAS_ERR_CUDA;
    const int kw = static_cast<int>(ceil_div(K, 128));
    const dim3 grid(static_cast<unsigned>(ceil_div(rows, 128) + groups),
                    static_cast<unsigned>(std::min<long long>(ceil_div(kw, 8), 65535)));
    mxfp4_regroup_kernel<<<grid, 256, 0, stream>>>(static_cast<const uint32_t*>(scalesA), ga, kw,
                                                   static_cast<uint4*>(workspace));
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e, "mxfp4 regroup kernel launch");
    scalesA = workspace;
  }
  return launch_mx_gemm(out_dtype, rows, groups, N, K, alpha, A, lda, scalesA, B, ldb, scalesB, group_sizes,
                        sizes_64, beta, C, ldc, D, ldd, false, stream);
}

size_t trnblas_mxfp4_gemm_x_workspace_size(int64_t rows, int64_t groups, int64_t K, int grouped) {
  if (rows <= 0 || groups <= 0 || K <= 0 || token_path(rows, K, grouped)) return 0;
  // packed values, then the scale blocks
  return static_cast<size_t>(rows) * (round_up(K, 32) / 2) + scale_bytes(rows, grouped ? groups : 0, K);
}

int trnblas_mxfp4_gemm_x(int a_dtype, int out_dtype, int64_t rows, int64_t groups, int64_t N, int64_t K,
                         float alpha, const void* X, int64_t ldx, const void* B, int64_t ldb,
                         const void* scalesB, const void* group_sizes, int sizes_64, float beta, const void* C,
                         int64_t ldc, void* D, int64_t ldd, void* workspace, size_t workspace_bytes,
                         void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (!kernel_dtype(a_dtype)) {
    set_error("trnblas_mxfp4_gemm_x: a_dtype must be F32, BF16 or F16");
    return TRNBLAS_ERR_ARG;
  }
  if (int rc = check_group_dims("trnblas_mxfp4_gemm_x", rows, groups, N, K)) return rc;
  const int64_t ldq = round_up(K, 32) / 2;
  uint8_t* data = static_cast<uint8_t*>(workspace);
  uint8_t* scales = data ? data + rows * ldq : nullptr;
  if (rows == 0 || N == 0 || K == 0 || groups == 0)
    return trnblas_mxfp4_gemm(out_dtype, rows, groups, N, K, alpha, X, ldq, X, B, ldb, scalesB, group_sizes, sizes_64,
                              beta, C, ldc, D, ldd, workspace, workspace_bytes, stream_);
  if (token_path(rows, K, group_sizes != nullptr)) {
    // (the checks on A's pointers: X stands for them)
    if (!X || ldx < K) {
      set_error("trnblas_mxfp4_gemm_x: NULL X, or ldx smaller than K");
      return TRNBLAS_ERR_ARG;
    }
    if (int rc = check_mx_gemm(out_dtype, rows, groups, N, K, B, ldq, scalesB, B, ldb, scalesB, group_sizes, beta, C,
                               ldc, D, ldd))
      return rc;
    return launch_token(a_dtype, out_dtype, rows, N, K, alpha, X, ldx, B, ldb, scalesB, beta, C, ldc, D, ldd, stream);
  }
  const size_t need = trnblas_mxfp4_gemm_x_workspace_size(rows, groups, K, group_sizes != nullptr);
  if (!workspace || !al16(workspace) || workspace_bytes < need) {
    set_error("trnblas_mxfp4_gemm_x: needs " + std::to_string(need) + " workspace bytes, 16-byte aligned");
    return TRNBLAS_ERR_WORKSPACE;
  }
  if (int rc = check_mx_gemm(out_dtype, rows, groups, N, K, data, ldq, scales, B, ldb, scalesB, group_sizes, beta, C,
                             ldc, D, ldd))
    return rc;
  if (int rc = check_quantize("trnblas_mxfp4_gemm_x", a_dtype, 1, rows, K, X, ldx, data, ldq, scales)) return rc;
  GroupArgs ga{group_sizes, sizes_64, static_cast<int>(groups), static_cast<int>(rows), status_word()};
  if (!ga.status) return TRNBLAS_ERR_CUDA;
  const int per = static_cast<int>(ceil_div(rows, 128));
  if (int rc = group_sizes
                   ? launch_quantize<true>(a_dtype, ga, ceil_div(rows, 32), per, K, X, ldx, data, ldq, scales, stream)
                   : launch_quantize<false>(a_dtype, ga, per * 4, per, K, X, ldx, data, ldq, scales, stream))
    return rc;
  return launch_mx_gemm(out_dtype, rows, groups, N, K, alpha, data, ldq, scales, B, ldb, scalesB, group_sizes,
                        sizes_64, beta, C, ldc, D, ldd, true, stream);
}

}  // extern "C"
