// Products grouped by expert, sm_100a: rows of A that belong to group g
// multiply matrix g of a stack of weights, groups of any length.
//
//   forward  D[r] = alpha * A[r] op(W[g]) + beta * C[r]     (experts_kernel)
//   wgrad    D[g] = alpha * A_g^T B_g + beta * C[g]         (experts_wgrad_sm100.cuh)
//
// The group sizes are read on the device: every CTA scans them once into a
// table of first rows and first tiles in shared memory (G <= kMaxGroups), then
// walks its tiles with a static stride. Sizes below zero count as zero and
// rows past the operand's end are cut off (recorded in the status word), so no
// index leaves the operands whatever the sizes hold.
//
// Forward: the weights are the M side of the MMA (128 of their output columns
// on the 128 TMEM lanes) and the rows of A the N side. An MMA's time goes with
// N, which may be any multiple of 16, so a group of m rows costs
// round_up(m, 16) whatever the tile size: groups of one row and of thousands
// run on the same kernel, and a group's rows are cut into equal tiles instead
// of full ones and a remainder. The epilogue turns 32 x 32 blocks through
// shared memory, since TMEM lanes run along a row of D.
//
// Operand kinds of the forward kernel:
//   kExpF16  bf16 / fp16, fp32 accumulate; weights stored N x K (K-major) or
//            K x N (MN-major), no transposed copy;
//   kExpMx4  E2M1 pairs with one power of two per 32 values along K
//            (kind::mxf4, block scaled by the tensor core). The scales lie in
//            blocks of 128 rows x 128 K (512 bytes) in the order that tcgen05.cp
//            copies to TMEM, the word of a row's four blocks at 16 * (row % 32)
//            + 4 * (row / 32 % 4), so TMA brings them with the operands. Groups
//            start at any row, but their scales at a block of their own; a
//            tile starts at a multiple of 64 rows of its group. Each pipeline
//            stage has its own TMEM scale columns, which its empty barrier frees
//            with the stage. (Scale words in row order, brought and reordered
//            by warps of the kernel, cost 2.4 times the time at 8192^3 on CTA
//            pairs, 470 us against 197: their loads, proxy fences and arrivals
//            were the slowest part of every stage.)
#pragma once

#include "gemm_sm100.cuh"

namespace tb {

enum ExpKind : int { kExpF16 = 0, kExpMx4 = 1 };
constexpr int kMaxGroups = 1024;
constexpr int kExpBlockBytes = 2048;  // an epilogue warp's block in shared memory
constexpr int kGroupTableBytes = (kMaxGroups + 2) * 12;

struct GroupTable {
  int* row0;   // [G + 2] first row of each group; [G] the rows behind the last group, [G + 1] rows
  int* tile0;  // [G + 2] first tile; [G + 1] all tiles
  int* blk0;   // [G + 1] first scale block (of 128 rows), kExpMx4
};

struct ExpertsParams {
  int rows, N, K;
  int groups;
  const void* sizes;  // device, int32 or int64; nullptr: one group of all rows
  int sizes64;
  int in_fmt;   // kExpF16: kFmtBF16 / kFmtF16
  int w_mn;     // kExpF16: weights stored K x N (2: read in boxes of 128 columns)
  int w_shared; // kExpF16: one matrix for every group
  int out_kind;
  float alpha, beta;
  const void* C;
  long long ldc;
  void* D;
  long long ldd;
  int tiles_w;  // weight tiles of 128
  int w_blocks;  // kExpMx4: scale blocks of one weight matrix
  int after_quantise;  // launched beside the kernel that writes the rows
  int* status;
  unsigned long long timeout_ns;
};

__device__ __forceinline__ long long load_size(const void* sizes, int sizes64, int g) {
  return sizes64 ? __ldg(reinterpret_cast<const long long*>(sizes) + g)
                 : static_cast<long long>(__ldg(reinterpret_cast<const int*>(sizes) + g));
}

// One warp: the first row of every group, the first tile with `bn` rows to a
// tile at most and `per` tiles for each of them (bn 0: none), and the first
// scale block (tb.blk0 null: none).
__device__ __forceinline__ void build_groups(const GroupTable& tb, const void* sizes, int sizes64,
                                             int groups, int rows, int bn, int per, int* status) {
  const int lane = threadIdx.x & 31;
  long long run = 0;
  int tiles = 0, blocks = 0;
  bool bad = false;
  for (int base = 0; base < groups; base += 32) {
    const int g = base + lane;
    long long s = 0;
    if (g < groups) s = sizes ? load_size(sizes, sizes64, g) : rows;
    bad |= s < 0;
    s = s < 0 ? 0 : (s > rows ? static_cast<long long>(rows) + 1 : s);
    long long inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const long long end = run + inc;
    const int hi = static_cast<int>(end < rows ? end : rows);
    const int lo = static_cast<int>(end - s < rows ? end - s : rows);
    const int nt = bn ? ((hi - lo + bn - 1) / bn) * per : 0;
    int tinc = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, tinc, o);
      if (lane >= o) tinc += u;
    }
    if (g < groups) {
      tb.row0[g] = lo;
      if (bn) tb.tile0[g] = tiles + tinc - nt;
    }
    if (tb.blk0) {
      const int nb = (hi - lo + 127) >> 7;
      int binc = nb;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, binc, o);
        if (lane >= o) binc += u;
      }
      if (g < groups) tb.blk0[g] = blocks + binc - nb;
      blocks += __shfl_sync(0xffffffffu, binc, 31);
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
    tiles += __shfl_sync(0xffffffffu, tinc, 31);
  }
  bad |= run > rows;
  if (__any_sync(0xffffffffu, bad) && blockIdx.x == 0 && lane == 0)
    atomicCAS(status, 0, static_cast<int>(kBadGroups));
  if (lane == 0) {
    const int end = static_cast<int>(run < rows ? run : rows);
    tb.row0[groups] = end;
    tb.row0[groups + 1] = rows;
    if (tb.blk0) tb.blk0[groups] = blocks;
    if (bn) {
      tb.tile0[groups] = tiles;
      tb.tile0[groups + 1] = tiles + ((rows - end + bn - 1) / bn) * per;
    }
  }
}

struct ExpTile {
  int g;       // group, or `groups` for the rows behind the last one
  int r0, nv;  // first row and number of rows
  int n0;      // first weight column
  int x0;      // first row within the group
};

// Tile t of the walk: within a group, bands of at most kBand row tiles; in a
// band, the row tiles of one weight block next to one another. The CTAs that
// run together then share a few weight blocks and a band's rows, and a long
// group's rows are not read from DRAM once for every weight block (16384 rows
// in one group, K = N = 4096, bf16: 351 us, without bands 444). BN: most rows of
// a tile, a multiple of STEP; WT: weight columns of a tile.
constexpr int kBand = 8;

template <int BN, int STEP = 16, int WT = 128>
__device__ __forceinline__ ExpTile exp_tile(const GroupTable& tb, int groups, int tiles_w, int t) {
  int lo = 0, hi = groups + 1;  // tile0[lo] <= t < tile0[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tb.tile0[mid] <= t) lo = mid;
    else hi = mid;
  }
  ExpTile e;
  e.g = lo;
  const int first = tb.row0[lo], m = tb.row0[lo + 1] - first;
  const int nt = (m + BN - 1) / BN;
  // equal tiles, a multiple of STEP rows each (the last one keeps the rest;
  // never empty, since nt - 1 tiles of at most BN rows do not cover m)
  const int step = ((m + nt - 1) / nt + STEP - 1) & ~(STEP - 1);
  const int i = t - tb.tile0[lo];
  const int band = i / (kBand * tiles_w), j = i - band * kBand * tiles_w;
  const int width = min(kBand, nt - band * kBand);
  const int w = j / width, x = band * kBand + j - w * width;
  e.x0 = x * step;
  e.r0 = first + e.x0;
  e.nv = min(step, m - x * step);
  e.n0 = w * WT;
  return e;
}

template <int KIND, int BN>
struct ExpCfg {
  static constexpr bool MX = KIND == kExpMx4;
  static constexpr int BK = MX ? 256 : 64;  // one 128-byte swizzle row of K
  static constexpr int W_TILE = 128 * 128;
  static constexpr int X_TILE = BN * 128;
  static constexpr int XBOX = BN == 64 ? 16 : 64;  // rows of a small box
  // rows start at a multiple of STEP in their group; with 64 a tile of 64 rows
  // lies in one scale block and one of 192 in two
  static constexpr int STEP = MX ? 64 : 16;
  static constexpr int XBLK = (BN + 127) / 128;       // scale blocks of the rows
  static_assert(!MX || BN == 64 || BN == 192, "scale blocks of a tile");
  static constexpr int SFW = MX ? 2 * 512 : 0;        // K = 256 is two blocks
  static constexpr int SFX = MX ? 2 * XBLK * 512 : 0;
  static constexpr int STAGE_BYTES = W_TILE + X_TILE + SFW + SFX;
  static_assert(STAGE_BYTES % 1024 == 0, "stages keep the swizzle atom's alignment");
  static constexpr int EPI_BYTES = 4 * kExpBlockBytes;
  // what fits beside the epilogue's blocks and the group table; at most 8
  static constexpr int FIT = (227 * 1024 - 1024 - 512 - EPI_BYTES - kGroupTableBytes) / STAGE_BYTES;
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int SF_COLS = MX ? 2 * 4 * (1 + XBLK) : 0;  // TMEM scale columns of a stage
  static constexpr int COLS = 2 * BN + STAGES * SF_COLS;
  static constexpr int TMEM_COLS = COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static_assert(COLS <= 512, "accumulators and scales fit TMEM");
  static constexpr int THREADS = 32 * 6;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + 512 + EPI_BYTES + kGroupTableBytes;
};

// Instruction descriptor of kind::mxf4 with E8M0 scales: E2M1 operands, N / 8
// at bit 17, the scale type at 23, M / 128 at 27, the scale bytes' position in
// their words (0 or 2) at bits 4 and 29.
__host__ __device__ constexpr uint32_t idesc_mx4(uint32_t N, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | (1u << 27) | (sf << 29);
}

__device__ __forceinline__ void mma_mx4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                        uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

// 32 rows x 16 bytes of shared memory into 4 TMEM columns, the same in all
// four lane quarters: the scale words of 128 rows, word of row r at lane
// r % 32, column r / 32.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

// Forward epilogue of one warp's block: lane l holds v[j] = accumulator of
// weight column n0 + l (n0: the warp's first) and row r0 + j, j < left.
__device__ __forceinline__ void exp_store(const ExpertsParams& p, int r0, int left, int n0,
                                          const float* v, void* tsm) {
  const int lane = threadIdx.x & 31;
  const int n = n0 + lane;
  const bool has_c = p.C != nullptr && p.beta != 0.0f;
  float out[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) out[j] = p.alpha * v[j];
  if (has_c && n < p.N) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < left) out[j] += p.beta * load_c(p.C, p.out_kind, (r0 + static_cast<long long>(j)) * p.ldc + n);
  }
  const bool wide = (reinterpret_cast<uintptr_t>(p.D) & 15) == 0 && n0 + 32 <= p.N;
  if (p.out_kind == kOutF32) {
    if (wide && p.ldd % 4 == 0) {
      float* T = reinterpret_cast<float*>(tsm);
      const int q4 = (lane & 7) * 4;
      float* D = reinterpret_cast<float*>(p.D) + n0 + q4;
#pragma unroll
      for (int h = 0; h < 32; h += 16) {  // 16 rows fill the block
#pragma unroll
        for (int j = 0; j < 16; ++j) T[j * 32 + lane] = out[h + j];
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = 4 * k + (lane >> 3);
          if (h + row < left)
            *reinterpret_cast<float4*>(D + (r0 + static_cast<long long>(h + row)) * p.ldd) =
                *reinterpret_cast<const float4*>(&T[row * 32 + q4]);
        }
        __syncwarp();  // the block is rewritten
      }
      return;
    }
  } else if (wide && p.ldd % 8 == 0) {
    unsigned short* T = reinterpret_cast<unsigned short*>(tsm);
#pragma unroll
    for (int j = 0; j < 32; ++j)
      T[j * 32 + lane] = (p.out_kind == kOutBF16) ? __bfloat16_as_ushort(__float2bfloat16_rn(out[j]))
                                                  : __half_as_ushort(__float2half_rn(out[j]));
    __syncwarp();
    const int q8 = (lane & 3) * 8;
    unsigned short* D = reinterpret_cast<unsigned short*>(p.D) + n0 + q8;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = 8 * k + (lane >> 2);
      if (row < left)
        *reinterpret_cast<uint4*>(D + (r0 + static_cast<long long>(row)) * p.ldd) =
            *reinterpret_cast<const uint4*>(&T[row * 32 + q8]);
    }
    __syncwarp();
    return;
  }
  if (n < p.N) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < left) store_d(p.D, p.out_kind, (r0 + static_cast<long long>(j)) * p.ldd + n, out[j]);
  }
}

// map_w: the weights (kExpF16: K-major boxes of 64 K x 128 N, MN-major ones of
// 64 N x 64 K, or (p.w_mn == 2) both 64-column blocks in one box; kExpMx4: 128
// bytes x 128 rows). map_x / map_xs: the rows, in boxes of BN and of XBOX: a
// tile of few rows loads only what it needs. A copy takes about 80 cycles and
// one more per 100 bytes whatever waits for it, which bounds tiles of few rows.
// map_sw / map_sx (kExpMx4): the scales as 128 words x K blocks x row blocks,
// in boxes of 2 K blocks and 1 / XBLK row blocks.
template <int KIND, int BN>
__global__ void __launch_bounds__(ExpCfg<KIND, BN>::THREADS, 1)
    experts_kernel(const __grid_constant__ CUtensorMap map_w,
                   const __grid_constant__ CUtensorMap map_x,
                   const __grid_constant__ CUtensorMap map_xs,
                   const __grid_constant__ CUtensorMap map_sw,
                   const __grid_constant__ CUtensorMap map_sx, const ExpertsParams p) {
  using Cfg = ExpCfg<KIND, BN>;
  constexpr int STAGES = Cfg::STAGES;
  constexpr uint32_t SB = Cfg::STAGE_BYTES;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * SB);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* accf_bar = empty_bar + STAGES;  // [2]
  uint64_t* acce_bar = accf_bar + 2;        // [2]
  uint64_t* drain_bar = acce_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint8_t* epi = smem + STAGES * SB + 512;
  GroupTable tb;
  tb.row0 = reinterpret_cast<int*>(epi + Cfg::EPI_BYTES);
  tb.tile0 = tb.row0 + kMaxGroups + 2;
  tb.blk0 = Cfg::MX ? tb.tile0 + kMaxGroups + 2 : nullptr;

  const int warp = warp_uniform(static_cast<int>(threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  const Abort ab{abort_flag, p.status, p.timeout_ns};

  if (threadIdx.x == 32) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&accf_bar[a], 1);
      mbar_init(&acce_bar[a], 4);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_xs);
    if (Cfg::MX) {
      tma_prefetch_desc(&map_sw);
      tma_prefetch_desc(&map_sx);
    }
  }
  if (warp == 0)
    build_groups(tb, p.sizes, p.sizes64, p.groups, p.rows, BN, p.tiles_w, p.status);
  __syncwarp();
  if (warp == 1) tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_slot);

  const int num_kb = (p.K + Cfg::BK - 1) / Cfg::BK;
  const int num_tiles = tb.tile0[p.groups + 1];
  // tiles with products; the ones behind are stores of beta * C alone
  const int work_tiles = num_kb ? tb.tile0[p.groups] : 0;

  if (warp == 0) {
    if (elect_one()) {
      // ---------------------------------------------------------- producer
      int stage = 0;
      uint32_t phase = 0;
      // above three quarters of the tile one full box of rows, else small boxes
      auto row_boxes = [](const ExpTile& e) {
        return e.nv > BN * 3 / 4 ? 0 : (e.nv + Cfg::XBOX - 1) / Cfg::XBOX;
      };
      auto load_weights = [&](const ExpTile& e, int boxes, int kb, int st) {
        uint8_t* sw = smem + st * SB;
        uint64_t* bar = &full_bar[st];
        mbar_arrive_expect_tx(bar, Cfg::W_TILE + Cfg::SFW + Cfg::SFX +
                                       (boxes ? boxes * Cfg::XBOX * 128 : Cfg::X_TILE));
        if constexpr (Cfg::MX) {
          tma_load_3d(sw, &map_w, bar, kb * 128, e.n0, e.g);  // (bytes)
          tma_load_3d(sw + Cfg::W_TILE + Cfg::X_TILE, &map_sw, bar, 0, 2 * kb, e.g * p.w_blocks + (e.n0 >> 7));
        } else {
          const int k0 = kb * Cfg::BK, gw = p.w_shared ? 0 : e.g;
          if (!p.w_mn) {
            tma_load_3d(sw, &map_w, bar, k0, e.n0, gw);
          } else if (p.w_mn == 2) {
            tma_load_4d(sw, &map_w, bar, 0, k0, e.n0 >> 6, gw);
          } else {
            tma_load_3d(sw, &map_w, bar, e.n0, k0, gw);
            tma_load_3d(sw + 8192, &map_w, bar, e.n0 + 64, k0, gw);
          }
        }
      };
      auto load_rows = [&](const ExpTile& e, int boxes, int kb, int st) {
        uint8_t* sx = smem + st * SB + Cfg::W_TILE;
        uint64_t* bar = &full_bar[st];
        const int k0 = kb * (Cfg::MX ? 128 : 64);
        if (boxes == 0) tma_load_3d(sx, &map_x, bar, k0, e.r0, 0);
        for (int j = 0; j < boxes; ++j)
          tma_load_3d(sx + j * Cfg::XBOX * 128, &map_xs, bar, k0, e.r0 + Cfg::XBOX * j, 0);
        if constexpr (Cfg::MX)
          tma_load_3d(sx + Cfg::X_TILE + Cfg::SFW, &map_sx, bar, 0, 2 * kb, tb.blk0[e.g] + (e.x0 >> 7));
      };
      // The weights of the first stages need not wait for the quantiser.
      int ahead = 0;
      if (Cfg::MX && p.after_quantise) {
        if (static_cast<int>(blockIdx.x) < work_tiles) {
          const ExpTile e = exp_tile<BN, Cfg::STEP>(tb, p.groups, p.tiles_w, blockIdx.x);
          ahead = min(STAGES, num_kb);
          for (int kb = 0; kb < ahead; ++kb) load_weights(e, row_boxes(e), kb, kb);
        }
        wait_prerequisites();
      }
      const bool aborted = [&] {
        for (int t = blockIdx.x; t < work_tiles; t += gridDim.x) {
          const ExpTile e = exp_tile<BN, Cfg::STEP>(tb, p.groups, p.tiles_w, t);
          const int boxes = row_boxes(e);
          for (int kb = 0; kb < num_kb; ++kb) {
            if (ahead > 0) {
              --ahead;
            } else {
              if (!mbar_wait(&empty_bar[stage], phase ^ 1u, ab, kTimeoutEmpty)) return true;
              load_weights(e, boxes, kb, stage);
            }
            load_rows(e, boxes, kb, stage);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        return false;
      }();
      if (aborted || ab.raised()) {
        // let copies already issued land before the CTA exits (bounded)
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 20000000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp walks the tiles, one elected lane issues a tile's K loop:
    // one loop with warp-uniform bounds inside the election keeps descriptors
    // and addresses in uniform registers (with both loops inside it an
    // instruction took about 106 cycles on CTA pairs, so 17).
    const uint32_t sw0 = smem_u32(smem), sx0 = sw0 + Cfg::W_TILE;
    uint64_t wd[4], xd[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      wd[kk] = (!Cfg::MX && p.w_mn) ? sdesc_sw128(sw0 + kk * 2048, 64 * 128, 1024)
                                    : sdesc_sw128(sw0 + kk * 32, 16, 1024);
      xd[kk] = sdesc_sw128(sx0 + kk * 32, 16, 1024);
    }
    const uint64_t sfd = sdesc_kmajor_noswz(sx0 + Cfg::X_TILE, 128, 128);
    int stage = 0, tc = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < work_tiles; t += gridDim.x, ++tc) {
      const ExpTile e = exp_tile<BN, Cfg::STEP>(tb, p.groups, p.tiles_w, t);
      const uint32_t nm = warp_uniform(static_cast<uint32_t>((e.nv + 15) & ~15));
      const uint32_t xcol = warp_uniform(static_cast<uint32_t>(e.x0 >> 5) & 3u);  // in its scale block
      const uint32_t id = Cfg::MX ? idesc_mx4(nm, 0) : idesc(kAccF32, p.in_fmt, p.in_fmt, p.w_mn ? 1 : 0, 0, 128, nm);
      const uint32_t id2 = idesc_mx4(nm, 2);
      const int buf = tc & 1;
      if (!mbar_wait_warp(&acce_bar[buf], ((tc >> 1) & 1) ^ 1u, ab, kTimeoutAccEmpty)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + buf * BN;
      bool ok = true;
      if (elect_one()) {
        int s = stage;
        uint32_t ph = phase;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full_bar[s], ph, ab, kTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t off = s * SB;
          if constexpr (Cfg::MX) {
            const uint32_t sfw = tmem_base + 2 * BN + s * Cfg::SF_COLS;
            const uint32_t sfx = sfw + 8;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              tmem_cp_scales(sfw + 4 * w, sdesc_add(sfd, off + w * 512));
#pragma unroll
              for (int b = 0; b < Cfg::XBLK; ++b)
                tmem_cp_scales(sfx + 4 * (w * Cfg::XBLK + b),
                               sdesc_add(sfd, off + Cfg::SFW + (b * 2 + w) * 512));
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_mx4(d, sdesc_add(wd[kk], off), sdesc_add(xd[kk], off), (kk & 1) ? id2 : id,
                      sfw + 4 * (kk >> 1), sfx + 4 * Cfg::XBLK * (kk >> 1) + xcol, (kb | kk) ? 1u : 0u);
          } else {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f16(d, sdesc_add(wd[kk], off), sdesc_add(xd[kk], off), id, (kb | kk) ? 1u : 0u);
          }
          tc_commit(&empty_bar[s]);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) tc_commit(&accf_bar[buf]);
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      const int adv = stage + num_kb;
      stage = adv % STAGES;
      phase ^= static_cast<uint32_t>(adv / STAGES) & 1u;
    }
    // Every MMA this warp issued must finish before TMEM is released.
    if (elect_one()) {
      tc_commit(drain_bar);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(drain_bar, 0)) {
        if (globaltimer_ns() - t0 > 100000000ull) {  // 100 ms
          ab.raise(kTimeoutDrain);
          break;
        }
      }
    }
    __syncwarp();
  } else if (warp >= 2 && warp < 6) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;  // TMEM lane quarter
    void* tsm = epi + (warp - 2) * (kExpBlockBytes);
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(32 * q) << 16);
    int tc = 0;
    for (int t = blockIdx.x; t < num_tiles; t += gridDim.x) {
      const ExpTile e = exp_tile<BN, Cfg::STEP>(tb, p.groups, p.tiles_w, t);
      const int n0 = e.n0 + 32 * q;
      if (t >= work_tiles) {
        float z[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = 0.0f;
        if (n0 < p.N)
          for (int c = 0; c < e.nv; c += 32) exp_store(p, e.r0 + c, min(32, e.nv - c), n0, z, tsm);
        continue;
      }
      const int buf = tc & 1;
      if (!mbar_wait_warp(&accf_bar[buf], (tc >> 1) & 1, ab, kTimeoutAccFull)) break;
      ++tc;
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < e.nv; c += 32) {
        uint32_t v[32];
        tmem_ld32(lane_base + buf * BN + c, v);
        tmem_ld_wait();
        if (n0 < p.N) {
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = u2f(v[j]);
          exp_store(p, e.r0 + c, min(32, e.nv - c), n0, f, tsm);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acce_bar[buf]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace tb
