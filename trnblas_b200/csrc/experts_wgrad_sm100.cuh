// Weight gradient of the products grouped by expert (a ragged contraction).
#pragma once

#include "experts_sm100.cuh"

namespace tb {

// ---------------------------------------------------------------------------
// Weight gradient: D[g] (M x N) = alpha * A_g^T B_g + beta * C[g], A_g the
// group's rows of A (rows x M), B_g of B (rows x N), both read MN-major in
// boxes of 64 columns x 64 rows. The contraction runs over a group's rows, so
// its last block reaches into the next group: a fixer warp overwrites those
// rows with zeros in shared memory (both operands: a zero times an infinity of
// another group would be a NaN) before the MMAs of the stage, which run only
// the 16-row steps that hold rows of the group. A group without rows stores
// beta * C.
// ---------------------------------------------------------------------------
struct WgradParams {
  GemmParams p;  // M, N, alpha, beta, C, D, out_kind, c_mode, status, timeout
  int rows, groups;
  const void* sizes;
  int sizes64;
  int in_fmt;
  int wide, tma_d;  // pair kernel: 128-column copies; stores by TMA
};

struct WgradCfg {
  static constexpr int BM = 128, BN = 256, BK = 64, STAGES = 4;
  static constexpr int A_TILE = BM * 128, B_TILE = BN * 128;
  static constexpr int STAGE_BYTES = A_TILE + B_TILE;
  static constexpr int TMEM_COLS = 512;
  static constexpr int THREADS = 32 * 7;  // producer, MMA, 4 epilogue, fixer
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + 512 + (kMaxGroups + 2) * 4;
};

__global__ void __launch_bounds__(WgradCfg::THREADS, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const WgradParams w) {
  using Cfg = WgradCfg;
  constexpr int STAGES = Cfg::STAGES;
  constexpr uint32_t SB = Cfg::STAGE_BYTES;
  const GemmParams& p = w.p;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * SB);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* fix_bar = empty_bar + STAGES;  // the stage's rows behind the group are zero
  uint64_t* accf_bar = fix_bar + STAGES;   // [2]
  uint64_t* acce_bar = accf_bar + 2;       // [2]
  uint64_t* drain_bar = acce_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  GroupTable tb;
  tb.row0 = reinterpret_cast<int*>(smem + STAGES * SB + 512);
  tb.tile0 = tb.blk0 = nullptr;

  const int warp = warp_uniform(static_cast<int>(threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  const Abort ab{abort_flag, p.status, p.timeout_ns};

  if (threadIdx.x == 32) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
      mbar_init(&fix_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&accf_bar[a], 1);
      mbar_init(&acce_bar[a], 4);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 0) build_groups(tb, w.sizes, w.sizes64, w.groups, w.rows, 0, 0, p.status);
  __syncwarp();
  if (warp == 1) tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_slot);

  const int per_group = p.tiles_m * p.tiles_n;
  struct Tile {
    int g, m0, n0, r0, m;
  };
  auto tile = [&](int t) -> Tile {
    Tile e;
    e.g = t / per_group;
    const int i = t - e.g * per_group;
    e.m0 = (i % p.tiles_m) * Cfg::BM;
    e.n0 = (i / p.tiles_m) * Cfg::BN;
    e.r0 = tb.row0[e.g];
    e.m = tb.row0[e.g + 1] - e.r0;
    return e;
  };

  if (warp == 0) {
    if (elect_one()) {
      // ---------------------------------------------------------- producer
      int stage = 0;
      uint32_t phase = 0;
      const bool aborted = [&] {
        for (int t = blockIdx.x; t < p.num_tiles; t += gridDim.x) {
          const Tile e = tile(t);
          for (int r = 0; r < e.m; r += Cfg::BK) {
            if (!mbar_wait(&empty_bar[stage], phase ^ 1u, ab, kTimeoutEmpty)) return true;
            uint8_t* sa = smem + stage * SB;
            uint8_t* sb = sa + Cfg::A_TILE;
            mbar_arrive_expect_tx(&full_bar[stage], SB);
#pragma unroll
            for (int j = 0; j < Cfg::BM / 64; ++j)
              tma_load_3d(sa + j * 8192, &map_a, &full_bar[stage], e.m0 + 64 * j, e.r0 + r, 0);
#pragma unroll
            for (int j = 0; j < Cfg::BN / 64; ++j)
              tma_load_3d(sb + j * 8192, &map_b, &full_bar[stage], e.n0 + 64 * j, e.r0 + r, 0);
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
    const uint32_t id = idesc(kAccF32, w.in_fmt, w.in_fmt, 1, 1, Cfg::BM, Cfg::BN);
    const uint32_t sa0 = smem_u32(smem), sb0 = sa0 + Cfg::A_TILE;
    uint64_t ad[4], bd[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      ad[kk] = sdesc_sw128(sa0 + kk * 2048, 64 * 128, 1024);
      bd[kk] = sdesc_sw128(sb0 + kk * 2048, 64 * 128, 1024);
    }
    int stage = 0, tc = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < p.num_tiles; t += gridDim.x) {
      const int m = warp_uniform(tile(t).m);
      if (m == 0) continue;
      const int buf = tc & 1;
      if (!mbar_wait_warp(&acce_bar[buf], ((tc >> 1) & 1) ^ 1u, ab, kTimeoutAccEmpty)) break;
      ++tc;
      tc_fence_after();
      const uint32_t d = tmem_base + buf * Cfg::BN;
      const int blocks = (m + Cfg::BK - 1) / Cfg::BK;
      bool ok = true;
      if (elect_one()) {
        int s = stage;
        uint32_t ph = phase;
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(&fix_bar[s], ph, ab, kTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t off = s * SB;
          const int steps = (m - kb * Cfg::BK + 15) >> 4;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            if (kk < steps)
              mma_f16(d, sdesc_add(ad[kk], off), sdesc_add(bd[kk], off), id, (kb | kk) ? 1u : 0u);
          tc_commit(&empty_bar[s]);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) tc_commit(&accf_bar[buf]);
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      const int adv = stage + blocks;
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
  } else if (warp == 6) {
    // ------------------------------------------------------------ fixer
    int stage = 0;
    uint32_t phase = 0;
    bool stop = false;
    for (int t = blockIdx.x; t < p.num_tiles && !stop; t += gridDim.x) {
      const Tile e = tile(t);
      for (int r = 0; r < e.m; r += Cfg::BK) {
        if (!mbar_wait_warp(&full_bar[stage], phase, ab, kTimeoutAux)) {
          stop = true;
          break;
        }
        const int v = e.m - r;  // rows of the group in this block
        if (v < Cfg::BK && (v & 15)) {
          // rows v .. round_up(v, 16) of each box, 128 bytes each (the swizzle
          // permutes 16-byte pieces within a row)
          const int pieces = (16 - (v & 15)) * 8;
          for (int b = 0; b < (Cfg::BM + Cfg::BN) / 64; ++b) {
            uint4* z = reinterpret_cast<uint4*>(smem + stage * SB + b * 8192 + v * 128);
            for (int i = lane; i < pieces; i += 32) z[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&fix_bar[stage]);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp >= 2 && warp < 6) {
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(32 * q) << 16);
    int tc = 0;
    for (int t = blockIdx.x; t < p.num_tiles; t += gridDim.x) {
      const Tile e = tile(t);
      const int r = e.m0 + 32 * q + lane;
      const int buf = tc & 1;
      if (e.m) {
        if (!mbar_wait_warp(&accf_bar[buf], (tc >> 1) & 1, ab, kTimeoutAccFull)) break;
        ++tc;
        tc_fence_after();
      }
#pragma unroll 1
      for (int c = 0; c < Cfg::BN / 32; ++c) {
        uint32_t v[32];
        if (e.m) {
          tmem_ld32(lane_base + buf * Cfg::BN + c * 32, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0;
        }
        if (e.n0 + c * 32 < p.N) {
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = u2f(v[j]);
          epilogue_row32(p, e.g, r, e.n0 + c * 32, f);
        }
      }
      if (e.m) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acce_bar[buf]);
      }
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

// ---------------------------------------------------------------------------
// The same on CTA pairs: 256 x 256 tiles, CTA r of a pair with columns 128 r ..
// of A's and of B's block. Both operands are MN-major: where their columns come
// in whole blocks of 64 (p.wide), one copy brings 128 columns (a map of 64
// columns x rows x blocks), else two. Loads complete on the leader's barrier,
// except a group's last block where it ends within a step of 16 rows: that
// completes on a barrier of each CTA, the CTA's fixer warp clears what lies
// behind the group, and the leader's passes the stage on when both are done (a
// fixer in the path of every stage, with its arrival at another CTA, ran at half
// the speed). Eight epilogue warps, two a TMEM lane quarter, write 32-row blocks
// of 64 bytes through shared memory with TMA stores: stored by lanes, a block's
// 32 rows cost 32 partial lines an instruction, and groups of few rows are bound
// by their stores (16 groups of 128 rows, 2048 x 4096: 65 us, four warps 81).
// ---------------------------------------------------------------------------
struct WgradPairCfg {
  static constexpr int BM = 256, BN = 256, BK = 64, STAGES = 6;
  static constexpr int A_TILE = 128 * 128, B_TILE = 128 * 128;
  static constexpr int STAGE_BYTES = A_TILE + B_TILE;
  static constexpr int EPI_WARPS = 8;
  static constexpr int EPI = EPI_WARPS * 2048;
  static constexpr int THREADS = 32 * (3 + EPI_WARPS);  // producer, MMA, fixer, epilogue
  static constexpr int SMEM = STAGES * STAGE_BYTES + EPI + 1024 + 512 + (kMaxGroups + 2) * 4;
};

__global__ void __launch_bounds__(WgradPairCfg::THREADS, 1)
    wgrad_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                      const __grid_constant__ CUtensorMap map_d, const WgradParams w) {
  using Cfg = WgradPairCfg;
  constexpr int STAGES = Cfg::STAGES;
  constexpr uint32_t SB = Cfg::STAGE_BYTES;
  const GemmParams& p = w.p;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* epi = smem + STAGES * SB;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi + Cfg::EPI);  // the leader's
  uint64_t* empty_bar = full_bar + STAGES;                           // each CTA's
  uint64_t* tail_bar = empty_bar + STAGES;                           // each CTA's: a last block has landed
  uint64_t* peer_bar = tail_bar + STAGES;                            // the leader's: the peer's is cleared
  uint64_t* accf_bar = peer_bar + STAGES;                            // [2] each CTA's
  uint64_t* acce_bar = accf_bar + 2;                                 // [2] the leader's
  uint64_t* drain_bar = acce_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  GroupTable tb;
  tb.row0 = reinterpret_cast<int*>(epi + Cfg::EPI + 512);
  tb.tile0 = tb.blk0 = nullptr;

  const int warp = warp_uniform(static_cast<int>(threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  const int rank = warp_uniform(static_cast<int>(cluster_ctarank()));
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int npairs = static_cast<int>(gridDim.x >> 1);
  const Abort ab{abort_flag, p.status, p.timeout_ns};

  if (threadIdx.x == 32) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
      mbar_init(&tail_bar[s], 1);
      mbar_init(&peer_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&accf_bar[a], 1);
      mbar_init(&acce_bar[a], 2 * Cfg::EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
    tma_prefetch_desc(&map_d);
  }
  if (warp == 0) build_groups(tb, w.sizes, w.sizes64, w.groups, w.rows, 0, 0, p.status);
  __syncwarp();
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();  // the peer's barriers are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_slot);

  const int per_group = p.tiles_m * p.tiles_n;
  struct Tile {
    int g, m0, n0, r0, m;
  };
  auto tile = [&](int t) -> Tile {
    Tile e;
    e.g = t / per_group;
    const int i = t - e.g * per_group;
    e.m0 = (i % p.tiles_m) * Cfg::BM;
    e.n0 = (i / p.tiles_m) * Cfg::BN;
    e.r0 = tb.row0[e.g];
    e.m = tb.row0[e.g + 1] - e.r0;
    return e;
  };

  // the block at row r of a group of m rows ends within a step of 16 rows
  auto cut = [](int m, int r) { return m - r < Cfg::BK && (m & 15) != 0; };

  if (warp == 0) {
    if (elect_one()) {
      // ---------------------------------------------------------- producer
      const uint32_t full_leader = mapa_shared(smem_u32(full_bar), 0);
      int stage = 0;
      uint32_t phase = 0;
      const bool aborted = [&] {
        for (int t = pair; t < p.num_tiles; t += npairs) {
          const Tile e = tile(t);
          const int m0 = e.m0 + 128 * rank, n0 = e.n0 + 128 * rank;
          for (int r = 0; r < e.m; r += Cfg::BK) {
            if (!mbar_wait(&empty_bar[stage], phase ^ 1u, ab, kTimeoutEmpty)) return true;
            uint8_t* sa = smem + stage * SB;
            uint8_t* sb = sa + Cfg::A_TILE;
            uint32_t fb;
            if (cut(e.m, r)) {
              mbar_arrive_expect_tx(&tail_bar[stage], SB);
              fb = mapa_shared(smem_u32(&tail_bar[stage]), static_cast<uint32_t>(rank));
            } else {
              if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * SB);
              fb = full_leader + static_cast<uint32_t>(stage) * 8u;
            }
            if (w.wide) {
              tma_load_3d_pair(sa, &map_a, fb, 0, e.r0 + r, m0 >> 6);
              tma_load_3d_pair(sb, &map_b, fb, 0, e.r0 + r, n0 >> 6);
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                tma_load_3d_pair(sa + j * 8192, &map_a, fb, m0 + 64 * j, e.r0 + r, 0);
                tma_load_3d_pair(sb + j * 8192, &map_b, fb, n0 + 64 * j, e.r0 + r, 0);
              }
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        return false;
      }();
      if (aborted || ab.raised()) {
        // copies already issued may complete on the leader's barriers, which this
        // CTA cannot observe: give them time to land (bounded)
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 20000000ull) {
        }
      } else {
        // wait until the MMA has released every stage, so that no commit is in
        // flight towards this CTA when it passes the exit barrier
        for (int i = 0; i < STAGES; ++i) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, ab, kTimeoutEmpty)) break;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer (leader)
    const uint32_t sa0 = smem_u32(smem), sb0 = sa0 + Cfg::A_TILE;
    uint64_t ad[4], bd[4];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      ad[kk] = sdesc_sw128(sa0 + kk * 2048, 64 * 128, 1024);
      bd[kk] = sdesc_sw128(sb0 + kk * 2048, 64 * 128, 1024);
    }
    const uint32_t id = idesc(kAccF32, w.in_fmt, w.in_fmt, 1, 1, Cfg::BM, Cfg::BN);
    int stage = 0, tc = 0;
    uint32_t phase = 0;
    for (int t = pair; t < p.num_tiles; t += npairs) {
      const int m = warp_uniform(tile(t).m);
      if (m == 0) continue;
      const int buf = tc & 1;
      if (!mbar_wait_warp(&acce_bar[buf], ((tc >> 1) & 1) ^ 1u, ab, kTimeoutAccEmpty)) break;
      ++tc;
      tc_fence_after();
      const uint32_t d = tmem_base + buf * Cfg::BN;
      const int blocks = (m + Cfg::BK - 1) / Cfg::BK;
      bool ok = true;
      if (elect_one()) {
        int s = stage;
        uint32_t ph = phase;
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(&full_bar[s], ph, ab, kTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t off = s * SB;
          const int steps = (m - kb * Cfg::BK + 15) >> 4;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            if (kk < steps)
              mma_f16_pair(d, sdesc_add(ad[kk], off), sdesc_add(bd[kk], off), id, (kb | kk) ? 1u : 0u);
          tc_commit_pair(&empty_bar[s], 0x3);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) tc_commit_pair(&accf_bar[buf], 0x3);
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      const int adv = stage + blocks;
      stage = adv % STAGES;
      phase ^= static_cast<uint32_t>(adv / STAGES) & 1u;
    }
    // Every MMA this warp issued must finish before TMEM is released.
    if (elect_one()) {
      tc_commit_pair(drain_bar, 0x1);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(drain_bar, 0)) {
        if (globaltimer_ns() - t0 > 100000000ull) {  // 100 ms
          ab.raise(kTimeoutDrain);
          break;
        }
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------ fixer (both CTAs)
    // Stages pass in the producer's order; the tail barriers' phases count the
    // uses of each stage by a cut block (one bit a stage).
    const uint32_t peer_leader = mapa_shared(smem_u32(peer_bar), 0);
    int stage = 0;
    uint32_t tphase = 0;
    for (int t = pair; t < p.num_tiles; t += npairs) {
      const int m = warp_uniform(tile(t).m);
      const int blocks = (m + Cfg::BK - 1) / Cfg::BK;
      if (blocks == 0) continue;
      stage = (stage + blocks - 1) % STAGES;
      const int r = (blocks - 1) * Cfg::BK;
      if (cut(m, r)) {
        const uint32_t ph = (tphase >> stage) & 1u;
        tphase ^= 1u << stage;
        if (!mbar_wait_warp(&tail_bar[stage], ph, ab, kTimeoutAux)) break;
        const int v = m - r;  // rows of the group in this block
        const int pieces = (16 - (v & 15)) * 8;
        for (int b = 0; b < 4; ++b) {
          uint4* z = reinterpret_cast<uint4*>(smem + stage * SB + b * 8192 + v * 128);
          for (int i = lane; i < pieces; i += 32) z[i] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (rank == 0) {
          if (!mbar_wait_warp(&peer_bar[stage], ph, ab, kTimeoutAux)) break;
          if (lane == 0) mbar_arrive(&full_bar[stage]);
        } else if (lane == 0) {
          mbar_arrive_cluster(peer_leader + static_cast<uint32_t>(stage) * 8u);
        }
      }
      if (++stage == STAGES) stage = 0;
    }
  } else if (warp >= 3) {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;
    const int half = 128 * ((warp - 3) >> 2);  // this warp's columns of the tile
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(32 * q) << 16);
    const uint32_t acce_leader = mapa_shared(smem_u32(acce_bar), 0);
    uint8_t* st = epi + (warp - 3) * 2048;
    // 64-byte rows: the 16-byte piece i of row l at i ^ (l / 2 & 3), the map's swizzle
    uint4* row = reinterpret_cast<uint4*>(st + lane * 64);
    const int swz = (lane >> 1) & 3;
    int tc = 0;
    for (int t = pair; t < p.num_tiles; t += npairs) {
      const Tile e = tile(t);
      const int m0 = e.m0 + 128 * rank + 32 * q;  // this warp's first row
      const int buf = tc & 1;
      const uint32_t acc = lane_base + buf * Cfg::BN;
      if (e.m) {
        if (!mbar_wait_warp(&accf_bar[buf], (tc >> 1) & 1, ab, kTimeoutAccFull)) break;
        ++tc;
        tc_fence_after();
      }
      const int cols = w.tma_d && p.out_kind == kOutF32 ? 16 : 32;
#pragma unroll 1
      for (int c = half; c < half + 128; c += cols) {
        float f[32];
        if (!e.m) {
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = 0.0f;
        } else if (cols == 16) {
          uint32_t v[16];
          tmem_ld16(acc + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] = u2f(v[j]);
        } else {
          uint32_t v[32];
          tmem_ld32(acc + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = u2f(v[j]);
        }
        if (!w.tma_d) {
          if (e.n0 + c < p.N) epilogue_row32(p, e.g, m0 + lane, e.n0 + c, f);
          continue;
        }
        tma_store_wait_read<0>();  // the last chunk's store has left the block
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 32; ++j) f[j] *= p.alpha;
        if (cols == 16) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            row[i ^ swz] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]),
                                      __float_as_uint(f[4 * i + 2]), __float_as_uint(f[4 * i + 3]));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t u[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const float lo = f[8 * i + 2 * h], hi = f[8 * i + 2 * h + 1];
              if (p.out_kind == kOutBF16) {
                __nv_bfloat162 b2 = __floats2bfloat162_rn(lo, hi);
                u[h] = *reinterpret_cast<uint32_t*>(&b2);
              } else {
                __half2 h2 = __floats2half2_rn(lo, hi);
                u[h] = *reinterpret_cast<uint32_t*>(&h2);
              }
            }
            row[i ^ swz] = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (m0 < p.M && e.n0 + c < p.N) tma_store_3d(&map_d, st, e.n0 + c, m0, e.g);
          tma_store_commit();
        }
      }
      if (e.m) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(acce_leader + static_cast<uint32_t>(buf) * 8u);
      }
    }
    tma_store_wait_all();
  }

  // Every role has finished (all waits are bounded): after this barrier no
  // MMA reads either CTA's shared memory and no remote arrive is pending.
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

}  // namespace tb
