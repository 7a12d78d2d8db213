// Products grouped by expert on CTA pairs (tcgen05 cta_group::2): one MMA of
// 256 weight columns x up to BN rows over two SMs.
//
// CTA r of a pair holds weight columns 128 r .. 128 r + 127 of the tile and
// rows r N / 2 .. (r + 1) N / 2 - 1 of its N (a multiple of 32): the pair
// stages half the row bytes per MMA that two single CTAs would, which is what
// bounds the one-CTA kernel on long groups (a 128 x 256 MMA reads 96 bytes of
// shared memory a cycle beside the same amount written by the loads; here 64).
// Loads carry no multicast; both CTAs' complete on the leader's barrier. The
// walk, the group table and the epilogue are the one-CTA kernel's.
//
// kExpMx4: each CTA's tensor core scales its own 128 weight columns and all N
// rows, so both bring the row scales. The scale columns are a ring of NSLOT
// beside the two accumulators; where that is shorter than the pipeline, the
// issuer waits for the MMAs that read a slot before it copies into it.
#pragma once

#include "experts_sm100.cuh"

namespace tb {

// NBUF accumulators: two, so that the next tile's MMAs run beside an epilogue,
// or one, where a pair has one tile anyway.
template <int KIND, int BN, int NBUF>
struct ExpPairCfg {
  static constexpr bool MX = KIND == kExpMx4;
  static constexpr int BK = MX ? 256 : 64;
  static constexpr int HN = BN / 2;  // rows of a CTA
  static constexpr int W_TILE = 128 * 128;
  static constexpr int X_TILE = HN * 128;
  // rows start at a multiple of STEP in their group, so that their scales lie in
  // two blocks
  static constexpr int STEP = !MX ? 32 : BN == 192 ? 64 : 128;
  static constexpr int XBLK = (BN + 127) / 128;
  static_assert(!MX || BN == 192 || BN == 256, "a tile's rows lie in two scale blocks");
  static constexpr int SFW = MX ? 2 * 512 : 0;
  static constexpr int SFX = MX ? 2 * XBLK * 512 : 0;
  static constexpr int STAGE_BYTES = W_TILE + X_TILE + SFW + SFX;
  static_assert(STAGE_BYTES % 1024 == 0 && BN % 32 == 0 && BN <= 256, "tile geometry");
  // two a TMEM lane quarter: the last tile's epilogue runs alone, and 4-bit tiles
  // pass in half the time (4133 rows of 8, 1024 x 2816 fp16, operands in L2: 23.7
  // us, four warps 25.4)
  static constexpr int EPI_WARPS = 8;
  static constexpr int EPI_BYTES = EPI_WARPS * kExpBlockBytes;
  static constexpr int FIT = (227 * 1024 - 1024 - 512 - EPI_BYTES - kGroupTableBytes) / STAGE_BYTES;
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int SF_COLS = MX ? 2 * 4 * (1 + XBLK) : 0;
  static constexpr int NSLOT_FIT = MX ? (512 - NBUF * BN) / (SF_COLS ? SF_COLS : 1) : 0;
  static constexpr int NSLOT = NSLOT_FIT < STAGES ? NSLOT_FIT : STAGES;
  static_assert(!MX || NSLOT >= 2, "two scale slots");
  static constexpr int THREADS = 32 * (2 + EPI_WARPS);
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + 512 + EPI_BYTES + kGroupTableBytes;
};

__device__ __forceinline__ void mma_mx4_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                             uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_cp_scales_pair(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

// map_w: as for the one-CTA kernel, or (p.w_mn == 2) MN-major in boxes of 64 N
// x 64 K x 2 blocks of 64 N, one copy instead of two. map_x / map_x32: the
// rows in boxes of HN and of 32.
template <int KIND, int BN, int NBUF>
__global__ void __launch_bounds__(ExpPairCfg<KIND, BN, NBUF>::THREADS, 1)
    experts_pair_kernel(const __grid_constant__ CUtensorMap map_w,
                        const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_x32,
                        const __grid_constant__ CUtensorMap map_sw,
                        const __grid_constant__ CUtensorMap map_sx, const ExpertsParams p) {
  using Cfg = ExpPairCfg<KIND, BN, NBUF>;
  constexpr int STAGES = Cfg::STAGES;
  constexpr uint32_t SB = Cfg::STAGE_BYTES;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * SB);  // the leader's
  uint64_t* empty_bar = full_bar + STAGES;                               // each CTA's
  uint64_t* accf_bar = empty_bar + STAGES;                               // [2] each CTA's
  uint64_t* acce_bar = accf_bar + 2;                                     // [2] the leader's
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
  const int rank = warp_uniform(static_cast<int>(cluster_ctarank()));
  const int pair = static_cast<int>(blockIdx.x >> 1);
  const int npairs = static_cast<int>(gridDim.x >> 1);
  const Abort ab{abort_flag, p.status, p.timeout_ns};

  if (threadIdx.x == 32) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&accf_bar[a], 1);
      mbar_init(&acce_bar[a], 2 * Cfg::EPI_WARPS);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_x32);
    if (Cfg::MX) {
      tma_prefetch_desc(&map_sw);
      tma_prefetch_desc(&map_sx);
    }
  }
  if (warp == 0)
    build_groups(tb, p.sizes, p.sizes64, p.groups, p.rows, BN, p.tiles_w, p.status);
  __syncwarp();
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();  // the peer's barriers are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_slot);

  const int num_kb = (p.K + Cfg::BK - 1) / Cfg::BK;
  const int num_tiles = tb.tile0[p.groups + 1];
  const int work_tiles = num_kb ? tb.tile0[p.groups] : 0;

  if (warp == 0) {
    if (elect_one()) {
      // ---------------------------------------------------------- producer
      const uint32_t full_leader = mapa_shared(smem_u32(full_bar), 0);
      int stage = 0;
      uint32_t phase = 0;
      auto half_rows = [](const ExpTile& e) { return ((e.nv + 31) & ~31) / 2; };  // of each CTA
      // above three quarters one full box, else boxes of 32 rows
      auto row_boxes = [](int half) { return half > Cfg::HN * 3 / 4 ? 0 : (half + 31) / 32; };
      auto load_weights = [&](const ExpTile& e, int boxes, int kb, int st) {
        if (rank == 0)
          mbar_arrive_expect_tx(&full_bar[st], 2 * (Cfg::W_TILE + Cfg::SFW + Cfg::SFX +
                                                    (boxes ? boxes * 32 * 128 : Cfg::X_TILE)));
        const uint32_t fb = full_leader + static_cast<uint32_t>(st) * 8u;
        uint8_t* sw = smem + st * SB;
        const int k0 = kb * (Cfg::MX ? 128 : 64);  // elements of the map
        const int n0 = e.n0 + 128 * rank;
        const int gw = p.w_shared ? 0 : e.g;
        if (Cfg::MX || !p.w_mn) {
          tma_load_3d_pair(sw, &map_w, fb, k0, n0, gw);
        } else if (p.w_mn == 2) {
          tma_load_4d_pair(sw, &map_w, fb, 0, k0, n0 >> 6, gw);
        } else {
          tma_load_3d_pair(sw, &map_w, fb, n0, k0, gw);
          tma_load_3d_pair(sw + 8192, &map_w, fb, n0 + 64, k0, gw);
        }
        if constexpr (Cfg::MX)
          tma_load_3d_pair(sw + Cfg::W_TILE + Cfg::X_TILE, &map_sw, fb, 0, 2 * kb, e.g * p.w_blocks + (n0 >> 7));
      };
      auto load_rows = [&](const ExpTile& e, int half, int boxes, int kb, int st) {
        const uint32_t fb = full_leader + static_cast<uint32_t>(st) * 8u;
        uint8_t* sx = smem + st * SB + Cfg::W_TILE;
        const int k0 = kb * (Cfg::MX ? 128 : 64), r0 = e.r0 + half * rank;
        if (boxes == 0) tma_load_3d_pair(sx, &map_x, fb, k0, r0, 0);
        for (int j = 0; j < boxes; ++j) tma_load_3d_pair(sx + j * 4096, &map_x32, fb, k0, r0 + 32 * j, 0);
        if constexpr (Cfg::MX)
          tma_load_3d_pair(sx + Cfg::X_TILE + Cfg::SFW, &map_sx, fb, 0, 2 * kb, tb.blk0[e.g] + (e.x0 >> 7));
      };
      // The weights of the first stages need not wait for the quantiser.
      int ahead = 0;
      if (Cfg::MX && p.after_quantise) {
        if (pair < work_tiles) {
          const ExpTile e = exp_tile<BN, Cfg::STEP, 256>(tb, p.groups, p.tiles_w, pair);
          ahead = min(STAGES, num_kb);
          for (int kb = 0; kb < ahead; ++kb) load_weights(e, row_boxes(half_rows(e)), kb, kb);
        }
        wait_prerequisites();
      }
      const bool aborted = [&] {
        for (int t = pair; t < work_tiles; t += npairs) {
          const ExpTile e = exp_tile<BN, Cfg::STEP, 256>(tb, p.groups, p.tiles_w, t);
          const int half = half_rows(e), boxes = row_boxes(half);
          for (int kb = 0; kb < num_kb; ++kb) {
            if (ahead > 0) {
              --ahead;
            } else {
              if (!mbar_wait(&empty_bar[stage], phase ^ 1u, ab, kTimeoutEmpty)) return true;
              load_weights(e, boxes, kb, stage);
            }
            load_rows(e, half, boxes, kb, stage);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        return false;
      }();
      if (aborted || ab.raised()) {
        // copies already issued complete on the leader's barriers, which this
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
    constexpr bool RING = Cfg::MX && Cfg::NSLOT < STAGES;  // fewer scale slots than stages
    int stage = 0, tc = 0;
    uint32_t phase = 0;
    long long g0 = 0;  // K blocks issued before this tile
    for (int t = pair; t < work_tiles; t += npairs, ++tc) {
      const ExpTile e = exp_tile<BN, Cfg::STEP, 256>(tb, p.groups, p.tiles_w, t);
      const uint32_t nm = warp_uniform(static_cast<uint32_t>((e.nv + 31) & ~31));
      const uint32_t xcol = warp_uniform(static_cast<uint32_t>(e.x0 >> 5) & 3u);  // in its scale block
      const uint32_t id = Cfg::MX ? idesc_mx4(nm, 0) + (1u << 27)  // M = 256
                                  : idesc(kAccF32, p.in_fmt, p.in_fmt, p.w_mn ? 1 : 0, 0, 256, nm);
      const uint32_t id2 = idesc_mx4(nm, 2) + (1u << 27);
      const int buf = tc % NBUF;
      if (!mbar_wait_warp(&acce_bar[buf], ((tc / NBUF) & 1) ^ 1u, ab, kTimeoutAccEmpty)) break;
      tc_fence_after();
      const uint32_t d = tmem_base + buf * BN;
      // the slot's last reader: the K block NSLOT back, its stage and phase
      const long long b0 = RING && g0 > Cfg::NSLOT ? g0 - Cfg::NSLOT : 0;
      bool ok = true;
      if (elect_one()) {
        int s = stage, slot = RING ? static_cast<int>(g0 % (RING ? Cfg::NSLOT : 1)) : 0;
        uint32_t ph = phase;
        int back = static_cast<int>(b0 % STAGES), skip = RING && g0 < Cfg::NSLOT ? Cfg::NSLOT - static_cast<int>(g0) : 0;
        uint32_t bph = static_cast<uint32_t>(b0 / STAGES) & 1u;
        for (int kb = 0; kb < num_kb; ++kb) {
          if constexpr (RING) {
            if (skip > 0) {
              --skip;
            } else {
              if (!mbar_wait(&empty_bar[back], bph, ab, kTimeoutEmpty)) {
                ok = false;
                break;
              }
              if (++back == STAGES) {
                back = 0;
                bph ^= 1u;
              }
            }
          }
          if (!mbar_wait(&full_bar[s], ph, ab, kTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t off = s * SB;
          if constexpr (Cfg::MX) {
            const uint32_t sfw = tmem_base + NBUF * BN + (RING ? slot : s) * Cfg::SF_COLS;
            const uint32_t sfx = sfw + 8;
            if (++slot == Cfg::NSLOT) slot = 0;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              tmem_cp_scales_pair(sfw + 4 * w, sdesc_add(sfd, off + w * 512));
#pragma unroll
              for (int b = 0; b < Cfg::XBLK; ++b)
                tmem_cp_scales_pair(sfx + 4 * (w * Cfg::XBLK + b),
                                    sdesc_add(sfd, off + Cfg::SFW + (b * 2 + w) * 512));
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_mx4_pair(d, sdesc_add(wd[kk], off), sdesc_add(xd[kk], off), (kk & 1) ? id2 : id,
                           sfw + 4 * (kk >> 1), sfx + 4 * Cfg::XBLK * (kk >> 1) + xcol, (kb | kk) ? 1u : 0u);
          } else {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f16_pair(d, sdesc_add(wd[kk], off), sdesc_add(xd[kk], off), id, (kb | kk) ? 1u : 0u);
          }
          tc_commit_pair(&empty_bar[s], 0x3);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) tc_commit_pair(&accf_bar[buf], 0x3);
      }
      g0 += num_kb;
      if (!__all_sync(0xffffffffu, ok)) break;
      const int adv = stage + num_kb;
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
  } else if (warp >= 2) {
    // ------------------------------------------------------------ epilogue (both CTAs)
    const int q = warp & 3;
    // chunks of 32 rows alternate between the two
    const int c0 = 32 * ((warp - 2) >> 2), cstep = 8 * Cfg::EPI_WARPS;
    void* tsm = epi + (warp - 2) * kExpBlockBytes;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(32 * q) << 16);
    const uint32_t acce_leader = mapa_shared(smem_u32(acce_bar), 0);
    int tc = 0;
    for (int t = pair; t < num_tiles; t += npairs) {
      const ExpTile e = exp_tile<BN, Cfg::STEP, 256>(tb, p.groups, p.tiles_w, t);
      const int n0 = e.n0 + 128 * rank + 32 * q;
      if (t >= work_tiles) {
        float z[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = 0.0f;
        if (n0 < p.N)
          for (int c = c0; c < e.nv; c += cstep) exp_store(p, e.r0 + c, min(32, e.nv - c), n0, z, tsm);
        continue;
      }
      const int buf = tc % NBUF;
      if (!mbar_wait_warp(&accf_bar[buf], (tc / NBUF) & 1, ab, kTimeoutAccFull)) break;
      ++tc;
      tc_fence_after();
#pragma unroll 1
      for (int c = c0; c < e.nv; c += cstep) {
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
      if (lane == 0) mbar_arrive_cluster_relaxed(acce_leader + static_cast<uint32_t>(buf) * 8u);
    }
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
