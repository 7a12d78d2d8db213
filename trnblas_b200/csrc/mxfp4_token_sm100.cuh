// The MXFP4 product for a few rows (single tokens): at most 16 rows of F32 /
// BF16 / F16 against quantised weights, quantised and multiplied in one launch.
//
// Bounded by the read of the weights, so each CTA takes 128 weight rows and a
// share of K: a cluster of S CTAs splits K (S a power of two chosen so that
// about one CTA an SM runs), and its first CTA adds the partial sums in rank
// order out of shared memory that the others write (deterministic, no
// workspace). While the producer's first weight tiles are on their way, eight
// warps quantise the CTA's share of the rows straight into shared memory in
// the MMA's layout, where it stays; separate quantising cost a launch, its
// latency, and a copy of the rows' tile in every pipeline stage.
#pragma once

#include "experts_sm100.cuh"
#include "mxfp4_convert.cuh"

namespace tb {

struct TokenParams {
  const void* X;
  long long ldx;
  int vec;  // 16-byte loads of X
  int rows, N, K;
  int kb_per_cta;  // K blocks of 256 of each cluster rank
  float alpha, beta;
  int out_kind;
  const void* C;
  long long ldc;
  void* D;
  long long ldd;
  int* status;
  unsigned long long timeout_ns;
};

struct TokenCfg {
  static constexpr int ROWS = 16;    // MMA N
  static constexpr int STAGES = 6;
  static constexpr int W_TILE = 128 * 128;
  static constexpr int STAGE_BYTES = W_TILE + 1024;       // weights and their scales
  static constexpr int X_BYTES = ROWS * 128 + 1024;       // rows and their scales, one K block
  static constexpr int MAX_KB = 22;                       // K blocks a CTA holds
  static constexpr int MAX_SPLIT = 8;
  static constexpr int PART_BYTES = ROWS * 128 * 4;       // one rank's partial sums
  static constexpr int SF_COLS = 16;
  static constexpr int TMEM_COLS = 128;
  static constexpr int CONV_WARPS = 8;
  static constexpr int THREADS = 32 * (2 + CONV_WARPS);
  static constexpr int smem(int kb, int split) {
    return STAGES * STAGE_BYTES + kb * X_BYTES + (split - 1) * PART_BYTES + 1024 + 256;
  }
  static_assert(STAGES * STAGE_BYTES + MAX_KB * X_BYTES + (MAX_SPLIT - 1) * PART_BYTES + 1280 <= 227 * 1024,
                "shared memory");
  static_assert(ROWS + STAGES * SF_COLS <= TMEM_COLS, "accumulator and scales fit TMEM");
};

template <typename T>
__global__ void __launch_bounds__(TokenCfg::THREADS, 1)
    mxfp4_token_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sw,
                       const TokenParams p) {
  using Cfg = TokenCfg;
  constexpr int STAGES = Cfg::STAGES;
  constexpr uint32_t SB = Cfg::STAGE_BYTES;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int split = warp_uniform(static_cast<int>(cluster_nctarank()));
  // (X tiles first: 3 KB a K block keeps them on 1024 bytes; the stages behind
  // them are 17 KB each)
  uint8_t* xq = smem;
  uint8_t* ring = smem + p.kb_per_cta * Cfg::X_BYTES;
  float* red = reinterpret_cast<float*>(ring + STAGES * SB);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(red) + (split - 1) * Cfg::PART_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* x_bar = empty_bar + STAGES;
  uint64_t* acc_bar = x_bar + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_uniform(static_cast<int>(threadIdx.x >> 5));
  const int lane = threadIdx.x & 31;
  const int rank = warp_uniform(static_cast<int>(cluster_ctarank()));
  const int n0 = static_cast<int>(blockIdx.x) / split * 128;
  const Abort ab{abort_flag, p.status, p.timeout_ns};

  if (threadIdx.x == 32) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(x_bar, Cfg::CONV_WARPS);
    mbar_init(acc_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_sw);
  }
  __syncwarp();
  if (warp == 1) tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();  // the first CTA's shared memory may be written from here on
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_slot);

  const int all_kb = (p.K + 255) / 256;
  const int kb0 = rank * p.kb_per_cta;
  const int num_kb = max(0, min(p.kb_per_cta, all_kb - kb0));

  if (warp == 0) {
    if (elect_one()) {
      // ---------------------------------------------------------- producer
      int stage = 0;
      uint32_t phase = 0;
      bool aborted = false;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, ab, kTimeoutEmpty)) {
          aborted = true;
          break;
        }
        uint8_t* sw = ring + stage * SB;
        mbar_arrive_expect_tx(&full_bar[stage], SB);
        tma_load_3d(sw, &map_w, &full_bar[stage], (kb0 + kb) * 128, n0, 0);
        tma_load_3d(sw + Cfg::W_TILE, &map_sw, &full_bar[stage], 0, 2 * (kb0 + kb), n0 >> 7);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
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
    bool ok = true;
    if (elect_one()) {
      const uint32_t w0 = smem_u32(ring), x0 = smem_u32(xq);
      const uint32_t id = idesc_mx4(Cfg::ROWS, 0), id2 = idesc_mx4(Cfg::ROWS, 2);
      const uint64_t wd = sdesc_sw128(w0, 16, 1024), xd = sdesc_sw128(x0, 16, 1024);
      const uint64_t swd = sdesc_kmajor_noswz(w0 + Cfg::W_TILE, 128, 128);
      const uint64_t sxd = sdesc_kmajor_noswz(x0 + Cfg::ROWS * 128, 128, 128);
      ok = mbar_wait(x_bar, 0, ab, kTimeoutAux);
      int s = 0;
      uint32_t ph = 0;
      for (int kb = 0; kb < num_kb && ok; ++kb) {
        if (!mbar_wait(&full_bar[s], ph, ab, kTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t off = s * SB, xoff = kb * Cfg::X_BYTES;
        const uint32_t sfw = tmem_base + Cfg::ROWS + s * Cfg::SF_COLS, sfx = sfw + 8;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          tmem_cp_scales(sfw + 4 * w, sdesc_add(swd, off + w * 512));
          tmem_cp_scales(sfx + 4 * w, sdesc_add(sxd, xoff + w * 512));
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_mx4(tmem_base, sdesc_add(wd, off + kk * 32), sdesc_add(xd, xoff + kk * 32), (kk & 1) ? id2 : id,
                  sfw + 4 * (kk >> 1), sfx + 4 * (kk >> 1), (kb | kk) ? 1u : 0u);
        tc_commit(&empty_bar[s]);
        if (++s == STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
      // every MMA issued so far has completed; also what the epilogue waits for
      tc_commit(acc_bar);
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(acc_bar, 0)) {
        if (globaltimer_ns() - t0 > 100000000ull) {  // 100 ms
          ab.raise(kTimeoutDrain);
          break;
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ quantise the rows
    const T* X = static_cast<const T*>(p.X);
    const int items = p.rows * num_kb;  // one row's 256 values to a warp
    constexpr int U = 4;                // loads in flight
    for (int i0 = warp - 2; i0 < items; i0 += U * Cfg::CONV_WARPS) {
      Raw8<T> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * Cfg::CONV_WARPS;
        const int row = i / num_kb, kb = i - row * num_kb;
        const int k = (kb0 + kb) * 256 + lane * 8;
        const bool in = i < items && k < p.K;
        r[u] = load8(X + (in ? row * p.ldx + k : 0), in ? p.K - k : 0, p.vec);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * Cfg::CONV_WARPS;
        if (i >= items) break;  // (the same for the whole warp)
        const int row = i / num_kb, kb = i - row * num_kb;
        const int k = (kb0 + kb) * 256 + lane * 8;
        uint32_t s;
        const uint32_t w = quantize8<T>(r[u], s);
        uint8_t* xt = xq + kb * Cfg::X_BYTES;
        // 128-byte row, its 16-byte piece c at c ^ (row & 7)
        *reinterpret_cast<uint32_t*>(xt + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4) = w;
        if ((k & ~31) >= p.K) s = 0;
        uint32_t b = s << (8 * ((lane >> 2) & 3));
        b |= __shfl_xor_sync(0xffffffffu, b, 4);
        b |= __shfl_xor_sync(0xffffffffu, b, 8);
        if ((lane & 15) == 0)
          *reinterpret_cast<uint32_t*>(xt + Cfg::ROWS * 128 + (lane >> 4) * 512 + row * 16) = b;
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(x_bar);
  }

  // ---------------------------------------------------------------- epilogue
  float v[Cfg::ROWS];
#pragma unroll
  for (int j = 0; j < Cfg::ROWS; ++j) v[j] = 0.0f;
  const int q = warp & 3;
  const bool epi = warp >= 2 && warp < 6;
  if (epi && num_kb > 0) {
    if (mbar_wait_warp(acc_bar, 0, ab, kTimeoutAccFull)) {
      tc_fence_after();
      uint32_t u[16];
      tmem_ld16(tmem_base + (static_cast<uint32_t>(32 * q) << 16), u);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < Cfg::ROWS; ++j) v[j] = u2f(u[j]);
    }
  }
  if (split > 1) {
    if (epi && rank > 0) {
      const uint32_t dst = mapa_shared(smem_u32(red + (rank - 1) * Cfg::ROWS * 128 + 32 * q + lane), 0);
#pragma unroll
      for (int j = 0; j < Cfg::ROWS; ++j)
        if (j < p.rows) st_cluster_f32(dst + j * 512, v[j]);
    }
    tc_fence_before();
    __syncthreads();
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
  }
  if (epi && rank == 0) {
    const int n = n0 + 32 * q + lane;
#pragma unroll
    for (int j = 0; j < Cfg::ROWS; ++j) {
      if (j >= p.rows || n >= p.N) continue;
      float a = v[j];
      for (int r = 0; r < split - 1; ++r) a += red[r * Cfg::ROWS * 128 + j * 128 + 32 * q + lane];
      float o = p.alpha * a;
      if (p.C != nullptr && p.beta != 0.0f) o += p.beta * load_c(p.C, p.out_kind, j * p.ldc + n);
      store_d(p.D, p.out_kind, j * p.ldd + n, o);
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
