// Linear and gated linear layers whose 256-row tiles are too few for the part:
// CTA pairs (tcgen05 cta_group::2) as in gemm_tc2.cu, with the products' depth
// split over the KS pairs of a cluster.
//
// A pair computes a 256 x 256 tile (gated: 128 columns of both projections)
// over its share of K; KS = 2 or 4 pairs share a tile.  Pair tiles pull half
// the operand bytes per FLOP of the 128-wide tiles that would fill the part
// without splitting (those run into the L2 bandwidth of an SM: 999 x 2048 x
// 5462 f16 took 35 us), and splitting keeps all SMs busy.  At the end a CTA
// holds partial sums of its 128 rows; pair p owns 1 / KS of the columns, and
// every CTA sends the others' columns to the CTA of the same rows in their
// pair, through distributed shared memory into the ring, which by then no
// product reads.  The owner adds the KS sums in pair order, so results do not
// depend on timing, and finishes with the layer epilogue.  Bound by the products and
// about 9 us (13 with four pairs) of set-up, exchange and epilogue around them
// (bf16 512 x 4096 x 4096 18.7 us, 918 TFLOP/s).
//
//   warp 0      TMA producer (both CTAs of a pair)
//   warp 1      TMEM allocation; MMA issuer (even CTA)
//   warps 2-9   partial sums out, then the epilogue of the owned columns
#include "common.cuh"
#include "dispatch.h"
#include "layer_epilogue.cuh"

namespace cuopx {

namespace {

constexpr int LP_BM = 128, LP_BN = 256, LP_BK = 64;
constexpr int LP_STAGES = 5;
constexpr int LP_EPI_WARPS = 8;
constexpr int LP_THREADS = 32 * (2 + LP_EPI_WARPS);
constexpr uint32_t LP_TMEM_COLS = 256;

struct LpSmem {
  static constexpr int A_STAGE = LP_BM * LP_BK * 2;
  static constexpr int B_STAGE = (LP_BN / 2) * LP_BK * 2;
  static constexpr int OFF_A = 0;
  static constexpr int OFF_B = LP_STAGES * A_STAGE;
  static constexpr int OFF_C = OFF_B + LP_STAGES * B_STAGE;  // staging: 8 warps x 2 or 4 warps x 3 buffers of 4 KB
  static constexpr int OFF_BAR = OFF_C + LP_EPI_WARPS * 2 * 4096;
  static constexpr int NUM_BARS = 2 * LP_STAGES + 2;  // full, empty, acc_full, drain
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int OFF_SCALES = OFF_MISC + 16;  // int8: 128 bytes a projection for each finishing warp
  static constexpr int ALLOC = OFF_SCALES + LP_EPI_WARPS * 128 + 1024;
  static_assert(ALLOC <= 232448, "shared memory budget exceeded");
  // Received sums: (KS - 1) x 128 rows x 256 / KS columns, 96 KB at most.
  static_assert(3 * LP_BM * (LP_BN / 4) * 4 <= OFF_C, "the ring holds the received sums");
};

struct LpParams {
  int M, N, tiles_m, k_blocks;
  int w_up;  // gated: first column of the second projection in W
  LayerEpi epi;
};

// Op: T, or int8 (K-major; the exchanged sums are int32, exact in any order).
template <typename T, bool A_MN, bool B_MN, bool GATED, int KS, typename Op = T>
__global__ void __launch_bounds__(LP_THREADS, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmZ,
                       const __grid_constant__ CUtensorMap tmZ2, const __grid_constant__ LpParams p) {
  using L = LpSmem;
  constexpr int COLS = GATED ? LP_BN / 2 : LP_BN;  // output columns of the tile
  constexpr int OWN = COLS / KS;                   // of a pair
  constexpr int FINAL_WARPS = OWN / 64 * 4 < LP_EPI_WARPS ? 4 : LP_EPI_WARPS;
  constexpr int PART = OWN * 4 / FINAL_WARPS;      // columns of one finishing warp
  static_assert(PART % 64 == 0, "whole TMA store boxes");
  constexpr uint32_t PAIR_TX = 2u * static_cast<uint32_t>(L::A_STAGE + L::B_STAGE);
  constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  constexpr bool I8 = std::is_same<Op, int8_t>::value;
  static_assert(!I8 || (!A_MN && !B_MN), "int8: K-major operands");
  constexpr int BK = I8 ? 2 * LP_BK : LP_BK;  // elements of a K block
  constexpr uint32_t IDESC = I8 ? make_idesc_i8(2 * LP_BM, LP_BN) : make_idesc(FMT, A_MN, B_MN, 2 * LP_BM, LP_BN);

  extern __shared__ __align__(1024) unsigned char lp_smem_raw[];
  unsigned char* smem = align_smem_1024(lp_smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + LP_STAGES;
  uint64_t* acc_full = full + 2 * LP_STAGES;
  uint64_t* drain = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t even = rank & ~1u;  // the pair's leader
  const int kp = static_cast<int>(rank >> 1), side = static_cast<int>(rank & 1u);
  const uint16_t pair_mask = static_cast<uint16_t>(3u << even);
  const int tile = static_cast<int>(blockIdx.x) / (2 * KS);
  const int m0 = (tile % p.tiles_m) * 2 * LP_BM + side * LP_BM, n0 = (tile / p.tiles_m) * COLS;
  const int kb0 = p.k_blocks * kp / KS, kb1 = p.k_blocks * (kp + 1) / KS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < LP_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(LP_TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_relaxed();  // barriers and TMEM of the whole cluster are ready
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued_mask = 0, phase_mask = 0;
      bool ok = true;
      // Gated: the even CTA loads the gate's columns of B, the odd one the other projection's.
      const int nb = GATED ? n0 + side * p.w_up : n0 + side * (LP_BN / 2);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, kDevErrWaitTimeoutEmpty, abort_flag)) {
          ok = false;
          break;
        }
        if (side == 0) mbar_arrive_expect_tx(&full[stage], PAIR_TX);
        const uint32_t mbar = map_to_rank(&full[stage], even);
        unsigned char* sa = smem + L::OFF_A + stage * L::A_STAGE;
        unsigned char* sb = smem + L::OFF_B + stage * L::B_STAGE;
        const int k0 = kb * BK;
        if constexpr (A_MN) {
#pragma unroll
          for (int j = 0; j < LP_BM / 64; ++j) tma_load_3d_pair(sa + j * (64 * LP_BK * 2), &tmA, mbar, m0 + 64 * j, k0, 0);
        } else {
          tma_load_3d_pair(sa, &tmA, mbar, k0, m0, 0);
        }
        if constexpr (B_MN) {
#pragma unroll
          for (int j = 0; j < LP_BN / 128; ++j) tma_load_3d_pair(sb + j * (64 * LP_BK * 2), &tmB, mbar, nb + 64 * j, k0, 0);
        } else {
          tma_load_3d_pair(sb, &tmB, mbar, k0, nb, 0);
        }
        issued_mask |= 1u << stage;
        phase_mask = (phase_mask & ~(1u << stage)) | (phase << stage);
        if (++stage == LP_STAGES) stage = 0, phase ^= 1u;
      }
      grid_launch_dependents();
      if (ok) {
        // No commit may still be on its way to this CTA's barriers when the ring is reused.
        for (int i = 0; i < LP_STAGES; ++i) {
          if ((issued_mask >> stage) & 1u)
            if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, kDevErrWaitTimeoutEmpty, abort_flag)) break;
          if (++stage == LP_STAGES) stage = 0, phase ^= 1u;
        }
      } else if (side == 0) {
        // Abort: let every phase this pair issued land.
        for (int s = 0; s < LP_STAGES; ++s) {
          if (!((issued_mask >> s) & 1u)) continue;
          const uint32_t addr = smem_u32(&full[s]);
          const unsigned long long t0 = global_timer_ns();
          while (!mbar_try_wait(addr, (phase_mask >> s) & 1u)) {
            if (global_timer_ns() - t0 > kWaitLimitNs) {
              record_device_error(kDevErrAbortDrain);
              break;
            }
          }
        }
      }
    }
    __syncwarp();
    cluster_sync_relaxed();  // every ring of the cluster is free
    cluster_arrive_relaxed();
    cluster_wait();  // partial sums have arrived
  } else if (warp == 1) {
    if (side == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, issued = false;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&full[stage], phase, kDevErrWaitTimeoutFull, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t sa = smem_u32(smem + L::OFF_A + stage * L::A_STAGE);
        const uint32_t sb = smem_u32(smem + L::OFF_B + stage * L::B_STAGE);
#pragma unroll
        for (int kk = 0; kk < LP_BK / 16; ++kk) {
          const uint64_t ad = A_MN ? make_smem_desc_sw128(sa + kk * 2048, 64 * LP_BK * 2, 1024)
                                   : make_smem_desc_sw128(sa + kk * 32, 16, 1024);
          const uint64_t bd = B_MN ? make_smem_desc_sw128(sb + kk * 2048, 64 * LP_BK * 2, 1024)
                                   : make_smem_desc_sw128(sb + kk * 32, 16, 1024);
          if constexpr (I8) umma_i8_pair(tmem_base, ad, bd, IDESC, (kb > kb0 || kk > 0) ? 1u : 0u);
          else umma_f16_pair(tmem_base, ad, bd, IDESC, (kb > kb0 || kk > 0) ? 1u : 0u);
        }
        issued = true;
        umma_commit_pair_mask(&empty[stage], pair_mask);
        if (++stage == LP_STAGES) stage = 0, phase ^= 1u;
      }
      if (ok) {
        umma_commit_pair_mask(acc_full, pair_mask);
      } else if (issued) {
        umma_commit_pair_mask(drain, static_cast<uint16_t>(1u << rank));
        const uint32_t addr = smem_u32(drain);
        const unsigned long long t0 = global_timer_ns();
        while (!mbar_try_wait(addr, 0)) {
          if (global_timer_ns() - t0 > kWaitLimitNs) {
            record_device_error(kDevErrAbortDrain);
            break;
          }
        }
      }
    }
    __syncwarp();
    cluster_sync_relaxed();
    cluster_arrive_relaxed();
    cluster_wait();
  } else {
    const int q = warp & 3, group = (warp - 2) / 4;  // two warps per TMEM lane quarter
    const int row = 32 * q + lane;
    const bool got = __all_sync(0xffffffffu, mbar_wait_bounded(acc_full, 0, kDevErrWaitTimeoutAccFull, abort_flag));
    tc_fence_after_sync();
    cluster_sync_relaxed();
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(32 * q) << 16);
    // Receive area of a CTA: [source, own pair left out][column][128 rows] fp32.  Columns of both
    // projections when gated: OWN of the gate's, then OWN of the other's.
    constexpr int OWN_ACC = LP_BN / KS;
    float* recv = reinterpret_cast<float*>(smem);
    for (int d = 1; d < KS; ++d) {
      const int to = (kp + d) % KS;
      const int slot = kp < to ? kp : kp - 1;  // among the sources of pair `to`, itself left out
      const uint32_t dst = map_to_rank(recv + (slot * OWN_ACC) * LP_BM + row, static_cast<uint32_t>(2 * to + side));
#pragma unroll 1
      for (int c = group; c < OWN_ACC / 32; c += 2) {
        const int first = GATED ? (c * 32 / OWN) * COLS + to * OWN + c * 32 % OWN : to * OWN + c * 32;
        uint32_t r[32];
        if (got) {
          tmem_ld_32x32b_x32(t_row + static_cast<uint32_t>(first), r);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0u;  // the error is already recorded
        }
#pragma unroll
        for (int i = 0; i < 32; ++i)
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(dst + static_cast<uint32_t>((c * 32 + i) * LP_BM * 4)), "r"(r[i])
                       : "memory");
      }
    }
    cluster_arrive();
    cluster_wait();
    if (group * 4 < FINAL_WARPS && got) {
      const int c0 = group * PART;  // among the pair's columns
      unsigned char* stage = smem + L::OFF_C + (warp - 2) * (GATED ? 3 : 2) * 4096;
      int ybuf = 0;
      Int8Scales<GATED> scales;
      if constexpr (I8) {
        scales = {p.epi.ws, p.N, reinterpret_cast<float*>(smem + L::OFF_SCALES + (warp - 2) * (GATED ? 256 : 128)),
                  m0 + row < p.M ? __ldg(p.epi.xs + m0 + row) : 0.f, {}};
        scales.fetch(n0 + kp * OWN + c0, lane);
      }
      layer_epilogue_tile<T, GATED, COLS, PART>(
          t_row + static_cast<uint32_t>(kp * OWN + c0), n0 + kp * OWN + c0, m0 + 32 * q, p.M, p.N, p.epi, &tmY, &tmZ, &tmZ2,
          stage, lane, ybuf, [] { return true; }, [] {},
          [&](int half, float (&a)[32], float (&b)[GATED ? 32 : 1]) {
            // The sums of all pairs in pair order; this pair's own are in a and b.
            const float* col = recv + (c0 + 32 * half) * LP_BM + row;
            if constexpr (I8) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                int sa = __float_as_int(a[i]), sb = 0;
                if constexpr (GATED) sb = __float_as_int(b[i]);
#pragma unroll
                for (int s = 0; s < KS - 1; ++s) {
                  const float* src = col + (s * OWN_ACC + i) * LP_BM;
                  sa += __float_as_int(*src);
                  if constexpr (GATED) sb += __float_as_int(src[OWN * LP_BM]);
                }
                a[i] = __int_as_float(sa);
                if constexpr (GATED) b[i] = __int_as_float(sb);
              }
              scales.apply(a, b, n0 + kp * OWN + c0 + 32 * (half + 1), lane);
              return;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float sa = 0.f, sb = 0.f;
#pragma unroll
              for (int s = 0; s < KS; ++s) {
                if (s == kp) {
                  sa += a[i];
                  if constexpr (GATED) sb += b[i];
                } else {
                  const float* src = col + ((s < kp ? s : s - 1) * OWN_ACC + i) * LP_BM;
                  sa += *src;
                  if constexpr (GATED) sb += src[OWN * LP_BM];
                }
              }
              a[i] = sa;
              if constexpr (GATED) b[i] = sb;
            }
          });
      if (lane == 0) bulk_wait_group<0>();
      __syncwarp();
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_relaxed();  // the pair partner is done with this CTA's TMEM
  if (warp == 1) {
    tc_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(LP_TMEM_COLS) : "memory");
  }
}

template <typename T, bool A_MN, bool B_MN, bool GATED, int KS, typename Op = T>
int prepare_linear_pair() {
  static std::atomic<bool> attr_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return CUOPX_CUDA_ERROR;
  if (!attr_set[dev].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(linear_pair_kernel<T, A_MN, B_MN, GATED, KS, Op>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize, LpSmem::ALLOC) != cudaSuccess)
      return CUOPX_CUDA_ERROR;
    attr_set[dev].store(true, std::memory_order_relaxed);
  }
  return CUOPX_SUCCESS;
}

template <typename T, bool A_MN, bool B_MN, bool GATED, int KS, typename Op = T>
int launch_linear_pair(const LinearProblem& p, cudaStream_t stream) {
  constexpr bool I8 = std::is_same<Op, int8_t>::value;
  constexpr int COLS = GATED ? LP_BN / 2 : LP_BN;
  const CUtensorMapDataType dt =
      std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap mA, mB, mY = {}, mZ = {}, mZ2 = {};
  LpParams prm = {};
  prm.epi = layer_epi(p);
  bool ok = A_MN ? make_map(&mA, dt, p.X, p.M, p.K, 1, p.ldx, 0, 64, LP_BK)
            : I8 ? make_map_i8(&mA, p.X, p.K, p.M, p.ldx, LP_BM)
                 : make_map(&mA, dt, p.X, p.K, p.M, 1, p.ldx, 0, LP_BK, LP_BM);
  if (B_MN) ok &= make_map(&mB, dt, p.W, p.w_cols(), p.K, 1, p.ldw, 0, 64, LP_BK);
  else if (I8) ok &= make_map_i8(&mB, p.W, p.K, p.w_cols(), p.ldw, LP_BN / 2);
  else ok &= make_map(&mB, dt, p.W, p.K, p.w_cols(), 1, p.ldw, 0, LP_BK, LP_BN / 2);
  if (prm.epi.tma_y) ok &= make_map(&mY, dt, p.Y, p.N, p.M, 1, p.ldy, 0, 64, 32);
  if (prm.epi.tma_z) {
    ok &= make_map(&mZ, dt, p.Z, p.N, p.M, 1, p.ldz, 0, 64, 32);
    if (GATED) ok &= make_map(&mZ2, dt, static_cast<const T*>(p.Z) + p.N, p.N, p.M, 1, p.ldz, 0, 64, 32);
  }
  if (!ok) return CUOPX_CUDA_ERROR;
  prm.M = static_cast<int>(p.M);
  prm.N = static_cast<int>(p.N);
  prm.tiles_m = static_cast<int>((p.M + 2 * LP_BM - 1) / (2 * LP_BM));
  prm.k_blocks = static_cast<int>(p.k_blocks());
  prm.w_up = static_cast<int>(p.w_up);
  const int64_t tiles = static_cast<int64_t>(prm.tiles_m) * ((p.N + COLS - 1) / COLS);
  auto kern = linear_pair_kernel<T, A_MN, B_MN, GATED, KS, Op>;
  if (const int rc = prepare_linear_pair<T, A_MN, B_MN, GATED, KS, Op>(); rc != CUOPX_SUCCESS) return rc;
  const cudaError_t err = launch_pdl_cluster(kern, dim3(static_cast<unsigned>(tiles * 2 * KS)), dim3(LP_THREADS), LpSmem::ALLOC,
                                             stream, 2 * KS, mA, mB, mY, mZ, mZ2, prm);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  if (I8) note_launch(GATED ? "int8_gated_linear_pair_k2" : KS == 2 ? "int8_linear_pair_k2" : "int8_linear_pair_k4");
  else note_launch(GATED ? "gated_linear_pair_k2" : KS == 2 ? "linear_pair_k2" : "linear_pair_k4");
  return check_launch();
}

template <typename T>
int linear_pair_typed(const LinearProblem& p, int ks, cudaStream_t stream) {
  if (p.int8) {
    if (p.gated) return launch_linear_pair<T, false, false, true, 2, int8_t>(p, stream);
    return ks == 2 ? launch_linear_pair<T, false, false, false, 2, int8_t>(p, stream)
                   : launch_linear_pair<T, false, false, false, 4, int8_t>(p, stream);
  }
  if (p.gated)
    return p.transW ? launch_linear_pair<T, false, false, true, 2>(p, stream)
                    : launch_linear_pair<T, false, true, true, 2>(p, stream);
  if (p.transX)
    return ks == 2 ? launch_linear_pair<T, true, true, false, 2>(p, stream)
                   : launch_linear_pair<T, true, true, false, 4>(p, stream);
  if (p.transW)
    return ks == 2 ? launch_linear_pair<T, false, false, false, 2>(p, stream)
                   : launch_linear_pair<T, false, false, false, 4>(p, stream);
  return ks == 2 ? launch_linear_pair<T, false, true, false, 2>(p, stream)
                 : launch_linear_pair<T, false, true, false, 4>(p, stream);
}

}  // namespace

// Clusters (tiles) that run at once; every instantiation has the same launch shape.
int linear_pair_capacity(int ks) {
  static std::atomic<int> cache[2][64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  std::atomic<int>& c = cache[ks == 4][dev];
  if (c.load(std::memory_order_relaxed) == 0) {
    int n = 0;
    if (ks == 4 ? prepare_linear_pair<__half, false, false, false, 4>() == CUOPX_SUCCESS
                : prepare_linear_pair<__half, false, false, false, 2>() == CUOPX_SUCCESS)
      n = ks == 4 ? cluster_capacity(linear_pair_kernel<__half, false, false, false, 4>, LP_THREADS, LpSmem::ALLOC, 8)
                  : cluster_capacity(linear_pair_kernel<__half, false, false, false, 2>, LP_THREADS, LpSmem::ALLOC, 4);
    c.store(n > 0 ? n : -1, std::memory_order_relaxed);
  }
  return std::max(0, c.load(std::memory_order_relaxed));
}

// Same operands as the unsplit pair kernel; ks is 2, or 4 for linear.
int linear_pair(const LinearProblem& p, int ks, cudaStream_t stream) {
  return p.dtype == CUOPX_BF16 ? linear_pair_typed<__nv_bfloat16>(p, ks, stream) : linear_pair_typed<__half>(p, ks, stream);
}

}  // namespace cuopx
