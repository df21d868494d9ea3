// Linear and gated linear layers for few rows (single tokens, small batches):
// the weights' bytes, or the depth of K, bound these, not the tensor pipe.
//
// The roles of the operands are swapped: the 128 accumulator lanes of a CTA
// are 128 columns of W and its accumulator columns are up to TOK rows of X, so
// a single token wastes 15 of 16 accumulator columns instead of 127 of 128
// rows of an M = 128 tile, and costs 2 KB of X per stage.  K is split over a
// cluster of `cs` CTAs so that about two CTAs per SM stream W at once through
// their TMA rings.  At the end each CTA sends its fp32 partial sums to the
// CTAs that own them (128 / cs columns each) through distributed shared
// memory, and the owner adds the cs sums in rank order: one launch, no
// workspace, no atomics, and the same bits at every run.  Measured (bf16):
// 1 x 8192 x 8192 22.0 us (6.1 TB/s of weights), 24 rows 23.0 us, gated 4 rows of
// 4096 by 2 x 8192 22.7 us; 1 x 1024 x 1024 3.7 us, of which the weights are 0.3.
//
//   warp 0     TMA producer: W tile (128 columns x 64 k, K- or MN-major) and X
//              tile (TOK x 64 k) per stage
//   warp 1     TMEM allocation, MMA issuer: M = 128, N = TOK, K = 16
//   warps 2-5  accumulator lanes -> owners' shared memory
//   all        sums, bias, activation, product, residual, stores
//
// Gated: lanes 0..63 are 64 columns of the gate's projection and lanes
// 64..127 the same columns of the other one.
#include "activation.cuh"
#include "common.cuh"
#include "dispatch.h"

namespace cuopx {

namespace {

constexpr int LSP_THREADS = 192;
constexpr int LSP_COLS = 128;  // columns of W per CTA
constexpr int LSP_BK = 64;

template <int TOK>
struct SplitSmem {
  static constexpr int STAGES = TOK <= 16 ? 5 : TOK <= 32 ? 4 : TOK <= 64 ? 3 : 6;
  static constexpr int CTAS = TOK <= 64 ? 2 : 1;  // resident per SM
  // With 128 rows the partial sums reuse the ring, once every CTA of the
  // cluster has finished its products; below, they have room of their own.
  static constexpr bool ALIAS = TOK == 128;
  static_assert(TOK <= 128, "one tile holds all rows");
  static constexpr int W_STAGE = LSP_COLS * LSP_BK * 2;
  static constexpr int X_STAGE = TOK * LSP_BK * 2;
  static constexpr int OFF_W = 0;
  static constexpr int OFF_X = OFF_W + STAGES * W_STAGE;
  static constexpr int OFF_SUM = ALIAS ? 0 : OFF_X + STAGES * X_STAGE;  // [cs][TOK][128 / cs] fp32
  static constexpr int OFF_BAR = OFF_X + STAGES * X_STAGE + (ALIAS ? 0 : TOK * LSP_COLS * 4);
  static_assert(!ALIAS || TOK * LSP_COLS * 4 <= OFF_BAR, "the ring holds the partial sums");
  static constexpr int NUM_BARS = 2 * STAGES + 2;  // full, empty, acc_full, drain
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;
  static constexpr uint32_t TMEM_COLS = TOK < 32 ? 32 : TOK;
  static_assert((ALLOC + 1024) * CTAS <= 233472, "CTAS CTAs must fit one SM's shared memory");
};

struct SplitParams {
  int M, N, k_blocks;
  int cs;       // CTAs per cluster
  int w_up;     // gated: first column of the second projection in W
  int act;
  int pairs;  // Y's stores take two columns: N is even, Y's rows start on 4-byte boundaries
  const void* bias;
  const void* R;
  int64_t ldr;
  void* Y;
  int64_t ldy;
  void* Z;
  int64_t ldz;
};

__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

template <typename T, bool W_MN, bool GATED, int TOK>
__global__ void __launch_bounds__(LSP_THREADS, SplitSmem<TOK>::CTAS)
    linear_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                        const SplitParams p) {
  using L = SplitSmem<TOK>;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t STAGE_TX = static_cast<uint32_t>(L::W_STAGE + L::X_STAGE);
  constexpr uint32_t FMT = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  constexpr uint32_t IDESC = make_idesc(FMT, W_MN, false, LSP_COLS, TOK);
  constexpr int TILE_N = GATED ? LSP_COLS / 2 : LSP_COLS;  // output columns per cluster

  extern __shared__ __align__(1024) unsigned char split_smem_raw[];
  unsigned char* smem = align_smem_1024(split_smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = full + 2 * STAGES;
  uint64_t* drain = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  float* sums = reinterpret_cast<float*>(smem + L::OFF_SUM);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cs = p.cs;
  const int rank = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / cs;
  const int n0 = tile * TILE_N;
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * rank / cs);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (rank + 1) / cs);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
    // Warm L2 with the first stages of W while the previous kernel on the
    // stream drains; the loads themselves come after the dependent-launch wait.
    for (int kb = kb0; kb < min(kb1, kb0 + STAGES); ++kb) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = n0 + (GATED ? j * p.w_up : 64 * j);
        if constexpr (W_MN) tma_prefetch_3d(&tmW, c, kb * LSP_BK, 0);
        else tma_prefetch_3d(&tmW, kb * LSP_BK, c, 0);
      }
    }
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, L::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // Remote stores come only after every CTA of the cluster has started (or,
  // into a ring, has read it: the epilogue warps arrive after their accumulator).
  if (cs > 1 && !L::ALIAS) cluster_arrive_relaxed();
  const uint32_t tmem_base = *tmem_slot;
  grid_dependency_wait();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued_mask = 0, phase_mask = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&empty[stage], phase ^ 1u, kDevErrWaitTimeoutEmpty, abort_flag)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[stage], STAGE_TX);
        unsigned char* sw = smem + L::OFF_W + stage * L::W_STAGE;
        const int k0 = kb * LSP_BK;
#pragma unroll
        for (int j = 0; j < 2; ++j) {  // 64 columns of W each
          const int c = n0 + (GATED ? j * p.w_up : 64 * j);
          if constexpr (W_MN) tma_load_3d(sw + j * (64 * LSP_BK * 2), &tmW, &full[stage], c, k0, 0);
          else tma_load_3d(sw + j * (64 * LSP_BK * 2), &tmW, &full[stage], k0, c, 0);
        }
        tma_load_3d(smem + L::OFF_X + stage * L::X_STAGE, &tmX, &full[stage], k0, 0, 0);
        issued_mask |= 1u << stage;
        phase_mask = (phase_mask & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) stage = 0, phase ^= 1u;
      }
      grid_launch_dependents();
      if (!ok) {
        // Abort: let every load already issued land before the CTA goes on.
        for (int s = 0; s < STAGES; ++s) {
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
    if (cs > 1 && L::ALIAS) cluster_arrive_relaxed();
    if (cs > 1) cluster_wait();
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true, issued = false;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(&full[stage], phase, kDevErrWaitTimeoutFull, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t sw = smem_u32(smem + L::OFF_W + stage * L::W_STAGE);
        const uint32_t sx = smem_u32(smem + L::OFF_X + stage * L::X_STAGE);
#pragma unroll
        for (int kk = 0; kk < LSP_BK / 16; ++kk) {
          const uint64_t wd = W_MN ? make_smem_desc_sw128(sw + kk * 2048, 64 * LSP_BK * 2, 1024)
                                   : make_smem_desc_sw128(sw + kk * 32, 16, 1024);
          const uint64_t xd = make_smem_desc_sw128(sx + kk * 32, 16, 1024);
          umma_f16(tmem_base, wd, xd, IDESC, (kb > kb0 || kk > 0) ? 1u : 0u);
        }
        issued = true;
        umma_commit(&empty[stage]);
        if (++stage == STAGES) stage = 0, phase ^= 1u;
      }
      if (ok && issued) {
        umma_commit(acc_full);
      } else if (issued) {
        umma_commit(drain);
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
    if (cs > 1 && L::ALIAS) cluster_arrive_relaxed();
    if (cs > 1) cluster_wait();
  } else {
    const int q = warp & 3;  // TMEM lane quarter of this warp
    const bool got = __all_sync(0xffffffffu, mbar_wait_bounded(acc_full, 0, kDevErrWaitTimeoutAccFull, abort_flag));
    tc_fence_after_sync();
    if (cs > 1 && L::ALIAS) cluster_arrive_relaxed();
    if (cs > 1) cluster_wait();
    // Owner of this lane's column of W, and the column's place among its own.
    const int l = 32 * q + lane;
    const int own = LSP_COLS / cs;
    int owner, local;
    if constexpr (GATED) {
      const int each = 64 / cs, c = l & 63;
      owner = c / each;
      local = (l >> 6) * each + c % each;
    } else {
      owner = l / own;
      local = l % own;
    }
    const uint32_t dst = map_to_rank(sums + rank * TOK * own + local, static_cast<uint32_t>(owner));
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(32 * q) << 16);
#pragma unroll
    for (int c = 0; c < TOK / 16; ++c) {
      uint32_t r[16];
      if (got) {
        tmem_ld_32x32b_x16(t_row + 16 * c, r);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = 0u;  // the error is already recorded
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) st_cluster_f32(dst + static_cast<uint32_t>((16 * c + i) * own * 4), __uint_as_float(r[i]));
    }
  }

  // Partial sums in place, accumulator read.
  tc_fence_before_sync();
  __syncthreads();
  if (cs > 1) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, L::TMEM_COLS);
  }

  // Two neighbouring output columns of one row per step.
  const int own = LSP_COLS / cs, outs = TILE_N / cs;
  const int col0 = n0 + rank * outs;
  const T* bias = static_cast<const T*>(p.bias);
  const T* R = static_cast<const T*>(p.R);
  T* Y = static_cast<T*>(p.Y);
  T* Z = static_cast<T*>(p.Z);
  with_activation(p.act, [&](auto act) {
    for (int e = threadIdx.x; e < p.M * (outs / 2); e += LSP_THREADS) {
      const int t = e / (outs / 2), f = 2 * (e % (outs / 2));
      const int col = col0 + f;
      if (col >= p.N) continue;
      const int64_t row = t;
      const bool two = col + 1 < p.N;
      float z[2][2] = {};  // [projection][column]
#pragma unroll
      for (int h = 0; h < (GATED ? 2 : 1); ++h) {
        for (int s = 0; s < cs; ++s) {
          const float2 v = *reinterpret_cast<const float2*>(sums + (s * TOK + t) * own + h * outs + f);
          z[h][0] += v.x;
          z[h][1] += v.y;
        }
        if (bias) {
          z[h][0] += to_acc<T>(bias[static_cast<int64_t>(h) * p.N + col]);
          if (two) z[h][1] += to_acc<T>(bias[static_cast<int64_t>(h) * p.N + col + 1]);
        }
        if (Z) {
          T* zp = Z + row * p.ldz + static_cast<int64_t>(h) * p.N + col;
          zp[0] = from_acc<T>(z[h][0]);
          if (two) zp[1] = from_acc<T>(z[h][1]);
        }
      }
      const float2 v = act_value2<act.value>(make_float2(z[0][0], z[0][1]));
      float y0 = v.x, y1 = v.y;
      if constexpr (GATED) y0 *= z[1][0], y1 *= z[1][1];
      if (R) {
        const T* rp = R + row * p.ldr + col;
        y0 += to_acc<T>(rp[0]);
        if (two) y1 += to_acc<T>(rp[1]);
      }
      T* yp = Y + row * p.ldy + col;
      if (p.pairs) {  // N is even: both columns exist
        T w[2] = {from_acc<T>(y0), from_acc<T>(y1)};
        *reinterpret_cast<uint32_t*>(yp) = *reinterpret_cast<const uint32_t*>(w);
      } else {
        yp[0] = from_acc<T>(y0);
        if (two) yp[1] = from_acc<T>(y1);
      }
    }
  });
}

template <typename T, bool W_MN, bool GATED, int TOK>
int launch_linear_split(const LinearProblem& p, cudaStream_t stream) {
  using L = SplitSmem<TOK>;
  const CUtensorMapDataType dt =
      std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap mW, mX;
  bool ok = W_MN ? make_map(&mW, dt, p.W, p.w_cols(), p.K, 1, p.ldw, 0, 64, LSP_BK)
                 : make_map(&mW, dt, p.W, p.K, p.w_cols(), 1, p.ldw, 0, LSP_BK, 64);
  // A single row has no stride: any multiple of 8 serves.
  ok &= make_map(&mX, dt, p.X, p.K, p.M, 1, p.M == 1 ? (p.K + 7) / 8 * 8 : p.ldx, 0, LSP_BK, TOK);
  if (!ok) return CUOPX_CUDA_ERROR;
  constexpr int TILE_N = GATED ? LSP_COLS / 2 : LSP_COLS;
  SplitParams prm;
  prm.M = static_cast<int>(p.M);
  prm.N = static_cast<int>(p.N);
  prm.k_blocks = static_cast<int>((p.K + LSP_BK - 1) / LSP_BK);
  prm.w_up = static_cast<int>(p.w_up);
  prm.act = p.act;
  prm.pairs = p.N % 2 == 0 && p.ldy % 2 == 0 && reinterpret_cast<uintptr_t>(p.Y) % 4 == 0;
  prm.bias = p.bias;
  prm.R = p.R;
  prm.ldr = p.ldr;
  prm.Y = p.Y;
  prm.ldy = p.ldy;
  prm.Z = p.Z;
  prm.ldz = p.ldz;
  const int64_t tiles = (p.N + TILE_N - 1) / TILE_N;
  auto kern = linear_split_kernel<T, W_MN, GATED, TOK>;
  static std::atomic<bool> attr_set[64] = {};
  static std::atomic<int> capacity[64][4] = {};  // clusters of 1, 2, 4, 8 CTAs that run at once, one CTA per SM
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return CUOPX_CUDA_ERROR;
  if (!attr_set[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::ALLOC) != cudaSuccess)
      return CUOPX_CUDA_ERROR;
    for (int i = 0; i < 4; ++i)
      capacity[dev][i].store(cluster_capacity(kern, LSP_THREADS, L::ALLOC, 1u << i), std::memory_order_relaxed);
    attr_set[dev].store(true, std::memory_order_release);
  }
  // Split K while the clusters still run in one wave and every CTA keeps two
  // K blocks.  The query counts one CTA per SM.  Where two fit, a few clusters
  // more than a wave cost less than a shallower split: the others have the
  // bandwidth meanwhile (us for clusters of 1, 2, 4, 8: 1 x 4096 x 4096, 32
  // tiles, 30 at once: 21.5, 12.7, 9.6, 8.8; 24 x 8192 x 8192, 64 tiles: 44.7,
  // 29.2, 23.6, 27.8; 128 x 2048 x 4096, one CTA per SM, 16 tiles, 15 at once:
  // 33.3, 19.6, 12.7, 18.7).
  int cs = 1;
  for (int i = 1; i < 4; ++i) {
    const int64_t once = capacity[dev][i].load(std::memory_order_relaxed);
    if (tiles <= (L::CTAS == 2 ? once * 20 / 9 : once) && prm.k_blocks >= (2 << i)) cs = 1 << i;
  }
  prm.cs = cs;
  const cudaError_t err = launch_pdl_cluster(kern, dim3(static_cast<unsigned>(tiles * cs)), dim3(LSP_THREADS), L::ALLOC,
                                             stream, static_cast<unsigned>(cs), mW, mX, prm);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  note_launch(GATED ? "gated_linear_split" : "linear_split");
  return check_launch();
}

template <typename T, int TOK>
int linear_split_layout(const LinearProblem& p, cudaStream_t stream) {
  if (p.gated)
    return p.transW ? launch_linear_split<T, false, true, TOK>(p, stream) : launch_linear_split<T, true, true, TOK>(p, stream);
  return p.transW ? launch_linear_split<T, false, false, TOK>(p, stream) : launch_linear_split<T, true, false, TOK>(p, stream);
}

template <typename T>
int linear_split_rows(const LinearProblem& p, cudaStream_t stream) {
  if (p.M <= 16) return linear_split_layout<T, 16>(p, stream);
  if (p.M <= 32) return linear_split_layout<T, 32>(p, stream);
  if (p.M <= 64) return linear_split_layout<T, 64>(p, stream);
  return linear_split_layout<T, 128>(p, stream);
}

}  // namespace

// Up to 128 rows.  TMA reads X and W; Y, Z, residual and bias may have any alignment.
bool linear_split_supported(const LinearProblem& p) {
  if (p.M <= 0 || p.M > 128 || p.N <= 0 || p.K <= 0) return false;
  if (p.w_cols() > INT32_MAX / 4 || p.K > INT32_MAX / 2) return false;
  if (p.transX) return false;
  if (!row_aligned16(p.X, p.M == 1 ? 0 : p.ldx) || !row_aligned16(p.W, p.ldw)) return false;
  return !p.gated || p.transW || p.w_up % 8 == 0;  // the second projection's first column in W's rows
}

int linear_split(const LinearProblem& p, cudaStream_t stream) {
  return p.dtype == CUOPX_BF16 ? linear_split_rows<__nv_bfloat16>(p, stream) : linear_split_rows<__half>(p, stream);
}

}  // namespace cuopx
