// Orthogonalised updates by Newton-Schulz products (cuopx_orthogonalize,
// cuopx_muon_step).  For G = U S V^T the iteration
//   X0 = G / (||G|| + eps),   X <- a X + (b A + c A A) X,   A = X X^T
// applies the odd polynomial a s + b s^3 + c s^5 to the singular values; with
// (3.4445, -4.7750, 2.0315) five steps take nearly all of (0, 1] to 0.7 .. 1.2
// (K. Jordan, "Muon", 2024; the quintic form is Bjorck and Bowie's, 1971).
//
// Everything works on the smaller Gram matrix, p = min(rows, columns): a tall X
// (rows > columns) has A = X^T X and X <- a X + X (b A + c A A).  Neither form
// is transposed: the tensor cores read X's rows or columns as its storage has them.
//
// Numbers.  The products take fp16 operands and sum in fp32.  Rounding X itself
// to 16 bits at every step would lose the small singular values, which a factor of
// 3.4 a step lifts out of the noise (of a gradient with a few large directions the result
// is off by 4 % in fp16, 30 % in bf16).  So X is kept as two fp16 numbers, hi + lo
// (22 bits): the products read hi, while a X, which carries the small directions, takes
// both, and errors of 2e-4 (few large directions) to 1.6e-3 (equal ones) remain.  Every matrix
// is stored times a power of two that its bound allows (2^15 / bound): the
// elements of A are far below fp16's normal range otherwise.
//
// One persistent launch does all products: 256 x PBN tiles on CTA pairs (tcgen05
// cta_group::2), tile i of a phase on pair i mod the number of pairs, grid
// barriers between phases.  A and the polynomial are symmetric: tiles on or below the
// diagonal are computed, and those below it stored twice, once transposed.
//   warp 0     TMA producer (both CTAs)
//   warp 1     TMEM allocation; MMA issuer (even CTA)
//   warps 2-9  epilogue: alpha * sums + beta * (what the phase adds), rounded, by TMA store
#include <cmath>

#include "common.cuh"
#include "dispatch.h"
#include "layer_epilogue.cuh"

namespace cuopx {

namespace {

constexpr int ORT_MAX_STEPS = 32;
constexpr int ORT_BM = 128;  // rows per CTA (pair: 256)
constexpr int ORT_BK = 64;
constexpr int ORT_EPI_WARPS = 8;
constexpr int ORT_THREADS = 32 * (2 + ORT_EPI_WARPS);
constexpr uint32_t ORT_TMEM_COLS = 512;

template <int PBN>
struct OrthoSmem {
  static constexpr int SLOTS = static_cast<int>(ORT_TMEM_COLS) / PBN;
  static constexpr int STAGES = PBN == 256 ? 5 : 6;
  static constexpr int A_STAGE = ORT_BM * ORT_BK * 2;
  static constexpr int B_STAGE = PBN / 2 * ORT_BK * 2;
  static constexpr int OFF_A = 0;
  static constexpr int OFF_B = STAGES * A_STAGE;
  static constexpr int OFF_C = OFF_B + STAGES * B_STAGE;  // per warp: two staging buffers of 4 KB
  static constexpr int OFF_BAR = OFF_C + ORT_EPI_WARPS * 2 * 4096;
  static constexpr int NUM_BARS = 2 * STAGES + 2 * SLOTS + 3;  // full, empty, acc_full, acc_empty, drain, done, go
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;
  static_assert(ALLOC <= 232448, "shared memory budget exceeded");
};

// The three phases of a step: A = X X^T, the polynomial P = bA + cAA, X <- aX + PX.
enum OrthoPhase { kGram = 0, kPoly = 1, kUpdate = 2 };

struct OrthoMaps {
  // Operands: [phase], for the two buffers that X alternates between.
  CUtensorMap a[3][2], b[3][2];
  CUtensorMap gram, gram_t, poly, poly_t;  // stores, and transposed ones (boxes of 32 x 64)
  CUtensorMap x[2], lo;
};

struct OrthoArgs {
  int batch, p, q, steps;
  bool tall;
  int tiles[3];     // of a phase, all batches
  int k_blocks[3];
  int tiles_m, tiles_n;  // of the update, one batch
  int sym_tiles;         // of the other two, one batch
  const __half* x[2];
  const __half* lo;
  const __half* gram;
  int64_t ldx, stride_x, ldp, stride_p;  // elements
  unsigned* barrier;
  float alpha[ORT_MAX_STEPS][3], beta[ORT_MAX_STEPS][3];
};

__device__ __forceinline__ unsigned ld_acquire_gpu(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void red_release_gpu(unsigned* p) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory");
}
// Between generic accesses and those of TMA, either way, any memory.
__device__ __forceinline__ void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }

// Waits until `count` CTAs have arrived (bounded).
__device__ __forceinline__ bool grid_wait(const unsigned* barrier, unsigned count, volatile int* abort) {
  const unsigned long long t0 = global_timer_ns();
  for (uint32_t it = 0; ld_acquire_gpu(barrier) < count; ++it) {
    if ((it & 63u) == 63u) {
      if (*abort) return false;
      if (global_timer_ns() - t0 > kWaitLimitNs) {
        record_device_error(kDevErrGridBarrier);
        *abort = 1;
        return false;
      }
    }
  }
  fence_proxy_async_all();
  return true;
}

// Tile t of a phase: batch, row tile (256 rows) and column tile (PBN columns).
// Symmetric phases have the tiles whose first column is at most their last row.
template <int PBN>
__device__ __forceinline__ void ortho_tile(const OrthoArgs& g, int phase, int t, int& b, int& mt, int& nt) {
  if (phase == kUpdate) {
    const int per = g.tiles_m * g.tiles_n;
    b = t / per;
    const int r = t - b * per;
    constexpr int GROUP = 8;  // row tiles that share the columns' operand while it is in L2
    const int span = GROUP * g.tiles_n, grp = r / span, first = grp * GROUP;
    const int rows = min(GROUP, g.tiles_m - first), rr = r - grp * span;
    mt = first + rr % rows;
    nt = rr / rows;
  } else {
    constexpr int R = 256 / PBN;
    b = t / g.sym_tiles;
    const int r = t - b * g.sym_tiles;
    int i = static_cast<int>((sqrtf(8.f * (r / R) + 1.f) - 1.f) * 0.5f);
    while (R * i * (i + 1) / 2 > r) --i;
    while (R * (i + 1) * (i + 2) / 2 <= r) ++i;
    mt = i;
    nt = r - R * i * (i + 1) / 2;
  }
}

// 32 halves of a row, from L2 (other CTAs have written them in this launch).
__device__ __forceinline__ void ortho_row32(const __half* row, int64_t col, int64_t cols, bool in, uint4 (&raw)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    raw[j] = make_uint4(0, 0, 0, 0);
    if (in && col + 8 * j < cols) raw[j] = __ldcg(reinterpret_cast<const uint4*>(row + col + 8 * j));
  }
}

// One warp's 32 rows of PART columns of a tile, in chunks of 64 columns.
// UPDATE: hi and lo of X in, hi and lo out.  Else the sums, plus beta * r0
// where beta is not 0, to `tm0`, and transposed to `tm1` if `mirror`.
template <bool UPDATE, int PART, typename Wait, typename Release>
__device__ __forceinline__ bool ortho_epilogue(uint32_t t_row, int n0, int m0, int b, int M, int N, float alpha, float beta,
                                               const __half* r0, const __half* r1, int64_t ld, bool mirror,
                                               const CUtensorMap* tm0, const CUtensorMap* tm1, unsigned char* stage, int lane,
                                               Wait&& wait, Release&& release) {
  constexpr int BUF = 4096;
  const bool in = m0 + lane < M && (UPDATE || beta != 0.f);
  const __half* row0 = r0 + (m0 + lane) * ld;
  const __half* row1 = r1 + (m0 + lane) * ld;
  uint4 next0[4], next1[UPDATE ? 4 : 1];
  auto fetch = [&](int64_t col) {
    ortho_row32(row0, col, N, in, next0);
    if constexpr (UPDATE) ortho_row32(row1, col, N, in, next1);
  };
  fetch(n0);
  if (!wait()) return false;
#pragma unroll 1
  for (int half = 0; half < PART / 32; ++half) {
    const int h = half & 1;
    uint32_t acc[32];
    tmem_ld_32x32b_x32(t_row + 32 * half, acc);
    tmem_wait_ld();
    if (half == PART / 32 - 1) release();
    float v[32];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w0[4] = {next0[j].x, next0[j].y, next0[j].z, next0[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 add = unpack2_layer<__half>(w0[i]);
        if constexpr (UPDATE) {
          const uint32_t w1[4] = {next1[j].x, next1[j].y, next1[j].z, next1[j].w};
          add = add2(add, unpack2_layer<__half>(w1[i]));
        }
        const float2 s = make_float2(__uint_as_float(acc[8 * j + 2 * i]), __uint_as_float(acc[8 * j + 2 * i + 1]));
        const float2 r = fma2(both(alpha), s, mul2(both(beta), add));
        v[8 * j + 2 * i] = r.x, v[8 * j + 2 * i + 1] = r.y;
      }
    }
    if (half + 1 < PART / 32) fetch(n0 + 32 * (half + 1));
    if (h == 0) {
      if (lane == 0) bulk_wait_group_read<0>();
      __syncwarp();
    }
    stage_row32<__half>(stage, lane, h, v);
    if constexpr (UPDATE) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] -= __half2float(__float2half_rn(v[i]));
      stage_row32<__half>(stage + BUF, lane, h, v);
    } else if (mirror) {
      // Row 32 h + i of the transposed chunk holds column i of this one, an
      // element per lane; lanes trade elements so that each stores two at once.
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const bool odd = lane & 1;
        const float got = __shfl_xor_sync(0xffffffffu, odd ? v[i] : v[i + 1], 1);
        const uint32_t w = odd ? pack2_layer<__half>(got, v[i + 1]) : pack2_layer<__half>(v[i], got);
        *reinterpret_cast<uint32_t*>(stage + BUF + (32 * h + i + (odd ? 1 : 0)) * 64 + (lane >> 1) * 4) = w;
      }
    }
    if (h == 1) {
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) {
        const int c = n0 + 32 * (half - 1);
        tma_store_3d(tm0, stage, c, m0, b);
        if constexpr (UPDATE) tma_store_3d(tm1, stage + BUF, c, m0, b);
        else if (mirror) tma_store_3d(tm1, stage + BUF, m0, c, b);
        bulk_commit_group();
      }
    }
  }
  return true;
}

template <int PBN>
__global__ void __launch_bounds__(ORT_THREADS, 1)
    ortho_pair_kernel(const __grid_constant__ OrthoMaps maps, const __grid_constant__ OrthoArgs g) {
  using L = OrthoSmem<PBN>;
  constexpr int STAGES = L::STAGES, SLOTS = L::SLOTS;
  constexpr uint32_t PAIR_TX = 2u * static_cast<uint32_t>(L::A_STAGE + L::B_STAGE);

  extern __shared__ __align__(1024) unsigned char ortho_smem_raw[];
  unsigned char* smem = align_smem_1024(ortho_smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = full + 2 * STAGES;
  uint64_t* acc_empty = acc_full + SLOTS;
  uint64_t* drain = acc_empty + SLOTS;
  uint64_t* done = drain + 1;  // the epilogue warps have stored a phase
  uint64_t* go = drain + 2;    // every CTA has: the producer has seen the grid barrier
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = static_cast<int>(cluster_id_x()), pairs = static_cast<int>(gridDim.x) / 2;
  const int phases = 3 * g.steps;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < SLOTS; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * ORT_EPI_WARPS);
    }
    mbar_init(drain, 1);
    mbar_init(done, ORT_EPI_WARPS);
    mbar_init(go, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(ORT_TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_relaxed();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    if (lane == 0) {
      int stage = 0;
      uint32_t phase_bit = 0, issued_mask = 0, phase_mask = 0;
      bool ok = true;
      for (int ph = 0; ok && ph < phases; ++ph) {
        const int kind = ph % 3, cur = (ph / 3) & 1;
        const bool a_mn = kind == kGram && g.tall, b_mn = kind == kGram ? g.tall : kind == kUpdate && !g.tall;
        const CUtensorMap* ma = &maps.a[kind][cur];
        const CUtensorMap* mb = &maps.b[kind][cur];
        // The first phase reads what the kernel before has written.
        if (ph > 0) {
          if (!grid_wait(g.barrier, static_cast<unsigned>(ph) * gridDim.x, abort_flag)) {
            ok = false;
            break;
          }
          mbar_arrive(go);
        }
        for (int t = pair; ok && t < g.tiles[kind]; t += pairs) {
          int b, mt, nt;
          ortho_tile<PBN>(g, kind, t, b, mt, nt);
          const int m0 = mt * 2 * ORT_BM + static_cast<int>(rank) * ORT_BM;
          const int n0 = nt * PBN + static_cast<int>(rank) * (PBN / 2);
          for (int kb = 0; kb < g.k_blocks[kind]; ++kb) {
            if (!mbar_wait_bounded(&empty[stage], phase_bit ^ 1u, kDevErrWaitTimeoutEmpty, abort_flag)) {
              ok = false;
              break;
            }
            if (leader) mbar_arrive_expect_tx(&full[stage], PAIR_TX);
            const uint32_t mbar = map_to_rank(&full[stage], 0);
            unsigned char* sa = smem + L::OFF_A + stage * L::A_STAGE;
            unsigned char* sb = smem + L::OFF_B + stage * L::B_STAGE;
            const int k0 = kb * ORT_BK;
            if (a_mn) {
              for (int j = 0; j < ORT_BM / 64; ++j) tma_load_3d_pair(sa + j * 8192, ma, mbar, m0 + 64 * j, k0, b);
            } else {
              tma_load_3d_pair(sa, ma, mbar, k0, m0, b);
            }
            if (b_mn) {
              for (int j = 0; j < PBN / 128; ++j) tma_load_3d_pair(sb + j * 8192, mb, mbar, n0 + 64 * j, k0, b);
            } else {
              tma_load_3d_pair(sb, mb, mbar, k0, n0, b);
            }
            issued_mask |= 1u << stage;
            phase_mask = (phase_mask & ~(1u << stage)) | (phase_bit << stage);
            if (++stage == STAGES) stage = 0, phase_bit ^= 1u;
          }
        }
      }
      if (ok) {
        // No commit may still be on its way to this CTA's barriers.
        for (int i = 0; i < STAGES; ++i) {
          if ((issued_mask >> stage) & 1u)
            if (!mbar_wait_bounded(&empty[stage], phase_bit ^ 1u, kDevErrWaitTimeoutEmpty, abort_flag)) break;
          if (++stage == STAGES) stage = 0, phase_bit ^= 1u;
        }
      } else if (leader) {
        // Abort: let every phase this pair issued land.
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
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader && lane == 0) {
      int stage = 0, slot = 0;
      uint32_t phase_bit = 0, empty_bits = 0;
      bool ok = true, issued = false;
      for (int ph = 0; ok && ph < phases; ++ph) {
        const int kind = ph % 3;
        const bool a_mn = kind == kGram && g.tall, b_mn = kind == kGram ? g.tall : kind == kUpdate && !g.tall;
        const uint32_t idesc = make_idesc(0u, a_mn, b_mn, 2 * ORT_BM, PBN);
        const uint32_t a_step = a_mn ? 2048u : 32u, b_step = b_mn ? 2048u : 32u;
        const uint32_t a_lbo = a_mn ? 8192u : 16u, b_lbo = b_mn ? 8192u : 16u;
        for (int t = pair; ok && t < g.tiles[kind]; t += pairs) {
          if (!mbar_wait_bounded(&acc_empty[slot], ((empty_bits >> slot) & 1u) ^ 1u, kDevErrWaitTimeoutAccEmpty, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(slot * PBN);
          for (int kb = 0; kb < g.k_blocks[kind]; ++kb) {
            // A wait for the data may last as long as the phase before (another
            // pair's tiles), which the producer's own limit covers.
            if (!mbar_wait_bounded(&full[stage], phase_bit, kDevErrWaitTimeoutFull, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const uint32_t sa = smem_u32(smem + L::OFF_A + stage * L::A_STAGE);
            const uint32_t sb = smem_u32(smem + L::OFF_B + stage * L::B_STAGE);
#pragma unroll
            for (int kk = 0; kk < ORT_BK / 16; ++kk)
              umma_f16_pair(d_tmem, make_smem_desc_sw128(sa + kk * a_step, a_lbo, 1024),
                            make_smem_desc_sw128(sb + kk * b_step, b_lbo, 1024), idesc, (kb > 0 || kk > 0) ? 1u : 0u);
            issued = true;
            umma_commit_pair(&empty[stage]);
            if (++stage == STAGES) stage = 0, phase_bit ^= 1u;
          }
          if (!ok) break;
          umma_commit_pair(&acc_full[slot]);
          empty_bits ^= 1u << slot;
          slot = slot + 1 == SLOTS ? 0 : slot + 1;
        }
      }
      if (!ok && issued) {
        umma_commit_pair(drain);
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
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    constexpr int PART = PBN / 2;
    const int quarter = warp & 3, c0 = (warp - 2) / 4 * PART;
    unsigned char* stage = smem + L::OFF_C + (warp - 2) * 2 * 4096;
    int slot = 0;
    uint32_t full_bits = 0;
    bool ok = true;
    for (int ph = 0; ok && ph < phases; ++ph) {
      const int kind = ph % 3, step = ph / 3, cur = step & 1;
      const float alpha = g.alpha[step][kind], beta = g.beta[step][kind];
      // What the epilogue adds was written in the phases before.
      if (ph > 0) {
        const bool there = mbar_wait_bounded(go, static_cast<uint32_t>(ph - 1) & 1u, kDevErrGridBarrier, abort_flag);
        if (!__all_sync(0xffffffffu, there)) break;
      }
      for (int t = pair; ok && t < g.tiles[kind]; t += pairs) {
        int b, mt, nt;
        ortho_tile<PBN>(g, kind, t, b, mt, nt);
        const int m0 = mt * 2 * ORT_BM + static_cast<int>(rank) * ORT_BM + 32 * quarter, n0 = nt * PBN + c0;
        const uint32_t t_row = tmem_base + (static_cast<uint32_t>(32 * quarter) << 16) + static_cast<uint32_t>(slot * PBN + c0);
        auto wait = [&] {
          const bool done = mbar_wait_bounded(&acc_full[slot], (full_bits >> slot) & 1u, kDevErrWaitTimeoutAccFull, abort_flag);
          tc_fence_after_sync();
          return static_cast<bool>(__all_sync(0xffffffffu, done));
        };
        auto release = [&] {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(map_to_rank(&acc_empty[slot], 0));
        };
        if (kind == kUpdate) {
          const int64_t off = b * g.stride_x;
          ok = ortho_epilogue<true, PART>(t_row, n0, m0, b, g.tall ? g.q : g.p, g.tall ? g.p : g.q, alpha, beta, g.x[cur] + off,
                                          g.lo + off, g.ldx, false, &maps.x[cur ^ 1], &maps.lo, stage, lane, wait, release);
        } else {
          const bool below = (nt + 1) * PBN <= mt * 2 * ORT_BM;
          const __half* add = g.gram + b * g.stride_p;
          ok = ortho_epilogue<false, PART>(t_row, n0, m0, b, g.p, g.p, alpha, kind == kPoly ? beta : 0.f, add, add, g.ldp, below,
                                           kind == kPoly ? &maps.poly : &maps.gram, kind == kPoly ? &maps.poly_t : &maps.gram_t,
                                           stage, lane, wait, release);
        }
        if (!ok) break;
        full_bits ^= 1u << slot;
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
      }
      if (!ok) break;
      // This CTA's share of the phase is in memory.
      if (lane == 0 && ph + 1 < phases) {
        bulk_wait_group<0>();
        fence_proxy_async_all();
        mbar_arrive(done);
        if (warp == 2 && mbar_wait_bounded(done, static_cast<uint32_t>(ph) & 1u, kDevErrGridBarrier, abort_flag)) {
          __threadfence();
          red_release_gpu(g.barrier);
        }
      }
      __syncwarp();
    }
    if (lane == 0) bulk_wait_group<0>();
    __syncwarp();
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_relaxed();  // the partner is done with this CTA's shared memory, barriers and TMEM
  if (warp == 1) {
    tc_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(ORT_TMEM_COLS) : "memory");
  }
}

// ---------------------------------------------------------------- in and out
// A stack of row-major matrices of any type, stride and alignment.
struct OrthoTensor {
  void* p;
  int dtype;  // CUOPX_*; -1: none
  int vec;    // rows start on 16-byte boundaries
  int64_t ld, stride;
};

// Eight elements from column c on, zeros from column n on.
__device__ __forceinline__ void ortho_load8(const OrthoTensor& t, int64_t b, int64_t row, int64_t c, int64_t n, float (&v)[8]) {
  const int64_t at = b * t.stride + row * t.ld + c;
  if (t.dtype == CUOPX_F32) {
    const float* p = static_cast<const float*>(t.p) + at;
    if (t.vec && c + 8 <= n) {
      const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < n ? p[i] : 0.f;
    }
    return;
  }
  const unsigned short* p = static_cast<const unsigned short*>(t.p) + at;
  uint32_t w[4] = {};
  if (t.vec && c + 8 <= n) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) w[i / 2] |= static_cast<uint32_t>(p[i]) << (16 * (i & 1));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = t.dtype == CUOPX_BF16 ? unpack2_layer<__nv_bfloat16>(w[i]) : unpack2_layer<__half>(w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}

// Rounds eight elements to the tensor's type, in v too, and stores those before column n.
__device__ __forceinline__ void ortho_store8(const OrthoTensor& t, int64_t b, int64_t row, int64_t c, int64_t n, float (&v)[8]) {
  const int64_t at = b * t.stride + row * t.ld + c;
  if (t.dtype == CUOPX_F32) {
    float* p = static_cast<float*>(t.p) + at;
    if (t.vec && c + 8 <= n) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < n) p[i] = v[i];
    }
    return;
  }
  unsigned short* p = static_cast<unsigned short*>(t.p) + at;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool bf = t.dtype == CUOPX_BF16;
    w[i] = bf ? pack2_layer<__nv_bfloat16>(v[2 * i], v[2 * i + 1]) : pack2_layer<__half>(v[2 * i], v[2 * i + 1]);
    const float2 f = bf ? unpack2_layer<__nv_bfloat16>(w[i]) : unpack2_layer<__half>(w[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
  if (t.vec && c + 8 <= n) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) p[i] = static_cast<unsigned short>(w[i / 2] >> (16 * (i & 1)));
  }
}

struct OrthoIo {
  int64_t rows, cols, groups;  // groups: of eight columns in a row
  int blocks;                  // CTAs to a matrix
  OrthoTensor g, m, w;         // gradient; momentum; weight, or the result
  float mu;
  int nesterov;
  double* partial;    // [batch][blocks] sums of squares
  unsigned* barrier;  // of ortho_pair_kernel
  float x_scale;      // of the stored X0
  double eps;
  __half* hi;
  __half* lo;
  int64_t ldx, stride_x;
  float out;        // of the result, X's scale taken out: or
  float keep, step;  // w = keep w - step * X (before lr_dev)
  float decay;
  const float* lr_dev;
};

// What is orthogonalised, from the momentum as stored.
__device__ __forceinline__ void ortho_update8(const OrthoIo& p, const float (&m)[8], float (&g)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = p.nesterov ? fmaf(p.mu, m[i], g[i]) : m[i];
}

// Momentum <- mu momentum + gradient, and the sum of the squares of what is
// orthogonalised: in 64 bits, which neither large nor small numbers leave.
__global__ void __launch_bounds__(256) ortho_sum_kernel(const OrthoIo p) {
  __shared__ double part[8];
  const int64_t b = blockIdx.y, n = p.rows * p.groups;
  grid_dependency_wait();
  if (blockIdx.x == 0 && b == 0 && threadIdx.x == 0) *p.barrier = 0u;
  double s = 0.0;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < n; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = e / p.groups, c = (e - row * p.groups) * 8;
    float g[8];
    ortho_load8(p.g, b, row, c, p.cols, g);
    if (p.m.dtype >= 0) {
      float m[8];
      ortho_load8(p.m, b, row, c, p.cols, m);
#pragma unroll
      for (int i = 0; i < 8; ++i) m[i] = fmaf(p.mu, m[i], g[i]);
      ortho_store8(p.m, b, row, c, p.cols, m);
      ortho_update8(p, m, g);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fma(static_cast<double>(g[i]), static_cast<double>(g[i]), s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) s += part[i];
    p.partial[b * p.blocks + blockIdx.x] = s;
  }
}

// X0 = G / (||G|| + eps), times its scale, as hi + lo.
__global__ void __launch_bounds__(256) ortho_scale_kernel(const OrthoIo p) {
  __shared__ double part[256];
  const int64_t b = blockIdx.y, n = p.rows * p.groups;
  grid_dependency_wait();
  double s = 0.0;
  for (int i = threadIdx.x; i < p.blocks; i += 256) s += p.partial[b * p.blocks + i];
  part[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
    __syncthreads();
  }
  // Small gradients: the factor leaves fp32's range below a norm of 1e-34, and is split.
  const double factor = p.x_scale / (sqrt(part[0]) + p.eps);
  const float pre = factor > 0x1p100 ? 0x1p100f : 1.f;
  const float f = static_cast<float>(factor > 0x1p100 ? factor * 0x1p-100 : factor);
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < n; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = e / p.groups, c = (e - row * p.groups) * 8;
    float g[8];
    ortho_load8(p.g, b, row, c, p.cols, g);
    if (p.m.dtype >= 0) {
      float m[8];
      ortho_load8(p.m, b, row, c, p.cols, m);
      ortho_update8(p, m, g);
    }
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = make_float2(g[2 * i] * pre * f, g[2 * i + 1] * pre * f);
      h[i] = pack2_layer<__half>(v.x, v.y);
      const float2 r = unpack2_layer<__half>(h[i]);
      l[i] = pack2_layer<__half>(v.x - r.x, v.y - r.y);
    }
    const int64_t at = b * p.stride_x + row * p.ldx + c;
    *reinterpret_cast<uint4*>(p.hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(p.lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// The result, or the weight's step.
__global__ void __launch_bounds__(256) ortho_out_kernel(const OrthoIo p, int update) {
  const int64_t b = blockIdx.y, n = p.rows * p.groups;
  grid_dependency_wait();
  float keep = p.keep, step = p.step;
  if (update && p.lr_dev) {
    const float lr = *p.lr_dev;
    keep = 1.f - lr * p.decay;
    step *= lr;
  }
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < n; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = e / p.groups, c = (e - row * p.groups) * 8;
    const int64_t at = b * p.stride_x + row * p.ldx + c;
    const uint4 h4 = *reinterpret_cast<const uint4*>(p.hi + at), l4 = *reinterpret_cast<const uint4*>(p.lo + at);
    const uint32_t h[4] = {h4.x, h4.y, h4.z, h4.w}, l[4] = {l4.x, l4.y, l4.z, l4.w};
    float v[8], w[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = add2(unpack2_layer<__half>(h[i]), unpack2_layer<__half>(l[i]));
      v[2 * i] = x.x, v[2 * i + 1] = x.y;
    }
    if (update) {
      ortho_load8(p.w, b, row, c, p.cols, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf(-step, v[i], keep * w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= p.out;
    }
    ortho_store8(p.w, b, row, c, p.cols, v);
  }
}

// ---------------------------------------------------------------- host
// Largest |a s + b s^3 + c s^5| for 0 <= s <= m, and |b t + c t^2| for 0 <= t <= m^2.
double quintic_bound(const double* k, double m) {
  auto f = [&](double s) { return std::fabs(s * (k[0] + s * s * (k[1] + s * s * k[2]))); };
  double best = f(m);
  // Zeros of the derivative: a + 3 b t + 5 c t^2, t = s^2.
  const double qa = 5 * k[2], qb = 3 * k[1], qc = k[0];
  double t[2] = {-1, -1};
  if (qa != 0) {
    const double d = qb * qb - 4 * qa * qc;
    if (d >= 0) t[0] = (-qb + std::sqrt(d)) / (2 * qa), t[1] = (-qb - std::sqrt(d)) / (2 * qa);
  } else if (qb != 0) {
    t[0] = -qc / qb;
  }
  for (double r : t)
    if (r > 0 && r < m * m) best = std::max(best, f(std::sqrt(r)));
  return best;
}
double quadratic_bound(const double* k, double t) {
  auto f = [&](double x) { return std::fabs(x * (k[1] + x * k[2])); };
  double best = f(t);
  if (k[2] != 0) {
    const double r = -k[1] / (2 * k[2]);
    if (r > 0 && r < t) best = std::max(best, f(r));
  }
  return best;
}
// The power of two that takes a bound to 2^14 .. 2^15: rounding errors have a factor of two to fp16's largest number.
double half_scale(double bound) { return bound > 0 ? std::ldexp(1.0, 15 - static_cast<int>(std::ceil(std::log2(bound)))) : 1.0; }

// Bounds on the singular values beyond this are refused: the polynomial does not
// bring them towards 1, and fp32 sums would soon leave their range.
constexpr double kOrthoMaxBound = 1024.0;

struct OrthoSchedule {
  float alpha[ORT_MAX_STEPS][3], beta[ORT_MAX_STEPS][3];
  double first, last;  // scales of X0 and of the result
};

// Singular values of X0 are at most 1, its Frobenius norm.
bool ortho_schedule(const double* coefficients, int steps, OrthoSchedule& o) {
  double m = 1.0, sx = half_scale(m);
  o.first = sx;
  for (int i = 0; i < steps; ++i) {
    const double* k = coefficients + 3 * i;
    for (int j = 0; j < 3; ++j)
      if (!std::isfinite(k[j])) return false;
    const double poly = quadratic_bound(k, m * m), next = quintic_bound(k, m);
    if (!(poly <= kOrthoMaxBound * kOrthoMaxBound) || !(next <= kOrthoMaxBound)) return false;
    const double sa = half_scale(m * m), sp = half_scale(poly), sn = half_scale(std::max(next, 0x1p-20));
    o.alpha[i][kGram] = static_cast<float>(sa / (sx * sx));
    o.beta[i][kGram] = 0.f;
    o.alpha[i][kPoly] = static_cast<float>(sp * k[2] / (sa * sa));
    o.beta[i][kPoly] = static_cast<float>(sp * k[1] / sa);
    o.alpha[i][kUpdate] = static_cast<float>(sn / (sp * sx));
    o.beta[i][kUpdate] = static_cast<float>(sn * k[0] / sx);
    m = std::max(next, 0x1p-20);
    sx = sn;
  }
  o.last = sx;
  return true;
}

struct OrthoPlan {
  int64_t batch, p, q, ldx, stride_x, ldp, stride_p;
  bool tall;
  int blocks;
  int64_t groups;
  size_t barrier_off, partial_off, hi_off[2], lo_off, gram_off, poly_off, bytes;
};

OrthoPlan ortho_plan(int64_t batch, int64_t rows, int64_t cols) {
  OrthoPlan o = {};
  if (batch <= 0 || rows <= 0 || cols <= 0) return o;
  o.batch = batch;
  o.tall = rows > cols;
  o.p = std::min(rows, cols), o.q = std::max(rows, cols);
  o.ldx = round8(cols), o.stride_x = rows * o.ldx;
  o.ldp = round8(o.p), o.stride_p = o.p * o.ldp;
  o.groups = (cols + 7) / 8;
  // About eight CTAs of 256 threads per SM over the whole stack, at least two groups a thread.
  const int64_t most = std::max<int64_t>(1, device_sm_count() * 8 / batch);
  o.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, rows * o.groups / 512)));
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += round256(bytes);
    return at;
  };
  o.barrier_off = take(4);
  o.partial_off = take(static_cast<size_t>(batch) * o.blocks * 8);
  for (int i = 0; i < 2; ++i) o.hi_off[i] = take(static_cast<size_t>(batch) * o.stride_x * 2);
  o.lo_off = take(static_cast<size_t>(batch) * o.stride_x * 2);
  o.gram_off = take(static_cast<size_t>(batch) * o.stride_p * 2);
  o.poly_off = take(static_cast<size_t>(batch) * o.stride_p * 2);
  o.bytes = off;
  return o;
}

template <int PBN>
int launch_ortho_pairs(const OrthoPlan& o, const OrthoSchedule& sched, int steps, char* ws, cudaStream_t stream) {
  using L = OrthoSmem<PBN>;
  auto kern = ortho_pair_kernel<PBN>;
  static std::atomic<int> capacity[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return CUOPX_CUDA_ERROR;
  if (capacity[dev].load(std::memory_order_acquire) == 0) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::ALLOC) != cudaSuccess)
      return CUOPX_CUDA_ERROR;
    const int n = cluster_capacity(kern, ORT_THREADS, L::ALLOC, 2);
    if (n <= 0) return cuda_failure_text("no room for a CTA pair");
    capacity[dev].store(n, std::memory_order_release);
  }
  const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  __half* hi[2] = {reinterpret_cast<__half*>(ws + o.hi_off[0]), reinterpret_cast<__half*>(ws + o.hi_off[1])};
  __half* lo = reinterpret_cast<__half*>(ws + o.lo_off);
  __half* gram = reinterpret_cast<__half*>(ws + o.gram_off);
  __half* poly = reinterpret_cast<__half*>(ws + o.poly_off);
  const int64_t xr = o.tall ? o.q : o.p, xc = o.tall ? o.p : o.q;  // X as stored
  OrthoMaps m;
  bool ok = true;
  auto map_x = [&](CUtensorMap* t, const __half* x, int inner, int rows) {
    ok &= make_map(t, dt, x, xc, xr, o.batch, o.ldx, o.stride_x, inner, rows);
  };
  auto map_p = [&](CUtensorMap* t, const __half* x, int inner, int rows) {
    ok &= make_map(t, dt, x, o.p, o.p, o.batch, o.ldp, o.stride_p, inner, rows);
  };
  for (int i = 0; i < 2; ++i) {
    // K-major operands come in boxes of 64 x rows, MN-major ones in 64 x 64.
    map_x(&m.a[kGram][i], hi[i], 64, o.tall ? ORT_BK : ORT_BM);
    map_x(&m.b[kGram][i], hi[i], 64, o.tall ? ORT_BK : PBN / 2);
    map_p(&m.a[kPoly][i], gram, 64, ORT_BM);
    map_p(&m.b[kPoly][i], gram, 64, PBN / 2);
    if (o.tall) {
      map_x(&m.a[kUpdate][i], hi[i], 64, ORT_BM);
      map_p(&m.b[kUpdate][i], poly, 64, PBN / 2);
    } else {
      map_p(&m.a[kUpdate][i], poly, 64, ORT_BM);
      map_x(&m.b[kUpdate][i], hi[i], 64, ORT_BK);
    }
    map_x(&m.x[i], hi[i], 64, 32);
  }
  map_x(&m.lo, lo, 64, 32);
  map_p(&m.gram, gram, 64, 32);
  map_p(&m.poly, poly, 64, 32);
  ok &= make_map_es(&m.gram_t, dt, 2, gram, o.p, o.p, o.batch, o.ldp, o.stride_p, 32, 64, CU_TENSOR_MAP_SWIZZLE_NONE);
  ok &= make_map_es(&m.poly_t, dt, 2, poly, o.p, o.p, o.batch, o.ldp, o.stride_p, 32, 64, CU_TENSOR_MAP_SWIZZLE_NONE);
  if (!ok) return CUOPX_CUDA_ERROR;
  OrthoArgs a = {};
  a.batch = static_cast<int>(o.batch);
  a.p = static_cast<int>(o.p), a.q = static_cast<int>(o.q);
  a.steps = steps;
  a.tall = o.tall;
  a.tiles_m = static_cast<int>((xr + 255) / 256), a.tiles_n = static_cast<int>((xc + PBN - 1) / PBN);
  // Symmetric phases: row tile i has min(256 / PBN (i + 1), all) column tiles.
  const int64_t rows = (o.p + 255) / 256;
  a.sym_tiles = static_cast<int>(256 / PBN * (rows * (rows + 1) / 2));
  a.tiles[kGram] = a.tiles[kPoly] = a.batch * a.sym_tiles;
  a.tiles[kUpdate] = a.batch * a.tiles_m * a.tiles_n;
  a.k_blocks[kGram] = static_cast<int>((o.q + ORT_BK - 1) / ORT_BK);
  a.k_blocks[kPoly] = a.k_blocks[kUpdate] = static_cast<int>((o.p + ORT_BK - 1) / ORT_BK);
  a.x[0] = hi[0], a.x[1] = hi[1], a.lo = lo, a.gram = gram;
  a.ldx = o.ldx, a.stride_x = o.stride_x, a.ldp = o.ldp, a.stride_p = o.stride_p;
  a.barrier = reinterpret_cast<unsigned*>(ws + o.barrier_off);
  for (int i = 0; i < steps; ++i)
    for (int j = 0; j < 3; ++j) a.alpha[i][j] = sched.alpha[i][j], a.beta[i][j] = sched.beta[i][j];
  // Cooperative: all CTAs run at once, whatever else the GPU does.
  cudaLaunchConfig_t cfg = {};
  const int pairs = std::min(capacity[dev].load(std::memory_order_relaxed), std::max(a.tiles[kGram], a.tiles[kUpdate]));
  cfg.gridDim = dim3(static_cast<unsigned>(2 * pairs));
  cfg.blockDim = dim3(ORT_THREADS);
  cfg.dynamicSmemBytes = L::ALLOC;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeCooperative;
  attr[1].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, m, a); err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  note_launch(PBN == 256 ? "ortho_pair_256x256" : "ortho_pair_256x128");
  return check_launch();
}

OrthoTensor ortho_tensor(const void* p, int dtype, int64_t ld, int64_t stride, int64_t batch, int64_t rows) {
  OrthoTensor t = {const_cast<void*>(p), p ? dtype : -1, 0, ld, stride};
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  t.vec = reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || ld * es % 16 == 0) && (batch == 1 || stride * es % 16 == 0);
  return t;
}

// All launches of a call.  `io` has the tensors and what the last pass does.
int ortho_run(OrthoIo io, const OrthoPlan& o, const double* coefficients, int steps, bool update, double out_factor, void* workspace,
              cudaStream_t stream) {
  OrthoSchedule sched;
  if (!ortho_schedule(coefficients, steps, sched)) return CUOPX_INVALID_ARGUMENT;
  char* ws = static_cast<char*>(workspace);
  io.groups = o.groups;
  io.blocks = o.blocks;
  io.partial = reinterpret_cast<double*>(ws + o.partial_off);
  io.barrier = reinterpret_cast<unsigned*>(ws + o.barrier_off);
  io.x_scale = static_cast<float>(sched.first);
  io.ldx = o.ldx, io.stride_x = o.stride_x;
  io.lo = reinterpret_cast<__half*>(ws + o.lo_off);
  io.hi = reinterpret_cast<__half*>(ws + o.hi_off[0]);
  const dim3 grid(static_cast<unsigned>(o.blocks), static_cast<unsigned>(o.batch));
  cudaError_t err = launch_pdl(ortho_sum_kernel, grid, dim3(256), 0, stream, io);
  note_launch("ortho_sum");
  if (err == cudaSuccess) err = launch_pdl(ortho_scale_kernel, grid, dim3(256), 0, stream, io);
  note_launch("ortho_scale");
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  if (steps > 0) {
    const int rc = o.q >= 2048 ? launch_ortho_pairs<256>(o, sched, steps, ws, stream) : launch_ortho_pairs<128>(o, sched, steps, ws, stream);
    if (rc != CUOPX_SUCCESS) return rc;
  }
  io.hi = reinterpret_cast<__half*>(ws + o.hi_off[steps & 1]);
  io.out = static_cast<float>(out_factor / sched.last);
  io.step = static_cast<float>(out_factor / sched.last);
  err = launch_pdl(ortho_out_kernel, grid, dim3(256), 0, stream, io, update ? 1 : 0);
  note_launch(update ? "ortho_step" : "ortho_out");
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  return check_launch();
}

bool ortho_type_ok(int dtype) { return dtype == CUOPX_F32 || dtype == CUOPX_F16 || dtype == CUOPX_BF16; }

// A stack of matrices: rows that do not overlap, matrices one after the other
// or side by side in wider rows (stride < ld: column slices of one buffer).
bool ortho_layout_ok(const void* p, int dtype, int64_t ld, int64_t stride, int64_t batch, int64_t rows, int64_t cols) {
  if (!p || !starts_on(dtype_size(dtype), p) || (rows > 1 && ld < cols)) return false;
  if (!extent_ok(rows, std::max(ld, cols))) return false;
  if (batch == 1) return true;
  if (stride <= 0 || !extent_ok(batch, stride)) return false;
  const int64_t span = rows > 1 ? (rows - 1) * ld + cols : cols;
  return stride >= span || (stride >= cols && batch <= ld / stride + (ld % stride >= cols ? 1 : 0));
}

size_t ortho_span(int dtype, int64_t ld, int64_t stride, int64_t batch, int64_t rows, int64_t cols) {
  return static_cast<size_t>((batch - 1) * (batch > 1 ? stride : 0) + (rows > 1 ? (rows - 1) * ld : 0) + cols) * dtype_size(dtype);
}

bool ortho_sizes_ok(int64_t batch, int64_t rows, int64_t cols) {
  if (batch < 0 || rows < 0 || cols < 0) return false;
  if (batch > 65535 || rows > (1 << 24) || cols > (1 << 24)) return false;
  // Tiles of a phase are counted in 32 bits.
  const double p = static_cast<double>(std::min(rows, cols)) / 128 + 1, q = static_cast<double>(std::max(rows, cols)) / 128 + 1;
  return static_cast<double>(batch) * p * q < double(1 << 30);
}

int orthogonalize(const cuopx_orthogonalize_args* a, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (!ortho_type_ok(a->dtype) || !ortho_type_ok(a->out_dtype)) return CUOPX_UNSUPPORTED_TYPE;
  if (a->steps < 0 || a->steps > ORT_MAX_STEPS || a->reserved != 0 || !(a->eps >= 0) || !std::isfinite(a->eps) ||
      (a->steps > 0 && !a->coefficients) || !ortho_sizes_ok(a->batch, a->rows, a->cols))
    return CUOPX_INVALID_ARGUMENT;
  OrthoSchedule sched;
  if (!ortho_schedule(a->coefficients, a->steps, sched)) return CUOPX_INVALID_ARGUMENT;
  if (a->batch == 0 || a->rows == 0 || a->cols == 0) return CUOPX_SUCCESS;
  if (!ortho_layout_ok(a->G, a->dtype, a->ldg, a->strideG, a->batch, a->rows, a->cols) ||
      !ortho_layout_ok(a->out, a->out_dtype, a->ldo, a->strideO, a->batch, a->rows, a->cols) || !starts_on(256, a->workspace))
    return CUOPX_INVALID_ARGUMENT;
  const OrthoPlan o = ortho_plan(a->batch, a->rows, a->cols);
  if (!a->workspace || a->workspace_bytes < o.bytes) return CUOPX_RESOURCE_UNAVAILABLE;
  const size_t g_span = ortho_span(a->dtype, a->ldg, a->strideG, a->batch, a->rows, a->cols);
  const size_t o_span = ortho_span(a->out_dtype, a->ldo, a->strideO, a->batch, a->rows, a->cols);
  const bool same = a->G == a->out && a->dtype == a->out_dtype && (a->rows == 1 || a->ldg == a->ldo) &&
                    (a->batch == 1 || a->strideG == a->strideO);
  if (!same && overlaps(a->G, g_span, a->out, o_span)) return CUOPX_INVALID_ARGUMENT;
  if (overlaps(a->workspace, o.bytes, a->G, g_span) || overlaps(a->workspace, o.bytes, a->out, o_span)) return CUOPX_INVALID_ARGUMENT;
  OrthoIo io = {};
  io.rows = a->rows, io.cols = a->cols;
  io.g = ortho_tensor(a->G, a->dtype, a->ldg, a->strideG, a->batch, a->rows);
  io.m.dtype = -1;
  io.w = ortho_tensor(a->out, a->out_dtype, a->ldo, a->strideO, a->batch, a->rows);
  io.eps = a->eps;
  return ortho_run(io, o, a->coefficients, a->steps, false, 1.0, a->workspace, stream);
}

int muon_step(const cuopx_muon_args* a, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (!ortho_type_ok(a->wdtype) || !ortho_type_ok(a->gdtype) || !ortho_type_ok(a->mdtype)) return CUOPX_UNSUPPORTED_TYPE;
  if (a->steps < 0 || a->steps > ORT_MAX_STEPS || (a->nesterov != 0 && a->nesterov != 1) || a->reserved != 0 || !(a->eps >= 0) ||
      (a->steps > 0 && !a->coefficients) || !ortho_sizes_ok(a->batch, a->rows, a->cols))
    return CUOPX_INVALID_ARGUMENT;
  for (double v : {a->eps, a->lr, a->mu, a->decay, a->scale})
    if (!std::isfinite(v)) return CUOPX_INVALID_ARGUMENT;
  OrthoSchedule sched;
  if (!ortho_schedule(a->coefficients, a->steps, sched)) return CUOPX_INVALID_ARGUMENT;
  if (a->batch == 0 || a->rows == 0 || a->cols == 0) return CUOPX_SUCCESS;
  const struct {
    const void* p;
    int dtype;
    int64_t ld, stride;
  } t[3] = {{a->W, a->wdtype, a->ldw, a->strideW}, {a->momentum, a->mdtype, a->ldm, a->strideM}, {a->G, a->gdtype, a->ldg, a->strideG}};
  for (const auto& x : t)
    if (!ortho_layout_ok(x.p, x.dtype, x.ld, x.stride, a->batch, a->rows, a->cols)) return CUOPX_INVALID_ARGUMENT;
  if (!starts_on(256, a->workspace) || !starts_on(4, a->lr_dev)) return CUOPX_INVALID_ARGUMENT;
  const OrthoPlan o = ortho_plan(a->batch, a->rows, a->cols);
  if (!a->workspace || a->workspace_bytes < o.bytes) return CUOPX_RESOURCE_UNAVAILABLE;
  size_t span[3];
  for (int i = 0; i < 3; ++i) {
    span[i] = ortho_span(t[i].dtype, t[i].ld, t[i].stride, a->batch, a->rows, a->cols);
    for (int j = 0; j < i; ++j)
      if (overlaps(t[i].p, span[i], t[j].p, span[j])) return CUOPX_INVALID_ARGUMENT;
    if (overlaps(a->workspace, o.bytes, t[i].p, span[i])) return CUOPX_INVALID_ARGUMENT;
    if (i < 2 && overlaps(a->lr_dev, 4, t[i].p, span[i])) return CUOPX_INVALID_ARGUMENT;
  }
  if (overlaps(a->workspace, o.bytes, a->lr_dev, 4)) return CUOPX_INVALID_ARGUMENT;
  OrthoIo io = {};
  io.rows = a->rows, io.cols = a->cols;
  io.w = ortho_tensor(a->W, a->wdtype, a->ldw, a->strideW, a->batch, a->rows);
  io.m = ortho_tensor(a->momentum, a->mdtype, a->ldm, a->strideM, a->batch, a->rows);
  io.g = ortho_tensor(a->G, a->gdtype, a->ldg, a->strideG, a->batch, a->rows);
  io.mu = static_cast<float>(a->mu);
  io.nesterov = a->nesterov;
  io.eps = a->eps;
  io.lr_dev = a->lr_dev;
  io.decay = static_cast<float>(a->lr * a->decay);
  io.keep = static_cast<float>(1.0 - a->lr * a->decay);
  return ortho_run(io, o, a->coefficients, a->steps, true, a->lr * a->scale, a->workspace, stream);
}

}  // namespace

}  // namespace cuopx

extern "C" {

size_t cuopx_orthogonalize_workspace_size(int64_t batch, int64_t rows, int64_t cols) {
  return cuopx::ortho_sizes_ok(batch, rows, cols) ? cuopx::ortho_plan(batch, rows, cols).bytes : 0;
}

int cuopx_orthogonalize(const cuopx_orthogonalize_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_orthogonalize", args ? args->rows : 0, args ? args->cols : 0, args ? args->steps : 0,
                        args ? args->batch : 0);
  return scope.done(cuopx::orthogonalize(args, static_cast<cudaStream_t>(stream)));
}

int cuopx_muon_step(const cuopx_muon_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_muon_step", args ? args->rows : 0, args ? args->cols : 0, args ? args->steps : 0,
                        args ? args->batch : 0);
  return scope.done(cuopx::muon_step(args, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
