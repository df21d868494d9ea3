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
// That is with operands of 11 bits, for results in bf16, whose rounding is above it.  With 22 (FULL),
// for fp16 and fp32, A and P are kept as hi + lo too, and every product is hi lo + lo hi + hi hi, one
// after the other along a depth three times as long; lo lo is 2^-24 of the sum.  What
// remains is the tensor cores' fp32 sums, 5e-6 (64 x 3000) to 2e-4 (8192 x 28672) of the result, growing
// with the depth.  Whole calls in fp32, us with 11 / 22 bits: 1024 x 1024 162 / 310, 5001 x 1777 494 / 1051,
// 4096 x 10240 2527 / 7187.
//
// One persistent launch does all products: tiles of 256 x 256 or 256 x 128 on CTA
// pairs (tcgen05 cta_group::2), tile i of a phase on pair i mod the number of pairs,
// grid barriers between phases.  A and the polynomial are symmetric: tiles on or below
// the diagonal are computed, and those below it stored twice, once transposed.
// Where A has few tiles and X is long, several pairs share a tile of X X^T, a part of the
// depth each (ortho_split_epilogue).
//   warps 0, 10  TMA producers of the two operands (both CTAs)
//   warp 1       TMEM allocation; MMA issuer (even CTA)
//   warps 2-9    epilogue: alpha * sums + beta * (what the phase adds), rounded
// Producers and issuer walk their loops as whole warps and let one elected lane
// issue, with the next stage's barrier tested a stage ahead: what they compute then
// stays in uniform registers, which TMA and MMA instructions take.  One producer
// thread for both operands under `lane == 0` took 305 ns a stage, more than twice
// what the tensor cores need for 256 x 128 x 64 (now 250; 256 x 256 x 64 300).
//
// Measured, whole calls, bf16 (11 bits), work with symmetric products counted by halves: 1024 x 1024 162
// us, of which 15 phases of about 10 us (4.4 with nothing to compute); 5001 x 1777 490 us
// (540 TFLOP/s); eight 2048 x 2048 1.39 ms (990); 8192 x 28672 28 ms (1.1 PFLOP/s, at the
// power cap).  Middle sizes are bound by L2: 256-wide tiles pull 10 TB/s from it.
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
constexpr int ORT_THREADS = 32 * (3 + ORT_EPI_WARPS);
constexpr uint32_t ORT_TMEM_COLS = 512;
constexpr int ORT_SLOTS = 2;  // accumulators of up to 256 columns

// The ring of operand stages: A's 128 rows, then B's columns of this CTA, 64 of K
// each.  Tiles of 512 columns (two MMAs of 256) have three stages of 48 KB, the
// others five of 32 KB.  It is divided anew where a phase starts: nothing of
// the phase before is on its way then.
struct OrthoSmem {
  static constexpr int STAGES = 5, WIDE_STAGES = 3;
  static constexpr int OPERAND = ORT_BM * ORT_BK * 2;  // 16 KB: A, or B of one MMA
  static constexpr int OFF_C = STAGES * 2 * OPERAND;   // per epilogue warp: two staging buffers of 4 KB
  static_assert(WIDE_STAGES * 3 * OPERAND <= OFF_C, "the ring");
  static constexpr int OFF_BAR = OFF_C + ORT_EPI_WARPS * 2 * 4096;
  static constexpr int NUM_BARS = 2 * STAGES + 2 * ORT_SLOTS + 3;  // full, empty, acc_full, acc_empty, drain, done, go
  static constexpr int OFF_MISC = OFF_BAR + NUM_BARS * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;
  static_assert(ALLOC <= 232448, "shared memory budget exceeded");
};

// The three phases of a step: A = X X^T, the polynomial P = bA + cAA, X <- aX + PX.
enum OrthoPhase { kGram = 0, kPoly = 1, kUpdate = 2 };

template <bool FULL>
struct OrthoMaps {
  // Operands: hi, and with FULL lo; [phase], for the two buffers that X alternates between.
  CUtensorMap a[FULL ? 2 : 1][3][2], b[FULL ? 2 : 1][3][2];
};

struct OrthoArgs {
  int batch, p, q, steps;
  bool tall;
  int width[3];     // columns of a phase's tiles: 128, 256 or 512
  int tiles[3];     // of a phase, all batches
  int k_blocks[3];  // of one product
  int tiles_m, tiles_n;  // of the update, one batch
  int sym_tiles[2];      // of the other two, one batch
  int splits;            // pairs that share a tile of kGram: 1, or 2 to 8 with a tile for every pair at most
  float* partial;        // their sums: [tile][pair of these][warp][column][32 rows]
  unsigned* tickets;     // [tile][warp]: pairs that have stored theirs
  __half* x[2];
  __half* lo[2];  // the same buffer twice where no product reads it
  __half* gram;
  __half* poly;
  __half* gram_lo;  // FULL
  __half* poly_lo;
  int64_t ldx, stride_x, ldp, stride_p;  // elements
  unsigned* barrier;
  // Of any wait: a second, and ten times what the largest phase takes, since a pair
  // waits for the others' tiles.
  unsigned long long limit_ns;
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
__device__ __forceinline__ bool grid_wait(const unsigned* barrier, unsigned count, volatile int* abort, unsigned long long limit_ns) {
  const unsigned long long t0 = global_timer_ns();
  for (uint32_t it = 0; ld_acquire_gpu(barrier) < count; ++it) {
    __nanosleep(40);
    if ((it & 63u) == 63u) {
      if (*abort) return false;
      if (global_timer_ns() - t0 > limit_ns) {
        record_device_error(kDevErrGridBarrier);
        *abort = 1;
        return false;
      }
    }
  }
  fence_proxy_async_all();
  return true;
}

// A whole warp's bounded wait, with one answer for all lanes; `ready`: a test has said so already.
__device__ __forceinline__ bool warp_wait(bool ready, uint64_t* bar, uint32_t parity, int err, volatile int* abort,
                                          unsigned long long limit_ns) {
  return __all_sync(0xffffffffu, ready || mbar_wait_bounded(bar, parity, err, abort, limit_ns));
}

// Tile t of a phase: batch, first row, first column.  Symmetric phases have the
// tiles whose first column is at most their last row.
__device__ __forceinline__ void ortho_tile(const OrthoArgs& g, int phase, int t, int& b, int& m, int& n) {
  const int width = g.width[phase];
  if (phase == kUpdate) {
    const int per = g.tiles_m * g.tiles_n;
    b = t / per;
    const int r = t - b * per;
    constexpr int GROUP = 8;  // row tiles that share the columns' operand while it is in L2
    const int span = GROUP * g.tiles_n, grp = r / span, first = grp * GROUP;
    const int rows = min(GROUP, g.tiles_m - first), rr = r - grp * span;
    m = (first + rr % rows) * 256;
    n = rr / rows * width;
  } else {
    // Row tile i has ceil((i + 1) 256 / width) tiles.
    b = t / g.sym_tiles[phase];
    const int r = t - b * g.sym_tiles[phase];
    auto before = [&](int i) {  // tiles in the row tiles before i
      const int64_t h = i >> 1;
      if (width == 512) return static_cast<int>(h * (h + 1) + (i & 1) * (h + 1));
      return (256 / width) * (i * (i + 1) / 2);
    };
    int i = static_cast<int>(sqrtf(2.f * r * width / 256.f));
    while (i > 0 && before(i) > r) --i;
    while (before(i + 1) <= r) ++i;
    m = i * 256;
    n = (r - before(i)) * width;
  }
}

// One warp's 32 rows of `part` columns of a tile, in chunks of 64 columns.
// The sums, plus beta times (r0, r1) where beta is not 0, to (o0, o1): hi and lo with TWO, else
// r0 and o0 alone.  SYM: also transposed below the diagonal block of rows `diag`.. (what
// lies above it belongs to other tiles).
//
// Rows pass through shared memory (128-byte swizzle), so that global accesses are whole
// 128-byte lines, eight lanes to a row; what the next chunk adds is on its way meanwhile.  Plain
// stores: the fence before a TMA store waited for those loads (1.6 us a chunk).
template <bool TWO, bool SYM, typename Wait, typename Release>
__device__ __forceinline__ bool ortho_epilogue(uint32_t t_row, int part, int n0, int m0, int M, int N, float alpha, float beta,
                                               const __half* r0, const __half* r1, __half* o0, __half* o1, int64_t ld, int diag,
                                               unsigned char* stage, int lane, Wait&& wait, Release&& release) {
  constexpr int BUF = 4096;
  const int sub = lane & 7, line = lane >> 3;
  const bool adds = !SYM || beta != 0.f;
  uint4 next0[8], next1[TWO ? 8 : 1];
  auto fetch = [&](int col) {
    col += 8 * sub;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = m0 + 4 * i + line;
      const bool in = adds && row < M && col < N;
      next0[i] = in ? __ldcg(reinterpret_cast<const uint4*>(r0 + row * ld + col)) : make_uint4(0, 0, 0, 0);
      if constexpr (TWO) next1[i] = in ? __ldcg(reinterpret_cast<const uint4*>(r1 + row * ld + col)) : make_uint4(0, 0, 0, 0);
    }
  };
  fetch(n0);
  if (!wait()) return false;
#pragma unroll 1
  for (int c = 0; c < part; c += 64) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = 4 * i + line, at = row * 128 + ((sub ^ (row & 7)) << 4);
      *reinterpret_cast<uint4*>(stage + at) = next0[i];
      if constexpr (TWO) *reinterpret_cast<uint4*>(stage + BUF + at) = next1[i];
    }
    __syncwarp();
    if (c + 64 < part) fetch(n0 + c + 64);
    const bool mirror = SYM && n0 + c < diag;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t acc[32];
      tmem_ld_32x32b_x32(t_row + c + 32 * h, acc);
      tmem_wait_ld();
      if (h == 1 && c + 64 == part) release();
      float v[32];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        unsigned char* at = stage + lane * 128 + (((4 * h + j) ^ (lane & 7)) << 4);
        uint4 w0 = *reinterpret_cast<const uint4*>(at), w1 = make_uint4(0, 0, 0, 0);
        if constexpr (TWO) w1 = *reinterpret_cast<const uint4*>(at + BUF);
        uint32_t* a0 = &w0.x;
        uint32_t* a1 = &w1.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 add = unpack2_layer<__half>(a0[i]);
          if constexpr (TWO) add = add2(add, unpack2_layer<__half>(a1[i]));
          const float2 s = make_float2(__uint_as_float(acc[8 * j + 2 * i]), __uint_as_float(acc[8 * j + 2 * i + 1]));
          const float2 r = fma2(both(alpha), s, mul2(both(beta), add));
          a0[i] = pack2_layer<__half>(r.x, r.y);
          if constexpr (TWO) {
            const float2 hi = unpack2_layer<__half>(a0[i]);
            a1[i] = pack2_layer<__half>(r.x - hi.x, r.y - hi.y);
          }
          v[8 * j + 2 * i] = r.x, v[8 * j + 2 * i + 1] = r.y;
        }
        *reinterpret_cast<uint4*>(at) = w0;
        if constexpr (TWO) *reinterpret_cast<uint4*>(at + BUF) = w1;
      }
      if (!TWO && mirror) {
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
    }
    __syncwarp();
    if (!SYM || n0 + c < diag + 256) {
      const int col = n0 + c + 8 * sub;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + line, row = m0 + r, at = r * 128 + ((sub ^ (r & 7)) << 4);
        if (row < M && col < N) {
          *reinterpret_cast<uint4*>(o0 + row * ld + col) = *reinterpret_cast<const uint4*>(stage + at);
          if constexpr (TWO) *reinterpret_cast<uint4*>(o1 + row * ld + col) = *reinterpret_cast<const uint4*>(stage + BUF + at);
        }
      }
    }
    if (mirror) {
      const int col = m0 + 8 * (lane & 3);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 8 * i + (lane >> 2), row = n0 + c + r;
        if constexpr (TWO) {
          // Both buffers hold rows: eight of them give an element each.
          uint32_t w0[4], w1[4];
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            auto two = [&](const unsigned char* buf) {
              const unsigned char* at = buf + (8 * (lane & 3) + j) * 128 + 2 * (r & 7);
              return static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(at + (((r >> 3) ^ j) << 4))) |
                     static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(at + 128 + (((r >> 3) ^ (j + 1)) << 4))) << 16;
            };
            w0[j / 2] = two(stage);
            w1[j / 2] = two(stage + BUF);
          }
          if (row < M && col < N) {
            *reinterpret_cast<uint4*>(o0 + row * ld + col) = make_uint4(w0[0], w0[1], w0[2], w0[3]);
            *reinterpret_cast<uint4*>(o1 + row * ld + col) = make_uint4(w1[0], w1[1], w1[2], w1[3]);
          }
        } else if (row < M && col < N) {
          *reinterpret_cast<uint4*>(o0 + row * ld + col) = *reinterpret_cast<const uint4*>(stage + BUF + r * 64 + 16 * (lane & 3));
        }
      }
    }
    __syncwarp();
  }
  return true;
}

// K blocks of unit t of a phase, and the tile that it works on.  FULL: those of the
// three products, small ones first.
template <bool FULL>
__device__ __forceinline__ int ortho_unit(const OrthoArgs& g, int kind, int t, int& kb0, int& kb1) {
  kb0 = 0;
  kb1 = (FULL ? 3 : 1) * g.k_blocks[kind];
  if (kind != kGram || g.splits == 1) return t;
  const int tile = t / g.splits, s = t - tile * g.splits, all = kb1;
  kb0 = all * s / g.splits;
  kb1 = all * (s + 1) / g.splits;
  return tile;
}

// One warp's 32 rows of `part` columns of a tile of X X^T whose depth `splits` pairs
// share (this one is number `split`): its sums go to memory, and when the same warps of the other
// pairs have stored theirs, each adds up a share of the columns, in the
// pairs' order, so that results do not depend on timing.  They run at once (there is a pair for every
// unit), so the wait ends.  A phase of 256 x 16384 65 -> 21 us.
template <bool FULL, typename Wait, typename Release>
__device__ __forceinline__ bool ortho_split_epilogue(const OrthoArgs& g, uint32_t t_row, int part, int n0, int m0, float alpha, int tile,
                                                     int split, int step, int where, __half* out, __half* out_lo, int diag, int lane,
                                                     volatile int* abort, Wait&& wait, Release&& release) {
  const int64_t region = 32ll * part, stride = region * 16;  // of a warp, of a pair
  float* base = g.partial + static_cast<int64_t>(tile) * g.splits * stride + where * region + lane;
  if (!wait()) return false;
#pragma unroll 1
  for (int c = 0; c < part; c += 32) {
    uint32_t acc[32];
    tmem_ld_32x32b_x32(t_row + c, acc);
    tmem_wait_ld();
    if (c + 32 == part) release();
    float* dst = base + split * stride + c * 32;
#pragma unroll
    for (int i = 0; i < 32; ++i) __stcg(dst + 32 * i, __uint_as_float(acc[i]));
  }
  __syncwarp();
  bool there = true;
  if (lane == 0) {
    unsigned* ticket = g.tickets + tile * 16 + where;
    red_release_gpu(ticket);
    there = grid_wait(ticket, static_cast<unsigned>((step + 1) * g.splits), abort, g.limit_ns);
  }
  if (!__all_sync(0xffffffffu, there)) return false;
  __syncwarp();  // what lane 0 has acquired is ordered before the other lanes' loads; the vote orders nothing
  const int share = part / g.splits, c0 = split * share, row = m0 + lane;  // 8 columns or more
#pragma unroll 1
  for (int c = c0; c < c0 + share; c += 8) {
    float v[8] = {};
    for (int s = 0; s < g.splits; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += __ldcg(base + s * stride + (c + i) * 32);
    const int col = n0 + c;
    if (col >= g.p || col >= diag + 256 || row >= g.p) continue;
#pragma unroll
    for (int part = 0; part < (FULL ? 2 : 1); ++part) {
      __half* o = part ? out_lo : out;
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (part == 0) v[2 * i] *= alpha, v[2 * i + 1] *= alpha;
        w[i] = pack2_layer<__half>(v[2 * i], v[2 * i + 1]);
        const float2 hi = unpack2_layer<__half>(w[i]);
        v[2 * i] -= hi.x, v[2 * i + 1] -= hi.y;
      }
      *reinterpret_cast<uint4*>(o + row * g.ldp + col) = make_uint4(w[0], w[1], w[2], w[3]);
      if (col < diag) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < g.p) o[(col + i) * g.ldp + row] = __ushort_as_half(static_cast<unsigned short>(w[i / 2] >> (16 * (i & 1))));
      }
    }
  }
  return true;
}

template <bool FULL>
__global__ void __launch_bounds__(ORT_THREADS, 1)
    ortho_pair_kernel(const __grid_constant__ OrthoMaps<FULL> maps, const __grid_constant__ OrthoArgs g) {
  using L = OrthoSmem;
  constexpr int STAGES = L::STAGES, SLOTS = ORT_SLOTS;

  extern __shared__ __align__(1024) unsigned char ortho_smem_raw[];
  unsigned char* smem = align_smem_1024(ortho_smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = full + 2 * STAGES;
  uint64_t* acc_empty = acc_full + SLOTS;
  uint64_t* drain = acc_empty + SLOTS;
  uint64_t* done = drain + 1;  // the epilogue warps have stored a phase
  uint64_t* go = drain + 2;    // every CTA has: a producer has seen the grid barrier
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & 1u;  // in the cluster of two
  const bool leader = rank == 0;
  const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x) / 2;
  const int phases = 3 * g.steps;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 2);   // leader: its two producers; both CTAs' bytes
      mbar_init(&empty[s], 1);  // one multicast commit per phase
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

  if (warp == 0 || warp == 2 + ORT_EPI_WARPS) {
    // ------------------------------------------------------------ producers (both CTAs)
    const bool of_a = warp == 0;
    uint32_t bits = 0, issued_mask = 0;  // bit s: parity of stage s's next phase; loaded at least once
    bool ok = true, ready = false;
    for (int ph = 0; ok && ph < phases; ++ph) {
      const int kind = ph % 3, cur = (ph / 3) & 1;
      const bool mn = kind == kGram ? g.tall : kind == kUpdate && !g.tall && !of_a;
      const CUtensorMap* const hi_map = of_a ? &maps.a[0][kind][cur] : &maps.b[0][kind][cur];
      const CUtensorMap* const lo_map = of_a ? &maps.a[FULL][kind][cur] : &maps.b[FULL][kind][cur];
      const int width = g.width[kind], pieces = !of_a && width == 512 ? 2 : 1;
      const int span = of_a ? ORT_BM : min(width, 256) / 2;  // rows or columns of the operand for one MMA
      const int stages = width == 512 ? L::WIDE_STAGES : L::STAGES, stride = (width == 512 ? 3 : 2) * L::OPERAND;
      const uint32_t bytes = static_cast<uint32_t>(pieces * span) * ORT_BK * 2;
      unsigned char* const ring = smem + (of_a ? 0 : L::OPERAND);
      int stage = 0;
      ready = false;
      if (elect_one_sync()) {
        prefetch_tmap(hi_map);
        if (FULL) prefetch_tmap(lo_map);
      }
      // The first phase reads what the kernel before has written.
      if (ph > 0) {
        if (!__all_sync(0xffffffffu, lane != 0 || grid_wait(g.barrier, static_cast<unsigned>(ph) * gridDim.x, abort_flag, g.limit_ns))) {
          ok = false;
          break;
        }
        __syncwarp();  // what lane 0 has acquired is ordered before the elected lane's loads
        if (of_a && elect_one_sync()) mbar_arrive(go);
      }
      for (int t = pair; ok && t < g.tiles[kind]; t += pairs) {
        int b, m, n, kb0, kb1;
        ortho_tile(g, kind, ortho_unit<FULL>(g, kind, t, kb0, kb1), b, m, n);
        const int first = (of_a ? m : n) + static_cast<int>(rank) * span;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!warp_wait(ready, &empty[stage], ((bits >> stage) & 1u) ^ 1u, kDevErrWaitTimeoutEmpty, abort_flag, g.limit_ns)) {
            ok = false;
            break;
          }
          if (elect_one_sync()) {
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * bytes);
            const uint32_t mbar = map_to_rank(&full[stage], 0);
            unsigned char* dst = ring + stage * stride;
            const int each = g.k_blocks[kind], product = !FULL ? 2 : kb >= 2 * each ? 2 : kb >= each ? 1 : 0;
            const CUtensorMap* const map = product == (of_a ? 1 : 0) ? lo_map : hi_map;  // hi lo, lo hi, hi hi
            const int k0 = (FULL ? kb - product * each : kb) * ORT_BK;
            for (int h = 0; h < pieces; ++h) {
              const int at = first + 256 * h;
              if (mn) {
                tma_load_3d_pair(dst + h * L::OPERAND, map, mbar, at, k0, b);
                if (span > 64) tma_load_3d_pair(dst + h * L::OPERAND + 8192, map, mbar, at + 64, k0, b);
              } else {
                tma_load_3d_pair(dst + h * L::OPERAND, map, mbar, k0, at, b);
              }
            }
          }
          __syncwarp();
          issued_mask |= 1u << stage;
          bits ^= 1u << stage;
          stage = stage + 1 == stages ? 0 : stage + 1;
          ready = mbar_test_wait(smem_u32(&empty[stage]), ((bits >> stage) & 1u) ^ 1u);
        }
      }
    }
    if (ok) {
      // No commit may still be on its way to this CTA's barriers.
      for (int s = 0; s < STAGES; ++s) {
        if ((issued_mask >> s) & 1u)
          if (!mbar_wait_bounded(&empty[s], ((bits >> s) & 1u) ^ 1u, kDevErrWaitTimeoutEmpty, abort_flag)) break;
      }
    } else if (leader && lane == 0) {
      // Abort: let every phase this pair issued land.
      for (int s = 0; s < STAGES; ++s) {
        if (!((issued_mask >> s) & 1u)) continue;
        const uint32_t addr = smem_u32(&full[s]);
        const unsigned long long t0 = global_timer_ns();
        while (!mbar_try_wait(addr, ((bits >> s) & 1u) ^ 1u)) {
          if (global_timer_ns() - t0 > kWaitLimitNs) {
            record_device_error(kDevErrAbortDrain);
            break;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader only)
    if (leader) {
      uint32_t bits = 0, empty_bits = 0;  // parities of full[], and of acc_empty[]'s next phases
      bool ok = true, issued = false, ready = false;
      auto slot_free = [&](int slot) {
        const bool free = warp_wait(false, &acc_empty[slot], ((empty_bits >> slot) & 1u) ^ 1u, kDevErrWaitTimeoutAccEmpty, abort_flag,
                                    g.limit_ns);
        tc_fence_after_sync();
        empty_bits ^= 1u << slot;
        return free;
      };
      for (int ph = 0; ok && ph < phases; ++ph) {
        const int kind = ph % 3;
        const bool a_mn = kind == kGram && g.tall, b_mn = kind == kGram ? g.tall : kind == kUpdate && !g.tall;
        const int width = g.width[kind];
        const bool wide = width == 512;
        const int stages = wide ? L::WIDE_STAGES : L::STAGES;
        const uint32_t idesc = make_idesc(0u, a_mn, b_mn, 2 * ORT_BM, min(width, 256));
        // Descriptors of the first stage's operands and what the next stage and K's
        // next 16 add to them.
        const uint32_t stride = (wide ? 3 : 2) * (L::OPERAND >> 4);
        const uint32_t a_step = (a_mn ? 2048u : 32u) >> 4, b_step = (b_mn ? 2048u : 32u) >> 4;
        const uint64_t a0 = make_smem_desc_sw128(smem_u32(smem), a_mn ? 8192u : 16u, 1024);
        const uint64_t b0 = make_smem_desc_sw128(smem_u32(smem + L::OPERAND), b_mn ? 8192u : 16u, 1024);
        int stage = 0, slot = 0;
        ready = false;
        for (int t = pair; ok && t < g.tiles[kind]; t += pairs) {
          if (!slot_free(slot)) {
            ok = false;
            break;
          }
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(slot * 256);
          int kb0, kb1;
          ortho_unit<FULL>(g, kind, t, kb0, kb1);
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!warp_wait(ready, &full[stage], (bits >> stage) & 1u, kDevErrWaitTimeoutFull, abort_flag, g.limit_ns)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const uint64_t ad = a0 + static_cast<uint32_t>(stage) * stride;
            const uint64_t bd = b0 + static_cast<uint32_t>(stage) * stride;
            if (elect_one_sync()) {
#pragma unroll
              for (uint32_t kk = 0; kk < ORT_BK / 16; ++kk)
                umma_f16_pair(d_tmem, ad + kk * a_step, bd + kk * b_step, idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
              if (!wide) umma_commit_pair(&empty[stage]);
            }
            __syncwarp();
            issued = true;
            if (wide) {
              // The second half of a wide tile may still be drained by the epilogue of the one before.
              if (kb == kb0 && !slot_free(1)) {
                ok = false;
                break;
              }
              if (elect_one_sync()) {
#pragma unroll
                for (uint32_t kk = 0; kk < ORT_BK / 16; ++kk)
                  umma_f16_pair(d_tmem + 256, ad + kk * a_step, bd + (L::OPERAND >> 4) + kk * b_step, idesc,
                                (kb > kb0 || kk > 0) ? 1u : 0u);
                umma_commit_pair(&empty[stage]);
              }
              __syncwarp();
            }
            bits ^= 1u << stage;
            stage = stage + 1 == stages ? 0 : stage + 1;
            ready = mbar_test_wait(smem_u32(&full[stage]), (bits >> stage) & 1u);
          }
          if (!ok) break;
          if (elect_one_sync()) umma_commit_pair(&acc_full[slot]);
          __syncwarp();
          if (!wide) slot ^= 1;
        }
      }
      if (!ok && issued) {
        if (elect_one_sync()) umma_commit_pair(drain);
        __syncwarp();
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
    const int quarter = warp & 3;
    unsigned char* stage = smem + L::OFF_C + (warp - 2) * 2 * 4096;
    uint32_t full_bits = 0;  // parities of acc_full[]'s next phases
    bool ok = true;
    for (int ph = 0; ok && ph < phases; ++ph) {
      const int kind = ph % 3, step = ph / 3, cur = step & 1;
      const float alpha = g.alpha[step][kind], beta = g.beta[step][kind];
      const int width = g.width[kind], part = min(width, 256) / 2, c0 = (warp - 2) / 4 * part;
      int slot = 0;
      // What the epilogue adds was written in the phases before.
      if (ph > 0) {
        const bool there = mbar_wait_bounded(go, static_cast<uint32_t>(ph - 1) & 1u, kDevErrGridBarrier, abort_flag, g.limit_ns);
        if (!__all_sync(0xffffffffu, there)) {
          ok = false;
          break;
        }
      }
      for (int t = pair; ok && t < g.tiles[kind]; t += pairs) {
        int b, m, n, kb0, kb1;
        const int tile = ortho_unit<FULL>(g, kind, t, kb0, kb1);
        ortho_tile(g, kind, tile, b, m, n);
        const int m0 = m + static_cast<int>(rank) * ORT_BM + 32 * quarter;
        for (int h = 0; ok && h < (width == 512 ? 2 : 1); ++h) {
          const int n0 = n + 256 * h + c0;
          const uint32_t t_row =
              tmem_base + (static_cast<uint32_t>(32 * quarter) << 16) + static_cast<uint32_t>((slot + h) * 256 + c0);
          auto wait = [&] {
            bool got = true;
            if (h == 0) {
              got = mbar_wait_bounded(&acc_full[slot], (full_bits >> slot) & 1u, kDevErrWaitTimeoutAccFull, abort_flag,
                                      g.limit_ns);
              tc_fence_after_sync();
            }
            return static_cast<bool>(__all_sync(0xffffffffu, got));
          };
          auto release = [&] {
            tc_fence_before_sync();
            __syncwarp();
            // The last tile's accumulator is not handed back: nobody waits for it, and an arrival on its way to the
            // leader's barrier could outlive the leader.
            if (lane == 0 && (ph + 1 < phases || t + pairs < g.tiles[kind]))
              mbar_arrive_remote(map_to_rank(&acc_empty[slot + h], 0));
          };
          if (kind == kUpdate) {
            const int64_t off = b * g.stride_x;
            ok = ortho_epilogue<true, false>(t_row, part, n0, m0, g.tall ? g.q : g.p, g.tall ? g.p : g.q, alpha, beta,
                                             g.x[cur] + off, g.lo[FULL ? cur : 0] + off, g.x[cur ^ 1] + off,
                                             g.lo[FULL ? cur ^ 1 : 0] + off, g.ldx, 0, stage, lane, wait, release);
          } else if (kind == kGram && g.splits > 1) {
            ok = ortho_split_epilogue<FULL>(g, t_row, part, n0, m0, alpha, tile, t - tile * g.splits, step,
                                      static_cast<int>(rank) * ORT_EPI_WARPS + warp - 2, g.gram + b * g.stride_p,
                                      g.gram_lo + b * g.stride_p, m, lane, abort_flag, wait, release);
          } else {
            const int64_t off = b * g.stride_p;
            __half* out = (kind == kPoly ? g.poly : g.gram) + off;
            __half* out_lo = (kind == kPoly ? g.poly_lo : g.gram_lo) + off;
            ok = ortho_epilogue<FULL, true>(t_row, part, n0, m0, g.p, g.p, alpha, kind == kPoly ? beta : 0.f, g.gram + off,
                                            g.gram_lo + off, out, out_lo, g.ldp, m, stage, lane, wait, release);
          }
        }
        if (!ok) break;
        full_bits ^= 1u << slot;
        if (width != 512) slot ^= 1;
      }
      if (!ok) break;
      // This CTA's share of the phase is in memory.
      __syncwarp();
      if (lane == 0 && ph + 1 < phases) {
        mbar_arrive(done);
        if (warp == 2 && mbar_wait_bounded(done, static_cast<uint32_t>(ph) & 1u, kDevErrGridBarrier, abort_flag, g.limit_ns)) {
          red_release_gpu(g.barrier);
        }
      }
      __syncwarp();
    }
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
  int64_t rows, cols;
  int groups;  // of eight columns in a row
  int across;  // log2 of the threads to a row; the others of a CTA have the next rows
  int blocks;  // CTAs to a matrix
  OrthoTensor g, m, w;         // gradient; momentum; weight, or the result
  float mu;
  int nesterov;
  double* partial;    // [batch][blocks] sums of squares
  unsigned* barrier;  // of ortho_pair_kernel, and its tickets behind it
  int words;          // of both
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

// Calls f(row, first column, a second row or -1) for this thread's groups: two
// rows at a time, so that their loads are on their way together.
template <typename F>
__device__ __forceinline__ void ortho_groups(const OrthoIo& p, F&& f) {
  const int tpr = 1 << p.across;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (256 >> p.across);
  for (int64_t row = blockIdx.x * static_cast<int64_t>(256 >> p.across) + (threadIdx.x >> p.across); row < p.rows; row += 2 * step)
    for (int g = threadIdx.x & (tpr - 1); g < p.groups; g += tpr) f(row, 8 * g, row + step < p.rows ? row + step : -1);
}

// Momentum <- mu momentum + gradient, and the sum of the squares of what is
// orthogonalised: in 64 bits, which neither large nor small numbers leave.
template <bool MOMENTUM>
__global__ void __launch_bounds__(256, 4) ortho_sum_kernel(const OrthoIo p) {
  __shared__ double part[8];
  const int64_t b = blockIdx.y;
  grid_dependency_wait();
  if (blockIdx.x == 0 && b == 0)
    for (int i = threadIdx.x; i < p.words; i += 256) p.barrier[i] = 0u;
  double s = 0.0;
  ortho_groups(p, [&](int64_t row, int64_t c, int64_t row2) {
    float g[2][8], m[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t r = k ? row2 : row;
      if (r < 0) break;
      ortho_load8(p.g, b, r, c, p.cols, g[k]);
      if constexpr (MOMENTUM) ortho_load8(p.m, b, r, c, p.cols, m[k]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t r = k ? row2 : row;
      if (r < 0) break;
      if constexpr (MOMENTUM) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m[k][i] = fmaf(p.mu, m[k][i], g[k][i]);
        ortho_store8(p.m, b, r, c, p.cols, m[k]);
        ortho_update8(p, m[k], g[k]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fma(static_cast<double>(g[k][i]), static_cast<double>(g[k][i]), s);
    }
  });
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
template <bool MOMENTUM>
__global__ void __launch_bounds__(256, 4) ortho_scale_kernel(const OrthoIo p) {
  __shared__ double part[256];
  const int64_t b = blockIdx.y;
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
  ortho_groups(p, [&](int64_t row, int64_t c, int64_t row2) {
    float g[2][8], m[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t r = k ? row2 : row;
      if (r < 0) break;
      if (!MOMENTUM || p.nesterov) ortho_load8(p.g, b, r, c, p.cols, g[k]);
      if constexpr (MOMENTUM) ortho_load8(p.m, b, r, c, p.cols, m[k]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t r = k ? row2 : row;
      if (r < 0) break;
      if constexpr (MOMENTUM) ortho_update8(p, m[k], g[k]);
      uint32_t h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = make_float2(g[k][2 * i] * pre * f, g[k][2 * i + 1] * pre * f);
        h[i] = pack2_layer<__half>(v.x, v.y);
        const float2 hi = unpack2_layer<__half>(h[i]);
        l[i] = pack2_layer<__half>(v.x - hi.x, v.y - hi.y);
      }
      const int64_t at = b * p.stride_x + r * p.ldx + c;
      *reinterpret_cast<uint4*>(p.hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(p.lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
    }
  });
}

// The result, or the weight's step.
template <bool UPDATE>
__global__ void __launch_bounds__(256, 4) ortho_out_kernel(const OrthoIo p) {
  const int64_t b = blockIdx.y;
  grid_dependency_wait();
  float keep = p.keep, step = p.step;
  if (UPDATE && p.lr_dev) {
    const float lr = *p.lr_dev;
    keep = 1.f - lr * p.decay;
    step *= lr;
  }
  ortho_groups(p, [&](int64_t row, int64_t c, int64_t row2) {
    uint4 h4[2], l4[2];
    float w[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t r = k ? row2 : row;
      if (r < 0) break;
      const int64_t at = b * p.stride_x + r * p.ldx + c;
      h4[k] = *reinterpret_cast<const uint4*>(p.hi + at);
      l4[k] = *reinterpret_cast<const uint4*>(p.lo + at);
      if constexpr (UPDATE) ortho_load8(p.w, b, r, c, p.cols, w[k]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t r = k ? row2 : row;
      if (r < 0) break;
      const uint32_t h[4] = {h4[k].x, h4[k].y, h4[k].z, h4[k].w}, l[4] = {l4[k].x, l4[k].y, l4[k].z, l4[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = add2(unpack2_layer<__half>(h[i]), unpack2_layer<__half>(l[i]));
        if constexpr (UPDATE) {
          w[k][2 * i] = fmaf(-step, x.x, keep * w[k][2 * i]), w[k][2 * i + 1] = fmaf(-step, x.y, keep * w[k][2 * i + 1]);
        } else {
          w[k][2 * i] = x.x * p.out, w[k][2 * i + 1] = x.y * p.out;
        }
      }
      ortho_store8(p.w, b, r, c, p.cols, w[k]);
    }
  });
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
  int blocks, groups, across;
  int gram_width, splits;  // of the first phase's tiles where pairs share them (splits > 1)
  int words;
  bool full;  // products of hi and lo
  size_t sums_off, barrier_off, partial_off, hi_off[2], lo_off[2], gram_off[2], poly_off[2], bytes;
};

// Tiles of a symmetric matrix of `rows` row tiles: those whose first column is at most their last row.
int64_t ortho_sym_tiles(int64_t rows, int width) {
  if (width == 512) return (rows / 2) * (rows / 2 + 1) + (rows & 1) * (rows / 2 + 1);
  return 256 / width * (rows * (rows + 1) / 2);
}

// Pairs that share a tile of X X^T, so that no more than `pairs` are at work: the
// exchange takes about as long as 16 K blocks.
int ortho_splits(int64_t tiles, int64_t k_blocks, int64_t pairs) {
  int s = 1;
  while (s < 8 && tiles * 2 * s <= pairs && k_blocks >= 8 * 2 * s) s *= 2;
  return k_blocks - k_blocks / s >= 24 ? s : 1;
}

OrthoPlan ortho_plan(int64_t batch, int64_t rows, int64_t cols, bool full) {
  OrthoPlan o = {};
  o.full = full;
  if (batch <= 0 || rows <= 0 || cols <= 0) return o;
  o.batch = batch;
  o.tall = rows > cols;
  o.p = std::min(rows, cols), o.q = std::max(rows, cols);
  o.ldx = round8(cols), o.stride_x = rows * o.ldx;
  o.ldp = round8(o.p), o.stride_p = o.p * o.ldp;
  o.groups = static_cast<int>((cols + 7) / 8);
  while (o.across < 8 && (1 << o.across) < o.groups) ++o.across;
  // Four CTAs of 256 threads an SM, two waves over the whole stack, two rows a thread.
  const int64_t most = std::max<int64_t>(1, device_sm_count() * 8 / batch), each = 2 * (256 >> o.across);
  o.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, (rows + each - 1) / each)));
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += round256(bytes);
    return at;
  };
  const int64_t tiles = (o.p + 255) / 256;
  o.gram_width = o.p <= 128 ? 128 : 256;
  const int64_t gram_tiles = o.p <= 128 ? batch : batch * ortho_sym_tiles(tiles, 256);
  o.splits = ortho_splits(gram_tiles, (full ? 3 : 1) * ((o.q + ORT_BK - 1) / ORT_BK), device_sm_count() / 2);
  o.words = 1 + (o.splits > 1 ? static_cast<int>(gram_tiles) * 16 : 0);
  o.sums_off = take(o.splits > 1 ? static_cast<size_t>(gram_tiles) * o.splits * 256 * o.gram_width * 4 : 0);
  o.barrier_off = take(static_cast<size_t>(o.words) * 4);
  o.partial_off = take(static_cast<size_t>(batch) * o.blocks * 8);
  for (int i = 0; i < 2; ++i) o.hi_off[i] = take(static_cast<size_t>(batch) * o.stride_x * 2);
  // Where products read lo it alternates as hi does; else a tile's owner alone reads and writes it.
  for (int i = 0; i < 2; ++i) o.lo_off[i] = i == 0 || full ? take(static_cast<size_t>(batch) * o.stride_x * 2) : o.lo_off[0];
  for (int i = 0; i < 2; ++i) {
    o.gram_off[i] = i == 0 || full ? take(static_cast<size_t>(batch) * o.stride_p * 2) : o.gram_off[0];
    o.poly_off[i] = i == 0 || full ? take(static_cast<size_t>(batch) * o.stride_p * 2) : o.poly_off[0];
  }
  o.bytes = off;
  return o;
}

// Width of a phase's tiles, by its waves.  A tile of 128 columns takes 0.65 of one of 256 (0.82
// alone on its SMs), one of 512 1.9 times it: it pulls three quarters of the operands from
// L2 (8192 x 28672, first phase, us: 2300 / 1840 / 1530 to 1760), but has one accumulator.
int ortho_width(int64_t tiles128, int64_t tiles256, int64_t tiles512, int64_t pairs) {
  const int64_t t128 = (tiles128 + pairs - 1) / pairs * 13;
  const int64_t t256 = (tiles256 + pairs - 1) / pairs * 20;
  const int64_t t512 = (tiles512 + pairs - 1) / pairs * 38;
  return t512 < std::min(t128, t256) ? 512 : t256 <= t128 ? 256 : 128;
}

// The products' launch.  Everything about it that can fail before it is queued is
// found out by prepare_ortho_pairs, which a call makes before its first kernel changes the momentum.
template <bool FULL>
struct OrthoLaunch {
  OrthoMaps<FULL> maps;
  OrthoArgs args;
  int pairs;
};

template <bool FULL>
int prepare_ortho_pairs(const OrthoPlan& o, const OrthoSchedule& sched, int steps, char* ws, OrthoLaunch<FULL>& launch) {
  using L = OrthoSmem;
  auto kern = ortho_pair_kernel<FULL>;
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
  auto half_at = [&](size_t off) { return reinterpret_cast<__half*>(ws + off); };
  const int64_t xr = o.tall ? o.q : o.p, xc = o.tall ? o.p : o.q;  // X as stored
  const int64_t most = capacity[dev].load(std::memory_order_relaxed);  // pairs at once
  const int64_t rows = (o.p + 255) / 256, tiles_m = (xr + 255) / 256;
  auto sym = [&](int w) { return o.batch * ortho_sym_tiles(rows, w); };
  auto upd = [&](int w) { return o.batch * tiles_m * ((xc + w - 1) / w); };
  const int ws_sym = ortho_width(sym(128), sym(256), sym(512), most);
  // X's tiles are read and written as hi and lo, in bursts of all pairs that take HBM's
  // time: only tiles of 256 columns, with two accumulators, hide those (8192 x 28672: 3.46 ms with 512, 3.2 with 256).
  const int ws_upd = ortho_width(upd(128), upd(256), INT32_MAX, most);
  // On a part with fewer pairs at once the planned split does not fit.
  const int64_t gram_tiles = o.words / 16;
  const int splits = gram_tiles * o.splits <= most ? o.splits : 1;
  const int width[3] = {splits > 1 ? o.gram_width : ws_sym, ws_sym, ws_upd};
  OrthoMaps<FULL>& m = launch.maps;
  bool ok = true;
  auto map_x = [&](CUtensorMap* t, const __half* x, int inner, int rows) {
    ok &= make_map(t, dt, x, xc, xr, o.batch, o.ldx, o.stride_x, inner, rows);
  };
  auto map_p = [&](CUtensorMap* t, const __half* x, int inner, int rows) {
    ok &= make_map(t, dt, x, o.p, o.p, o.batch, o.ldp, o.stride_p, inner, rows);
  };
  for (int l = 0; l < (FULL ? 2 : 1); ++l) {  // hi, lo
    const __half* gram = half_at(o.gram_off[l]);
    const __half* poly = half_at(o.poly_off[l]);
    for (int i = 0; i < 2; ++i) {
      const __half* x = half_at(l ? o.lo_off[i] : o.hi_off[i]);
      // K-major operands come in boxes of 64 x rows, MN-major ones in 64 x 64.
      map_x(&m.a[l][kGram][i], x, 64, o.tall ? ORT_BK : ORT_BM);
      map_x(&m.b[l][kGram][i], x, 64, o.tall ? ORT_BK : std::min(width[kGram], 256) / 2);
      map_p(&m.a[l][kPoly][i], gram, 64, ORT_BM);
      map_p(&m.b[l][kPoly][i], gram, 64, std::min(width[kPoly], 256) / 2);
      if (o.tall) {
        map_x(&m.a[l][kUpdate][i], x, 64, ORT_BM);
        map_p(&m.b[l][kUpdate][i], poly, 64, std::min(width[kUpdate], 256) / 2);
      } else {
        map_p(&m.a[l][kUpdate][i], poly, 64, ORT_BM);
        map_x(&m.b[l][kUpdate][i], x, 64, ORT_BK);
      }
    }
  }
  if (!ok) return CUOPX_CUDA_ERROR;
  OrthoArgs& a = launch.args;
  a = {};
  a.batch = static_cast<int>(o.batch);
  a.p = static_cast<int>(o.p), a.q = static_cast<int>(o.q);
  a.steps = steps;
  a.tall = o.tall;
  for (int j = 0; j < 3; ++j) a.width[j] = width[j];
  a.tiles_m = static_cast<int>(tiles_m), a.tiles_n = static_cast<int>((xc + ws_upd - 1) / ws_upd);
  for (int j = 0; j < 2; ++j) {
    // p <= 128: the second tile of 128 columns holds nothing.
    a.sym_tiles[j] = o.p <= 128 && width[j] == 128 ? 1 : static_cast<int>(ortho_sym_tiles(rows, width[j]));
    a.tiles[j] = a.batch * a.sym_tiles[j] * (j == kGram ? splits : 1);
  }
  a.splits = splits;
  a.partial = reinterpret_cast<float*>(ws + o.sums_off);
  a.tickets = reinterpret_cast<unsigned*>(ws + o.barrier_off) + 1;
  a.tiles[kUpdate] = a.batch * a.tiles_m * a.tiles_n;
  a.k_blocks[kGram] = static_cast<int>((o.q + ORT_BK - 1) / ORT_BK);
  a.k_blocks[kPoly] = a.k_blocks[kUpdate] = static_cast<int>((o.p + ORT_BK - 1) / ORT_BK);
  for (int i = 0; i < 2; ++i) a.x[i] = half_at(o.hi_off[i]), a.lo[i] = half_at(o.lo_off[i]);
  a.gram = half_at(o.gram_off[0]), a.gram_lo = half_at(o.gram_off[1]);
  a.poly = half_at(o.poly_off[0]), a.poly_lo = half_at(o.poly_off[1]);
  a.ldx = o.ldx, a.stride_x = o.stride_x, a.ldp = o.ldp, a.stride_p = o.stride_p;
  a.barrier = reinterpret_cast<unsigned*>(ws + o.barrier_off);
  const double work = (FULL ? 6.0 : 2.0) * static_cast<double>(o.batch) * static_cast<double>(o.p) * static_cast<double>(o.p) * static_cast<double>(o.q);
  a.limit_ns = kWaitLimitNs + static_cast<unsigned long long>(work / 1e5);  // at 100 TFLOP/s
  for (int i = 0; i < steps; ++i)
    for (int j = 0; j < 3; ++j) a.alpha[i][j] = sched.alpha[i][j], a.beta[i][j] = sched.beta[i][j];
  launch.pairs = std::min(static_cast<int>(most), std::max({a.tiles[kGram], a.tiles[kPoly], a.tiles[kUpdate]}));
  return CUOPX_SUCCESS;
}

template <bool FULL>
int launch_ortho_pairs(const OrthoLaunch<FULL>& launch, cudaStream_t stream) {
  // Cooperative: all CTAs run at once, whatever else the GPU does.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * launch.pairs));
  cfg.blockDim = dim3(ORT_THREADS);
  cfg.dynamicSmemBytes = OrthoSmem::ALLOC;
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
  if (const cudaError_t err = cudaLaunchKernelEx(&cfg, ortho_pair_kernel<FULL>, launch.maps, launch.args); err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  note_launch(FULL ? "ortho_pair_full" : "ortho_pair");
  return check_launch();
}

OrthoTensor ortho_tensor(const void* p, int dtype, int64_t ld, int64_t stride, int64_t batch, int64_t rows) {
  OrthoTensor t = {const_cast<void*>(p), p ? dtype : -1, 0, ld, stride};
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  t.vec = reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || ld * es % 16 == 0) && (batch == 1 || stride * es % 16 == 0);
  return t;
}

// All launches of a call.  `io` has the tensors and what the last pass does.
template <bool FULL>
int ortho_run_as(OrthoIo io, const OrthoPlan& o, const double* coefficients, int steps, bool update, double out_factor, void* workspace,
              cudaStream_t stream) {
  OrthoSchedule sched;
  if (!ortho_schedule(coefficients, steps, sched)) return CUOPX_INVALID_ARGUMENT;
  char* ws = static_cast<char*>(workspace);
  OrthoLaunch<FULL> products;
  if (steps > 0) {
    if (const int rc = prepare_ortho_pairs(o, sched, steps, ws, products); rc != CUOPX_SUCCESS) return rc;
  }
  io.groups = o.groups, io.across = o.across, io.blocks = o.blocks, io.words = o.words;
  io.partial = reinterpret_cast<double*>(ws + o.partial_off);
  io.barrier = reinterpret_cast<unsigned*>(ws + o.barrier_off);
  io.x_scale = static_cast<float>(sched.first);
  io.ldx = o.ldx, io.stride_x = o.stride_x;
  io.lo = reinterpret_cast<__half*>(ws + o.lo_off[0]);
  io.hi = reinterpret_cast<__half*>(ws + o.hi_off[0]);
  const dim3 grid(static_cast<unsigned>(o.blocks), static_cast<unsigned>(o.batch));
  const bool momentum = io.m.dtype >= 0;
  cudaError_t err = launch_pdl(momentum ? ortho_sum_kernel<true> : ortho_sum_kernel<false>, grid, dim3(256), 0, stream, io);
  if (err == cudaSuccess) {
    note_launch("ortho_sum");
    err = launch_pdl(momentum ? ortho_scale_kernel<true> : ortho_scale_kernel<false>, grid, dim3(256), 0, stream, io);
  }
  if (err == cudaSuccess) note_launch("ortho_scale");
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  if (steps > 0) {
    if (const int rc = launch_ortho_pairs(products, stream); rc != CUOPX_SUCCESS) return rc;
  }
  io.hi = reinterpret_cast<__half*>(ws + o.hi_off[steps & 1]);
  io.lo = reinterpret_cast<__half*>(ws + o.lo_off[steps & 1]);
  io.out = static_cast<float>(out_factor / sched.last);
  io.step = static_cast<float>(out_factor / sched.last);
  err = launch_pdl(update ? ortho_out_kernel<true> : ortho_out_kernel<false>, grid, dim3(256), 0, stream, io);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  // Named after the products' widest tiles, which have a ring and an accumulator of their own.
  if (steps > 0 && products.args.width[kPoly] == 512) note_launch(update ? "ortho_step_w512" : "ortho_out_w512");
  else note_launch(update ? "ortho_step" : "ortho_out");
  return check_launch();
}

int ortho_run(const OrthoIo& io, const OrthoPlan& o, const double* coefficients, int steps, bool update, double out_factor,
              void* workspace, cudaStream_t stream) {
  return o.full ? ortho_run_as<true>(io, o, coefficients, steps, update, out_factor, workspace, stream)
                : ortho_run_as<false>(io, o, coefficients, steps, update, out_factor, workspace, stream);
}

// Bits that the products' operands keep: as asked for, or by the result's type.  Operands of 11
// leave 1.2e-3 of the result, less than bf16's own rounding (1.7e-3) but six times fp16's.
bool ortho_bits_ok(int bits) { return bits == 0 || bits == 11 || bits == 22; }
bool ortho_full(int bits, int result) { return bits == 0 ? result != CUOPX_BF16 : bits == 22; }

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
  if (a->steps < 0 || a->steps > ORT_MAX_STEPS || !ortho_bits_ok(a->operand_bits) || !(a->eps >= 0) || !std::isfinite(a->eps) ||
      (a->steps > 0 && !a->coefficients) || !ortho_sizes_ok(a->batch, a->rows, a->cols))
    return CUOPX_INVALID_ARGUMENT;
  OrthoSchedule sched;
  if (!ortho_schedule(a->coefficients, a->steps, sched)) return CUOPX_INVALID_ARGUMENT;
  if (a->batch == 0 || a->rows == 0 || a->cols == 0) return CUOPX_SUCCESS;
  if (!ortho_layout_ok(a->G, a->dtype, a->ldg, a->strideG, a->batch, a->rows, a->cols) ||
      !ortho_layout_ok(a->out, a->out_dtype, a->ldo, a->strideO, a->batch, a->rows, a->cols) || !starts_on(256, a->workspace))
    return CUOPX_INVALID_ARGUMENT;
  const OrthoPlan o = ortho_plan(a->batch, a->rows, a->cols, ortho_full(a->operand_bits, a->out_dtype));
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
  if (a->steps < 0 || a->steps > ORT_MAX_STEPS || (a->nesterov != 0 && a->nesterov != 1) || !ortho_bits_ok(a->operand_bits) || !(a->eps >= 0) ||
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
  const OrthoPlan o = ortho_plan(a->batch, a->rows, a->cols, ortho_full(a->operand_bits, a->wdtype));
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

size_t cuopx_orthogonalize_workspace_size_bits(int64_t batch, int64_t rows, int64_t cols, int operand_bits) {
  return cuopx::ortho_sizes_ok(batch, rows, cols) ? cuopx::ortho_plan(batch, rows, cols, operand_bits != 11).bytes : 0;
}
size_t cuopx_orthogonalize_workspace_size(int64_t batch, int64_t rows, int64_t cols) {
  return cuopx_orthogonalize_workspace_size_bits(batch, rows, cols, 22);
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
