// Feed-forward layer operators on the GEMM kernels: the linear layer with
// bias, activation and residual in its epilogue, the gated linear layer, and
// their gradients (cuopx_linear, cuopx_gated_linear and their backward forms).
//
//   linear    Z = X W + b              Y = act(Z) + R
//   gated     Z = [G | U] = X W + b    Y = act(G) * U
//   backward  dZ = dY * act'(Z)   or   [dY * U * act'(G) | dY * act(G)],
//             dX = dZ W^T, dW = X^T dZ, db = column sums of dZ
//
// Products and epilogue in fp32 from 16-bit operands.  Y is rounded once,
// from the unrounded Z.  Backward rounds dZ once to the 16-bit type, because
// the products that follow take 16-bit operands; db sums the unrounded dZ.
#include "activation.cuh"
#include "common.cuh"
#include "dispatch.h"
#include "layer_epilogue.cuh"

namespace cuopx {

namespace {

// ---------------------------------------------------------------- any size, stride and alignment
// 64 x 64 outputs per CTA, 16-deep steps through shared memory, 4 x 4 outputs
// per thread (of both projections when gated).
constexpr int LS_T = 64, LS_K = 16;

template <typename T, bool GATED>
__global__ void __launch_bounds__(256) linear_simt_kernel(const LinearProblem p) {
  constexpr int NB = GATED ? 2 : 1;
  __shared__ float xs[LS_K][LS_T + 4];
  __shared__ float ws[NB][LS_K][LS_T + 4];
  const T* X = static_cast<const T*>(p.X);
  const T* W = static_cast<const T*>(p.W);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t tiles_n = (p.N + LS_T - 1) / LS_T, tiles = tiles_n * ((p.M + LS_T - 1) / LS_T);
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t m0 = t / tiles_n * LS_T, n0 = t % tiles_n * LS_T;
    float acc[NB][4][4] = {};
    for (int64_t k0 = 0; k0 < p.K; k0 += LS_K) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = threadIdx.x + 256 * i;
        const int64_t m = m0 + e / LS_K, k = k0 + e % LS_K;
        xs[e % LS_K][e / LS_K] = m < p.M && k < p.K ? to_acc<T>(X[m * p.ldx + k]) : 0.f;
#pragma unroll
        for (int h = 0; h < NB; ++h) {
          // Consecutive threads read consecutive addresses in either layout.
          const int wk = p.transW ? e % LS_K : e / LS_T, wn = p.transW ? e / LS_K : e % LS_T;
          const int64_t kk = k0 + wk, n = n0 + wn;
          float v = 0.f;
          if (kk < p.K && n < p.N) v = to_acc<T>(p.transW ? W[(h * p.w_up + n) * p.ldw + kk] : W[kk * p.ldw + h * p.w_up + n]);
          ws[h][wk][wn] = v;
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < LS_K; ++k) {
        float a[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = xs[k][4 * ty + i];
#pragma unroll
        for (int h = 0; h < NB; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float b = ws[h][k][tx + 16 * j];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[h][i][j] = fmaf(a[i], b, acc[h][i][j]);
          }
      }
    }
    with_activation(p.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t m = m0 + 4 * ty + i, n = n0 + tx + 16 * j;
          if (m >= p.M || n >= p.N) continue;
          float z[NB];
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            z[h] = acc[h][i][j];
            if (p.bias) z[h] += to_acc<T>(static_cast<const T*>(p.bias)[h * p.N + n]);
            if (p.Z) static_cast<T*>(p.Z)[m * p.ldz + h * p.N + n] = from_acc<T>(z[h]);
          }
          float y = act_value<act.value>(z[0]);
          if constexpr (GATED) y *= z[1];
          if (p.R) y += to_acc<T>(static_cast<const T*>(p.R)[m * p.ldr + n]);
          static_cast<T*>(p.Y)[m * p.ldy + n] = from_acc<T>(y);
        }
      }
    });
  }
}

int linear_simt(const LinearProblem& p, cudaStream_t stream) {
  const int64_t tiles = ((p.N + LS_T - 1) / LS_T) * ((p.M + LS_T - 1) / LS_T);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(tiles, 1 << 30));
  if (p.dtype == CUOPX_BF16) {
    if (p.gated) linear_simt_kernel<__nv_bfloat16, true><<<grid, 256, 0, stream>>>(p);
    else linear_simt_kernel<__nv_bfloat16, false><<<grid, 256, 0, stream>>>(p);
  } else {
    if (p.gated) linear_simt_kernel<__half, true><<<grid, 256, 0, stream>>>(p);
    else linear_simt_kernel<__half, false><<<grid, 256, 0, stream>>>(p);
  }
  note_launch(p.gated ? "gated_linear_simt" : "linear_simt");
  return check_launch();
}

// ---------------------------------------------------------------- copies on 16-byte boundaries
// TMA reads rows that start on 16-byte boundaries.  An operand whose rows do
// not is first copied to rows that do (one read and one write of it, which
// buys the tensor cores for the product).  `halves`: the row's two
// projections are copied apart, so that the second starts on a boundary too.
struct RepackParams {
  int64_t rows, cols;  // of one half
  int halves;
  const unsigned short* src;
  int64_t ld, src_half;
  unsigned short* dst;
  int64_t ldd, dst_half;
};

__global__ void __launch_bounds__(256) linear_repack_kernel(const RepackParams p) {
  const int64_t groups = (p.cols + 7) / 8, per_row = groups * p.halves;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < p.rows * per_row; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = e / per_row, g = e - row * per_row;
    const int64_t half = g >= groups, c = (g - half * groups) * 8;
    const unsigned short* s = p.src + row * p.ld + half * p.src_half + c;
    uint32_t w[4];
    if (c > 0 && c + 9 < p.cols) {
      // Five aligned words around the eight elements, all inside the row.
      const bool odd = reinterpret_cast<uintptr_t>(s) & 2;
      const uint32_t* a = reinterpret_cast<const uint32_t*>(s - (odd ? 1 : 0));
      uint32_t v[5];
#pragma unroll
      for (int i = 0; i < 5; ++i) v[i] = a[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = odd ? __funnelshift_r(v[i], v[i + 1], 16) : v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = c + 2 * i < p.cols ? s[2 * i] : 0u, hi = c + 2 * i + 1 < p.cols ? s[2 * i + 1] : 0u;
        w[i] = lo | hi << 16;
      }
    }
    *reinterpret_cast<uint4*>(p.dst + row * p.ldd + half * p.dst_half + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// rows x cols of src to rows of round8(cols) at dst (halves: two such rows side by side).
void linear_repack(const void* src, int64_t rows, int64_t cols, int64_t ld, int halves, int64_t src_half, void* dst,
                   cudaStream_t stream) {
  RepackParams r;
  r.rows = rows;
  r.cols = cols;
  r.halves = halves;
  r.src = static_cast<const unsigned short*>(src);
  r.ld = ld;
  r.src_half = src_half;
  r.dst = static_cast<unsigned short*>(dst);
  r.dst_half = round8(cols);
  r.ldd = halves * r.dst_half;
  const int64_t n = rows * halves * (r.dst_half / 8);
  const unsigned ctas = static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, static_cast<int64_t>(device_sm_count()) * 32));
  linear_repack_kernel<<<ctas, 256, 0, stream>>>(r);
  note_launch("linear_repack");
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// ---------------------------------------------------------------- dZ and its column sums
// One pass over dY (and Z): writes dZ and, per share of the rows, the fp32
// column sums of the unrounded dZ.  A thread owns V columns (V = 8: one
// 16-byte load per matrix and row) of every row that it walks; `across` of a
// CTA's eight warps lie side by side, so that a row is read in runs of up to 4
// KB (512-byte runs of eight rows measured 3.3 TB/s), and the others take the
// rows between.  Several rows are loaded before the first is used.  Bound by
// HBM (4096 x 28672 bf16, GELU: 127 us for the sums alone, 152 with dZ stored,
// 4.6 TB/s), in single elements by the number of loads (999 x 2731 f16, gated: 18
// us).
struct DzParams {
  int64_t M, N;
  int act, across;
  const void* dY;
  int64_t lddy;
  const void* Z;
  int64_t ldz;
  void* dZ;  // NULL: only sums
  int64_t lddz;
  float* partial;  // [splits][wide]; NULL: no sums
  void* db;        // written directly when splits == 1
  int splits;
};

template <typename T, int V>
struct Packed {
  uint32_t w[V == 8 ? 4 : 1];
};

template <typename T, int V>
__device__ __forceinline__ Packed<T, V> load_packed(const T* src) {
  Packed<T, V> r;
  if constexpr (V == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(src);
    r.w[0] = q.x, r.w[1] = q.y, r.w[2] = q.z, r.w[3] = q.w;
  } else {
    r.w[0] = *reinterpret_cast<const unsigned short*>(src);
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_packed(T* dst, const Packed<T, V>& r) {
  if constexpr (V == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  else *reinterpret_cast<unsigned short*>(dst) = static_cast<unsigned short>(r.w[0]);
}

// A kept pre-activation is infinite where the number itself left the range of
// the 16-bit type (in fp16 from 65520 on), while the forward pass went on with
// the number.  It counts as 3e38, with its sign: a factor that has vanished
// (dY, act', act) makes 0 of it, as it did of the number, and act' (1.13 at
// most) does not take it out of fp32's range before dY multiplies it.  NaN
// stays NaN.  One minimum of magnitudes an element.
__device__ __forceinline__ float2 kept2(float2 z) {
  float2 r;
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r.x) : "f"(z.x), "f"(3.0e38f));
  asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r.y) : "f"(z.y), "f"(3.0e38f));
  return r;
}

template <typename T, bool GATED, int V>
__global__ void __launch_bounds__(256) linear_dz_kernel(const DzParams p) {
  constexpr int NB = GATED ? 2 : 1;
  constexpr int PAIRS = V == 8 ? 4 : 1;   // a single column is the first half of a pair
  constexpr int ROWS = V == 1 ? 8 : GATED ? 2 : 4;  // loaded ahead
  __shared__ float sums[8][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int side = warp % p.across, phase = warp / p.across, phases = 8 / p.across;
  const int64_t c = ((blockIdx.x * static_cast<int64_t>(p.across) + side) * 32 + lane) * V;
  const int64_t r0 = p.M * blockIdx.y / p.splits, r1 = p.M * (blockIdx.y + 1) / p.splits;
  const bool reads_z = GATED || p.act != CUOPX_ACT_NONE;
  float2 sum[NB][PAIRS];
#pragma unroll
  for (int h = 0; h < NB; ++h)
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) sum[h][i] = both(0.f);
  grid_dependency_wait();
  if (c < p.N) {
    with_activation(p.act, [&](auto act) {
      for (int64_t rb = r0 + phase; rb < r1; rb += ROWS * phases) {
        Packed<T, V> g[ROWS], z[ROWS][NB];
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const int64_t r = rb + j * phases;
          if (r >= r1) break;
          g[j] = load_packed<T, V>(static_cast<const T*>(p.dY) + r * p.lddy + c);
          if (reads_z) {
#pragma unroll
            for (int h = 0; h < NB; ++h) z[j][h] = load_packed<T, V>(static_cast<const T*>(p.Z) + r * p.ldz + h * p.N + c);
          }
        }
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const int64_t r = rb + j * phases;
          if (r >= r1) break;
          Packed<T, V> out[NB];
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            const float2 gg = unpack2_layer<T>(g[j].w[i]);
            float2 d[NB], value;
            if constexpr (GATED) {
              const float2 slope = act_slope2<act.value>(kept2(unpack2_layer<T>(z[j][0].w[i])), value);
              // act'(G) first: where it has vanished, dY * U may be beyond fp32's range.
              d[0] = mul2(mul2(kept2(unpack2_layer<T>(z[j][NB - 1].w[i])), slope), gg);
              d[NB - 1] = mul2(gg, value);
            } else if constexpr (act.value != CUOPX_ACT_NONE) {
              d[0] = mul2(gg, act_slope2<act.value>(unpack2_layer<T>(z[j][0].w[i]), value));
            } else {
              d[0] = gg;
            }
#pragma unroll
            for (int h = 0; h < NB; ++h) {
              sum[h][i] = add2(sum[h][i], d[h]);
              out[h].w[i] = pack2_layer<T>(d[h].x, d[h].y);
            }
          }
          if (p.dZ) {
#pragma unroll
            for (int h = 0; h < NB; ++h) store_packed<T, V>(static_cast<T*>(p.dZ) + r * p.lddz + h * p.N + c, out[h]);
          }
        }
      }
    });
  }
  if (p.partial == nullptr && p.db == nullptr) return;
#pragma unroll
  for (int h = 0; h < NB; ++h) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) sums[warp][i * 32 + lane] = i % 2 ? sum[h][i / 2].y : sum[h][i / 2].x;
    __syncthreads();
    // Adds the row phases' sums of every column of the CTA, in phase order.
    for (int e = threadIdx.x; e < p.across * 32 * V; e += 256) {
      const int w = e / (32 * V), k = e % (32 * V);
      float s = 0.f;
      for (int q = 0; q < phases; ++q) s += sums[q * p.across + w][k];
      const int64_t col = ((blockIdx.x * static_cast<int64_t>(p.across) + w) * 32 + (k & 31)) * V + (k >> 5);
      if (col >= p.N) continue;
      if (p.splits > 1) p.partial[blockIdx.y * (NB * p.N) + h * p.N + col] = s;
      else static_cast<T*>(p.db)[h * p.N + col] = from_acc<T>(s);
    }
  }
}

// Adds the shares' sums: 32 columns per CTA, every eighth share per warp (eight
// loads in flight), then the warps' sums in order; one rounding.
template <typename T>
__global__ void __launch_bounds__(256) linear_db_finish(const float* partial, int splits, int64_t wide, T* db) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  grid_dependency_wait();
  float s = 0.f;
  if (c < wide) {
#pragma unroll 8
    for (int i = warp; i < splits; i += 8) s += partial[i * wide + c];
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < wide) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][lane];
    db[c] = from_acc<T>(s);
  }
}

// Below this many multiplications the SIMT kernel, which takes any alignment,
// beats copying unaligned operands and running on the tensor cores: two more
// launches cost about 4 us.
constexpr double kRepackMinWork = 1048576.0;

// How many pairs share a 256 x 256 tile's K loop.  Measured on B200 (bf16, us
// for 1, 2 and 4 pairs): 256 x 2048 x 8192: 43.1, 26.4, 21.8; 512 x 4096 x
// 4096: 25.3, 19.3, 48.0 (32 tiles: two waves of clusters of eight); 256 x
// 1024 x 1024: 10.5, 9.7, 11.4; 1024 x 4096 x 4096 (64 tiles): 27.6, 37.6,
// 81.1.  So: split while one wave holds all tiles, in four only for deep K.
int pair_split(const LinearProblem& p) {
  const int64_t cols = p.gated ? 128 : 256;
  const int64_t tiles = ((p.M + 255) / 256) * ((p.N + cols - 1) / cols), k_blocks = (p.K + 63) / 64;
  if (!p.gated && k_blocks >= 96 && tiles <= linear_pair_capacity(4)) return 4;
  return k_blocks >= 12 && tiles <= linear_pair_capacity(2) ? 2 : 1;
}

// Whether few rows are better served by the split kernel than by pair tiles.
// Up to 64 rows W's bytes bound it and two CTAs share an SM.  Above, a CTA's
// 128 x 128 tile costs as many L2 bytes per K block as a pair's 256 x 256 one,
// and it wins only while the pairs do not fill the part (128 rows, bf16, us,
// split / pairs: 1024 x 1024 7.2 / 9.8; 4096 x 4096 14.2 / 17.5; N 16384, K
// 4096 36.8 / 30.1; N 2048, K 8192 26.7 / 21.6).
bool few_rows(const LinearProblem& p) {
  if (p.M <= 64) return true;
  if (p.M > 128) return false;
  const int64_t tiles = (p.wide() + 255) / 256;
  return tiles <= 32 && (p.K < 6144 || tiles > linear_pair_capacity(4));
}

// The kernel for a problem whose operands are as aligned as they will be.
int linear_route(const LinearProblem& p, cudaStream_t stream) {
  const bool pair = linear_tc2_supported(p);
  if (linear_split_supported(p) && few_rows(p)) return linear_split(p, stream);
  if (pair) {
    const int ks = pair_split(p);
    return ks > 1 ? linear_pair(p, ks, stream) : linear_tc2(p, stream);
  }
  if (p.transX) return CUOPX_NOT_IMPLEMENTED;  // not reached: its operands are aligned copies
  return linear_simt(p, stream);
}

// ---------------------------------------------------------------- backward plan
struct BackwardPlan {
  bool need_dz;          // dZ differs from dY, or dY's rows are not aligned
  bool copy_x, copy_w;   // aligned copies for the products
  bool tensor;           // products on the tensor cores whatever the alignment of dX and dW
  int64_t lddz;
  int v, across, splits;
  size_t dz_off, partial_off, x_off, w_off, bytes;
};

BackwardPlan backward_plan(const cuopx_linear_backward_args& a, bool gated) {
  BackwardPlan q = {};
  const int64_t wide = gated ? 2 * a.N : a.N;
  if (a.M <= 0 || a.N <= 0 || dtype_size(a.dtype) != 2) return q;
  const bool dx = a.dX && a.K > 0, dw = a.dW && a.K > 0;
  const bool act = gated || a.activation != CUOPX_ACT_NONE;
  q.tensor = static_cast<double>(a.M) * static_cast<double>(wide) * static_cast<double>(a.K) >= kRepackMinWork;
  q.need_dz = (dx || dw) && (act || (q.tensor && !row_aligned16(a.dY, a.lddy)));
  q.copy_x = dw && q.tensor && !row_aligned16(a.X, a.ldx);
  q.copy_w = dx && q.tensor && !row_aligned16(a.W, a.ldw);
  q.lddz = round8(wide);
  const bool vec = a.N % 8 == 0 && row_aligned16(a.dY, a.lddy) && (!act || row_aligned16(a.preact, a.ldz));
  q.v = vec ? 8 : 1;
  // Up to 64 rows all eight warps of a CTA share its columns' rows and the sums
  // need no second launch (64 x 4096 bf16: 6.1 -> 4.4 us; at 128 rows it is even).
  const bool few = a.M <= 64;
  q.across = few ? 1 : a.N > 128 * q.v ? 8 : a.N > 64 * q.v ? 4 : a.N > 32 * q.v ? 2 : 1;
  const int64_t strips = (a.N + 32 * q.v * q.across - 1) / (32 * q.v * q.across);
  // About 16 CTAs per SM, several times what is resident, so that the last
  // wave costs little; at least 8 rows (two batches of loads) for every row phase.
  const int64_t want = (static_cast<int64_t>(device_sm_count()) * 16 + strips - 1) / strips;
  const int64_t least = 8 * (8 / q.across);
  q.splits = few ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, (a.M + least - 1) / least, 1024})));
  size_t off = 0;
  auto take = [&](bool want_it, size_t bytes) {
    const size_t at = off;
    if (want_it) off += round256(bytes);
    return at;
  };
  q.dz_off = take(q.need_dz, static_cast<size_t>(a.M) * q.lddz * 2);
  q.partial_off = take(a.dbias && q.splits > 1, static_cast<size_t>(q.splits) * wide * sizeof(float));
  q.x_off = take(q.copy_x, static_cast<size_t>(a.M) * round8(a.K) * 2);
  const int64_t w_rows = a.transW ? wide : a.K, w_cols = a.transW ? a.K : wide;
  q.w_off = take(q.copy_w, static_cast<size_t>(w_rows) * round8(w_cols) * 2);
  q.bytes = off;
  return q;
}

// C [M][N] = X op(W) for the backward pass, without an epilogue: the GEMM
// back-ends when C's rows are aligned and there are tiles enough for them,
// else the layer kernels, which store any rows and split K.
int backward_product(const LinearProblem& p, bool tensor, cudaStream_t stream) {
  if (tensor && p.K > 0) {
    const bool few = !p.transX && p.M <= 128 && linear_split_supported(p);
    const bool pair = linear_tc2_supported(p);
    if (few || (pair && (!row_aligned16(p.Y, p.ldy) || pair_split(p) > 1))) return linear_route(p, stream);
  }
  GemmProblem g{p.dtype, p.transX, p.transW, p.M, p.N, p.K, 1.0, 0.0, p.X, p.ldx, 0, p.W, p.ldw, 0, p.Y, p.ldy, 0, 1};
  return gemm_route(g, stream);
}

template <typename T, bool GATED>
int launch_dz(const DzParams& d, int v, cudaStream_t stream) {
  const int64_t strip = 32ll * v * d.across;
  const dim3 grid(static_cast<unsigned>((d.N + strip - 1) / strip), static_cast<unsigned>(d.splits));
  cudaError_t e = launch_pdl(v == 8 ? linear_dz_kernel<T, GATED, 8> : linear_dz_kernel<T, GATED, 1>, grid, dim3(256), 0, stream, d);
  note_launch("linear_dz");
  if (e == cudaSuccess && d.splits > 1 && d.db) {
    const int64_t wide = GATED ? 2 * d.N : d.N;
    e = launch_pdl(linear_db_finish<T>, dim3(static_cast<unsigned>((wide + 31) / 32)), dim3(256), 0, stream, d.partial,
                   d.splits, wide, static_cast<T*>(d.db));
    note_launch("linear_db_finish");
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(e);
  }
  return check_launch();
}

bool activation_ok(int act) { return act >= CUOPX_ACT_NONE && act <= CUOPX_ACT_SIGMOID; }

// ---------------------------------------------------------------- entry points
int validate_linear(const cuopx_linear_args& a, bool gated) {
  if (a.dtype != CUOPX_F16 && a.dtype != CUOPX_BF16) return CUOPX_UNSUPPORTED_TYPE;
  if (!activation_ok(a.activation) || a.reserved != 0) return CUOPX_INVALID_ARGUMENT;
  if (a.M < 0 || a.N < 0 || a.K < 0 || a.N > INT64_MAX / 4) return CUOPX_INVALID_ARGUMENT;
  if (gated && a.residual) return CUOPX_INVALID_ARGUMENT;
  if (a.M == 0 || a.N == 0) return CUOPX_SUCCESS;
  const int64_t wide = gated ? 2 * a.N : a.N;
  const int64_t w_rows = a.transW ? wide : a.K, w_cols = a.transW ? a.K : wide;
  if (!starts_on(2, a.X, a.W, a.bias, a.residual, a.Y, a.preact) || !starts_on(256, a.workspace)) return CUOPX_INVALID_ARGUMENT;
  if (!extent_ok(a.M, a.ldy) || (a.K > 0 && (!extent_ok(a.M, a.ldx) || !extent_ok(w_rows, a.ldw))) ||
      (a.preact && !extent_ok(a.M, a.ldz)) || (a.residual && !extent_ok(a.M, a.ldr)))
    return CUOPX_INVALID_ARGUMENT;
  if (!a.Y || a.ldy < a.N || (a.preact && a.ldz < wide) || (a.residual && a.ldr < a.N)) return CUOPX_INVALID_ARGUMENT;
  if (a.K > 0 && (!a.X || !a.W || a.ldx < a.K || a.ldw < w_cols)) return CUOPX_INVALID_ARGUMENT;
  const size_t es = 2;
  const Extent x{a.X, a.M, a.K, a.ldx, es}, w{a.W, w_rows, w_cols, a.ldw, es}, r{a.residual, a.M, a.N, a.ldr, es};
  const Extent y{a.Y, a.M, a.N, a.ldy, es}, z{a.preact, a.M, wide, a.ldz, es};
  const Extent bias = vector_extent(a.bias, static_cast<size_t>(wide) * es);
  const Extent scratch = vector_extent(a.workspace, a.workspace_bytes);
  if (overlaps(y, x) || overlaps(y, w) || overlaps(y, bias) || overlaps(y, z)) return CUOPX_INVALID_ARGUMENT;
  if (overlaps(z, x) || overlaps(z, w) || overlaps(z, bias) || overlaps(z, r)) return CUOPX_INVALID_ARGUMENT;
  if (a.residual && !alias_ok(a.Y, a.ldy, a.residual, a.ldr, a.M, a.N, es)) return CUOPX_INVALID_ARGUMENT;
  for (const Extent& e : {x, w, bias, r, y, z})
    if (overlaps(scratch, e)) return CUOPX_INVALID_ARGUMENT;
  return -1;
}

// Bytes of aligned copies of X and W, and the problem on them when `ws` is given.
size_t repack_plan(LinearProblem& p, char* ws, cudaStream_t stream) {
  size_t off = 0;
  const bool x = !row_aligned16(p.X, p.M == 1 ? 0 : p.ldx);
  const bool split = p.gated && !p.transW && p.w_up % 8;  // the second projection's columns
  const bool w = split || !row_aligned16(p.W, p.ldw);
  if (!x && !w) return 0;
  if (static_cast<double>(p.M) * static_cast<double>(p.wide()) * static_cast<double>(p.K) < kRepackMinWork) return 0;
  if (x) {
    if (ws) {
      linear_repack(p.X, p.M, p.K, p.ldx, 1, 0, ws + off, stream);
      p.X = ws + off;
      p.ldx = round8(p.K);
    }
    off += round256(static_cast<size_t>(p.M) * round8(p.K) * 2);
  }
  if (w) {
    const int64_t rows = p.transW ? p.w_cols() : p.K, cols = p.transW ? p.K : split ? p.N : p.w_cols();
    const int halves = split ? 2 : 1;
    if (ws) {
      linear_repack(p.W, rows, cols, p.ldw, halves, p.w_up, ws + off, stream);
      p.W = ws + off;
      p.ldw = halves * round8(cols);
      if (split) p.w_up = round8(cols);
    }
    off += round256(static_cast<size_t>(rows) * halves * round8(cols) * 2);
  }
  return off;
}

LinearProblem linear_problem(const cuopx_linear_args& a, bool gated) {
  LinearProblem p{a.dtype, a.transW != 0, a.activation, gated, a.M,   a.N,   a.K,      a.X,   a.ldx, a.W,
                  a.ldw,   a.bias,        a.residual,   a.ldr, a.Y, a.ldy, a.preact, a.ldz};
  p.w_up = a.N;
  return p;
}

size_t linear_workspace(const cuopx_linear_args* a, bool gated) {
  if (!a || a->M <= 0 || a->N <= 0 || a->K <= 0) return 0;
  LinearProblem p = linear_problem(*a, gated);
  return repack_plan(p, nullptr, nullptr);
}

int linear_forward(const cuopx_linear_args* a, bool gated, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (const int v = validate_linear(*a, gated); v >= 0) return v;
  LinearProblem p = linear_problem(*a, gated);
  const size_t need = p.K > 0 ? repack_plan(p, nullptr, nullptr) : 0;
  if (need > 0 && a->workspace && a->workspace_bytes >= need) repack_plan(p, static_cast<char*>(a->workspace), stream);
  return linear_route(p, stream);
}

int validate_linear_backward(const cuopx_linear_backward_args& a, bool gated) {
  if (a.dtype != CUOPX_F16 && a.dtype != CUOPX_BF16) return CUOPX_UNSUPPORTED_TYPE;
  if (!activation_ok(a.activation) || a.reserved != 0) return CUOPX_INVALID_ARGUMENT;
  if (a.M < 0 || a.N < 0 || a.K < 0 || a.N > INT64_MAX / 4) return CUOPX_INVALID_ARGUMENT;
  const int64_t wide = gated ? 2 * a.N : a.N;
  const int64_t w_rows = a.transW ? wide : a.K, w_cols = a.transW ? a.K : wide;
  const bool reads_z = gated || a.activation != CUOPX_ACT_NONE;
  const bool dx = a.dX && a.K > 0 && a.M > 0, dw = a.dW && a.K > 0 && a.N > 0, db = a.dbias && a.N > 0;
  if (!dx && !dw && !db) return CUOPX_SUCCESS;
  if (!starts_on(2, a.dY, a.X, a.W, a.preact, a.dX, a.dW, a.dbias) || !starts_on(256, a.workspace)) return CUOPX_INVALID_ARGUMENT;
  if (a.M > 0 && a.N > 0) {
    if (!a.dY || a.lddy < a.N || (reads_z && (!a.preact || a.ldz < wide))) return CUOPX_INVALID_ARGUMENT;
    if (dx && (!a.W || a.ldw < w_cols)) return CUOPX_INVALID_ARGUMENT;
    if (dw && (!a.X || a.ldx < a.K)) return CUOPX_INVALID_ARGUMENT;
  }
  if ((dx && a.lddx < a.K) || (dw && a.lddw < w_cols)) return CUOPX_INVALID_ARGUMENT;
  if (!extent_ok(a.M, a.lddy) || !extent_ok(a.M, wide) || !extent_ok(a.M, a.K) || (reads_z && !extent_ok(a.M, a.ldz)) ||
      (dx && (!extent_ok(a.M, a.lddx) || !extent_ok(w_rows, a.ldw))) ||
      (dw && (!extent_ok(a.M, a.ldx) || !extent_ok(w_rows, a.lddw))))
    return CUOPX_INVALID_ARGUMENT;
  const size_t need = backward_plan(a, gated).bytes;
  if (need > 0 && (!a.workspace || a.workspace_bytes < need)) return CUOPX_RESOURCE_UNAVAILABLE;
  const size_t es = 2;
  const Extent in[4] = {{a.dY, a.M, a.N, a.lddy, es},
                        {dw ? a.X : nullptr, a.M, a.K, a.ldx, es},
                        {dx ? a.W : nullptr, w_rows, w_cols, a.ldw, es},
                        {reads_z ? a.preact : nullptr, a.M, wide, a.ldz, es}};
  const Extent out[4] = {{dx ? a.dX : nullptr, a.M, a.K, a.lddx, es},
                         {dw ? a.dW : nullptr, w_rows, w_cols, a.lddw, es},
                         vector_extent(db ? a.dbias : nullptr, static_cast<size_t>(wide) * es),
                         vector_extent(need ? a.workspace : nullptr, need)};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < 4; ++j)
      if (overlaps(out[i], in[j])) return CUOPX_INVALID_ARGUMENT;
    for (int j = 0; j < i; ++j)
      if (overlaps(out[i], out[j])) return CUOPX_INVALID_ARGUMENT;
  }
  return -1;
}

int linear_backward(const cuopx_linear_backward_args* a, bool gated, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (const int v = validate_linear_backward(*a, gated); v >= 0) return v;
  const int64_t wide = gated ? 2 * a->N : a->N;
  const BackwardPlan q = backward_plan(*a, gated);
  char* ws = static_cast<char*>(a->workspace);
  const void* dz = a->dY;
  int64_t lddz = a->lddy;
  if (a->M == 0 && a->dbias && a->N > 0 && cudaMemsetAsync(a->dbias, 0, static_cast<size_t>(wide) * 2, stream) != cudaSuccess)
    return cuda_failure(cudaGetLastError());
  if (a->M > 0 && a->N > 0 && (q.need_dz || a->dbias)) {
    DzParams d = {};
    d.M = a->M;
    d.N = a->N;
    d.act = a->activation;
    d.dY = a->dY;
    d.lddy = a->lddy;
    d.Z = a->preact;
    d.ldz = a->ldz;
    d.splits = q.splits;
    d.across = q.across;
    if (q.need_dz) {
      d.dZ = ws + q.dz_off;
      d.lddz = q.lddz;
      dz = d.dZ;
      lddz = q.lddz;
    }
    d.db = a->dbias;
    if (a->dbias && q.splits > 1) d.partial = reinterpret_cast<float*>(ws + q.partial_off);
    int rc;
    if (a->dtype == CUOPX_BF16)
      rc = gated ? launch_dz<__nv_bfloat16, true>(d, q.v, stream) : launch_dz<__nv_bfloat16, false>(d, q.v, stream);
    else
      rc = gated ? launch_dz<__half, true>(d, q.v, stream) : launch_dz<__half, false>(d, q.v, stream);
    if (rc != CUOPX_SUCCESS) return rc;
  }
  if (a->dX && a->M > 0 && a->K > 0) {
    // dX [M][K] = dZ [M][wide] op(W)^T: W's columns are the products' depth.
    LinearProblem p{};
    p.dtype = a->dtype;
    p.transW = a->transW == 0;
    p.M = a->M, p.N = a->K, p.K = wide;
    p.X = dz, p.ldx = lddz;
    p.W = a->W, p.ldw = a->ldw;
    p.Y = a->dX, p.ldy = a->lddx;
    if (q.copy_w && wide > 0) {
      const int64_t w_rows = a->transW ? wide : a->K, w_cols = a->transW ? a->K : wide;
      linear_repack(a->W, w_rows, w_cols, a->ldw, 1, 0, ws + q.w_off, stream);
      p.W = ws + q.w_off, p.ldw = round8(w_cols);
    }
    if (const int rc = backward_product(p, q.tensor, stream); rc != CUOPX_SUCCESS) return rc;
  }
  if (a->dW && a->N > 0 && a->K > 0) {
    // dW [K][wide] = X^T dZ, or [wide][K] = dZ^T X.
    const void* x = a->X;
    int64_t ldx = a->ldx;
    if (q.copy_x) {
      linear_repack(a->X, a->M, a->K, a->ldx, 1, 0, ws + q.x_off, stream);
      x = ws + q.x_off, ldx = round8(a->K);
    }
    LinearProblem p{};
    p.dtype = a->dtype;
    p.transX = true;
    p.K = a->M;
    p.M = a->transW ? wide : a->K, p.N = a->transW ? a->K : wide;
    p.X = a->transW ? dz : x, p.ldx = a->transW ? lddz : ldx;
    p.W = a->transW ? x : dz, p.ldw = a->transW ? ldx : lddz;
    p.Y = a->dW, p.ldy = a->lddw;
    if (const int rc = backward_product(p, q.tensor, stream); rc != CUOPX_SUCCESS) return rc;
  }
  return CUOPX_SUCCESS;
}

}  // namespace

}  // namespace cuopx

extern "C" {

size_t cuopx_linear_workspace_size(const cuopx_linear_args* args) { return cuopx::linear_workspace(args, false); }
size_t cuopx_gated_linear_workspace_size(const cuopx_linear_args* args) { return cuopx::linear_workspace(args, true); }

int cuopx_linear(const cuopx_linear_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_linear", args ? args->M : 0, args ? args->N : 0, args ? args->K : 0);
  return scope.done(cuopx::linear_forward(args, false, static_cast<cudaStream_t>(stream)));
}

int cuopx_gated_linear(const cuopx_linear_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_gated_linear", args ? args->M : 0, args ? args->N : 0, args ? args->K : 0);
  return scope.done(cuopx::linear_forward(args, true, static_cast<cudaStream_t>(stream)));
}

size_t cuopx_linear_backward_workspace_size(const cuopx_linear_backward_args* args) {
  return args ? cuopx::backward_plan(*args, false).bytes : 0;
}

size_t cuopx_gated_linear_backward_workspace_size(const cuopx_linear_backward_args* args) {
  return args ? cuopx::backward_plan(*args, true).bytes : 0;
}

int cuopx_linear_backward(const cuopx_linear_backward_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_linear_backward", args ? args->M : 0, args ? args->N : 0, args ? args->K : 0);
  return scope.done(cuopx::linear_backward(args, false, static_cast<cudaStream_t>(stream)));
}

int cuopx_gated_linear_backward(const cuopx_linear_backward_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_gated_linear_backward", args ? args->M : 0, args ? args->N : 0, args ? args->K : 0);
  return scope.done(cuopx::linear_backward(args, true, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
