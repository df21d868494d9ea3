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
          if (kk < p.K && n < p.N) v = to_acc<T>(p.transW ? W[(h * p.N + n) * p.ldw + kk] : W[kk * p.ldw + h * p.N + n]);
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

// ---------------------------------------------------------------- dZ and its column sums
// One pass over dY (and Z): writes dZ and, per share of the rows, the fp32
// column sums of the unrounded dZ.  A thread owns V columns (V = 8: one
// 16-byte load per matrix and row), a warp 32 V of them; the eight warps of a
// CTA walk interleaved rows of its share.  Bound by HBM.
struct DzParams {
  int64_t M, N;
  int act;
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
__device__ __forceinline__ void load_acc(const T* src, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_acc<T>(*src);
  } else {
    static_assert(V == 8, "16-byte groups");
    const uint4 raw = *reinterpret_cast<const uint4*>(src);
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_acc<T>(e[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_acc(T* dst, const float (&v)[V]) {
  if constexpr (V == 1) {
    *dst = from_acc<T>(v[0]);
  } else {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_acc<T>(v[i]);
    *reinterpret_cast<uint4*>(dst) = raw;
  }
}

template <typename T, bool GATED, int V>
__global__ void __launch_bounds__(256) linear_dz_kernel(const DzParams p) {
  constexpr int NB = GATED ? 2 : 1;
  __shared__ float sums[8][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (blockIdx.x * 32ll + lane) * V;
  const int64_t r0 = p.M * blockIdx.y / p.splits, r1 = p.M * (blockIdx.y + 1) / p.splits;
  float sum[NB][V] = {};
  if (c < p.N) {
    with_activation(p.act, [&](auto act) {
#pragma unroll 2
      for (int64_t r = r0 + warp; r < r1; r += 8) {
        float g[V], d[NB][V];
        load_acc<T, V>(static_cast<const T*>(p.dY) + r * p.lddy + c, g);
        if constexpr (GATED) {
          float a[V], b[V];
          load_acc<T, V>(static_cast<const T*>(p.Z) + r * p.ldz + c, a);
          load_acc<T, V>(static_cast<const T*>(p.Z) + r * p.ldz + p.N + c, b);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float value;
            const float slope = act_slope<act.value>(a[i], value);
            d[0][i] = g[i] * b[i] * slope;
            d[NB - 1][i] = g[i] * value;
          }
        } else if constexpr (act.value != CUOPX_ACT_NONE) {
          float z[V];
          load_acc<T, V>(static_cast<const T*>(p.Z) + r * p.ldz + c, z);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float value;
            d[0][i] = g[i] * act_slope<act.value>(z[i], value);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) d[0][i] = g[i];
        }
#pragma unroll
        for (int h = 0; h < NB; ++h) {
          if (p.dZ) store_acc<T, V>(static_cast<T*>(p.dZ) + r * p.lddz + h * p.N + c, d[h]);
#pragma unroll
          for (int i = 0; i < V; ++i) sum[h][i] += d[h][i];
        }
      }
    });
  }
  if (p.partial == nullptr && p.db == nullptr) return;
#pragma unroll
  for (int h = 0; h < NB; ++h) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) sums[warp][i * 32 + lane] = sum[h][i];
    __syncthreads();
    // Thread t adds the eight warps' sums of V / 8 (at least one) column of the CTA.
    for (int e = threadIdx.x; e < 32 * V; e += 256) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += sums[w][e];
      const int64_t col = (blockIdx.x * 32ll + (e & 31)) * V + (e >> 5);
      if (col >= p.N) continue;
      if (p.splits > 1) p.partial[blockIdx.y * (NB * p.N) + h * p.N + col] = s;
      else static_cast<T*>(p.db)[h * p.N + col] = from_acc<T>(s);
    }
  }
}

// Adds the shares' sums in ascending order and rounds once.
template <typename T>
__global__ void __launch_bounds__(256) linear_db_finish(const float* partial, int splits, int64_t wide, T* db) {
  const int64_t c = blockIdx.x * 256ll + threadIdx.x;
  if (c >= wide) return;
  float s = 0.f;
  for (int i = 0; i < splits; ++i) s += partial[i * wide + c];
  db[c] = from_acc<T>(s);
}

// ---------------------------------------------------------------- backward plan
struct BackwardPlan {
  bool need_dz;  // dZ differs from dY
  int64_t lddz;
  int v, splits;
  size_t dz_off, partial_off, bytes;
};

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

BackwardPlan backward_plan(const cuopx_linear_backward_args& a, bool gated) {
  BackwardPlan q = {};
  const int64_t wide = gated ? 2 * a.N : a.N;
  if (a.M <= 0 || a.N <= 0 || dtype_size(a.dtype) == 0) return q;
  q.need_dz = (gated || a.activation != CUOPX_ACT_NONE) && (a.dX || a.dW) && a.K > 0;
  q.lddz = (wide + 7) / 8 * 8;
  const bool vec = a.N % 8 == 0 && row_aligned16(a.dY, a.lddy) &&
                   ((!gated && a.activation == CUOPX_ACT_NONE) || row_aligned16(a.preact, a.ldz));
  q.v = vec ? 8 : 1;
  const int64_t strips = (a.N + 32 * q.v - 1) / (32 * q.v);
  const int64_t want = (static_cast<int64_t>(device_sm_count()) * 4 + strips - 1) / strips;
  q.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, (a.M + 15) / 16, 1024})));
  size_t off = 0;
  if (q.need_dz) {
    q.dz_off = off;
    off += round256(static_cast<size_t>(a.M) * q.lddz * dtype_size(a.dtype));
  }
  if (a.dbias && q.splits > 1) {
    q.partial_off = off;
    off += round256(static_cast<size_t>(q.splits) * wide * sizeof(float));
  }
  q.bytes = off;
  return q;
}

template <typename T, bool GATED>
void launch_dz(const DzParams& d, int v, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((d.N + 32 * v - 1) / (32 * v)), static_cast<unsigned>(d.splits));
  if (v == 8) linear_dz_kernel<T, GATED, 8><<<grid, 256, 0, stream>>>(d);
  else linear_dz_kernel<T, GATED, 1><<<grid, 256, 0, stream>>>(d);
  note_launch("linear_dz");
  if (d.splits > 1 && d.db) {
    const int64_t wide = GATED ? 2 * d.N : d.N;
    linear_db_finish<T><<<static_cast<unsigned>((wide + 255) / 256), 256, 0, stream>>>(d.partial, d.splits, wide,
                                                                                      static_cast<T*>(d.db));
    note_launch("linear_db_finish");
  }
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
  if (!a.Y || a.ldy < a.N || (a.preact && a.ldz < wide) || (a.residual && a.ldr < a.N)) return CUOPX_INVALID_ARGUMENT;
  if (a.K > 0 && (!a.X || !a.W || a.ldx < a.K || a.ldw < w_cols)) return CUOPX_INVALID_ARGUMENT;
  const size_t es = 2;
  const size_t yb = span_bytes(a.M, a.N, a.ldy, es), zb = a.preact ? span_bytes(a.M, wide, a.ldz, es) : 0;
  const size_t xb = span_bytes(a.M, a.K, a.ldx, es), wb = span_bytes(w_rows, w_cols, a.ldw, es);
  const size_t bb = static_cast<size_t>(wide) * es, rb = a.residual ? span_bytes(a.M, a.N, a.ldr, es) : 0;
  if (overlaps(a.Y, yb, a.X, xb) || overlaps(a.Y, yb, a.W, wb) || overlaps(a.Y, yb, a.bias, bb) ||
      overlaps(a.Y, yb, a.preact, zb))
    return CUOPX_INVALID_ARGUMENT;
  if (overlaps(a.preact, zb, a.X, xb) || overlaps(a.preact, zb, a.W, wb) || overlaps(a.preact, zb, a.bias, bb) ||
      overlaps(a.preact, zb, a.residual, rb))
    return CUOPX_INVALID_ARGUMENT;
  if (a.residual && !alias_ok(a.Y, a.ldy, a.residual, a.ldr, a.M, a.N, es)) return CUOPX_INVALID_ARGUMENT;
  return -1;
}

int linear_forward(const cuopx_linear_args* a, bool gated, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (const int v = validate_linear(*a, gated); v >= 0) return v;
  LinearProblem p{a->dtype, a->transW != 0, a->activation, gated, a->M,   a->N,   a->K,      a->X,   a->ldx, a->W,
                  a->ldw,   a->bias,        a->residual,   a->ldr, a->Y, a->ldy, a->preact, a->ldz};
  if (p.M <= 128 && linear_split_supported(p)) return linear_split(p, stream);
  if (linear_tc2_supported(p) && p.M >= 64) return linear_tc2(p, stream, 256);
  return linear_simt(p, stream);
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
  if (a.M > 0 && a.N > 0) {
    if (!a.dY || a.lddy < a.N || (reads_z && (!a.preact || a.ldz < wide))) return CUOPX_INVALID_ARGUMENT;
    if (dx && (!a.W || a.ldw < w_cols)) return CUOPX_INVALID_ARGUMENT;
    if (dw && (!a.X || a.ldx < a.K)) return CUOPX_INVALID_ARGUMENT;
  }
  if ((dx && a.lddx < a.K) || (dw && a.lddw < w_cols)) return CUOPX_INVALID_ARGUMENT;
  const size_t need = backward_plan(a, gated).bytes;
  if (need > 0 && (!a.workspace || a.workspace_bytes < need)) return CUOPX_RESOURCE_UNAVAILABLE;
  const size_t es = 2;
  const void* in[4] = {a.dY, dw ? a.X : nullptr, dx ? a.W : nullptr, reads_z ? a.preact : nullptr};
  const size_t inb[4] = {span_bytes(a.M, a.N, a.lddy, es), span_bytes(a.M, a.K, a.ldx, es),
                         span_bytes(w_rows, w_cols, a.ldw, es), span_bytes(a.M, wide, a.ldz, es)};
  const void* out[4] = {dx ? a.dX : nullptr, dw ? a.dW : nullptr, db ? a.dbias : nullptr, need ? a.workspace : nullptr};
  const size_t outb[4] = {span_bytes(a.M, a.K, a.lddx, es), span_bytes(w_rows, w_cols, a.lddw, es),
                          static_cast<size_t>(wide) * es, need};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < 4; ++j)
      if (overlaps(out[i], outb[i], in[j], inb[j])) return CUOPX_INVALID_ARGUMENT;
    for (int j = 0; j < i; ++j)
      if (overlaps(out[i], outb[i], out[j], outb[j])) return CUOPX_INVALID_ARGUMENT;
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
    if (q.need_dz) {
      d.dZ = ws + q.dz_off;
      d.lddz = q.lddz;
      dz = d.dZ;
      lddz = q.lddz;
    }
    d.db = a->dbias;
    if (a->dbias && q.splits > 1) d.partial = reinterpret_cast<float*>(ws + q.partial_off);
    if (a->dtype == CUOPX_BF16) gated ? launch_dz<__nv_bfloat16, true>(d, q.v, stream) : launch_dz<__nv_bfloat16, false>(d, q.v, stream);
    else gated ? launch_dz<__half, true>(d, q.v, stream) : launch_dz<__half, false>(d, q.v, stream);
    if (const int rc = check_launch(); rc != CUOPX_SUCCESS) return rc;
  }
  if (a->dX && a->M > 0 && a->K > 0) {
    // dX [M][K] = dZ [M][wide] W^T
    GemmProblem g{a->dtype, false, a->transW == 0, a->M, a->K, wide, 1.0, 0.0, dz, lddz, 0, a->W, a->ldw, 0,
                  a->dX, a->lddx, 0, 1};
    if (const int rc = gemm_route(g, stream); rc != CUOPX_SUCCESS) return rc;
  }
  if (a->dW && a->N > 0 && a->K > 0) {
    // dW [K][wide] = X^T dZ, or [wide][K] = dZ^T X
    GemmProblem g = a->transW ? GemmProblem{a->dtype, true, false, wide, a->K, a->M, 1.0, 0.0, dz, lddz, 0, a->X, a->ldx,
                                            0, a->dW, a->lddw, 0, 1}
                              : GemmProblem{a->dtype, true, false, a->K, wide, a->M, 1.0, 0.0, a->X, a->ldx, 0, dz, lddz,
                                            0, a->dW, a->lddw, 0, 1};
    if (const int rc = gemm_route(g, stream); rc != CUOPX_SUCCESS) return rc;
  }
  return CUOPX_SUCCESS;
}

}  // namespace

}  // namespace cuopx

extern "C" {

size_t cuopx_linear_workspace_size(const cuopx_linear_args*) { return 0; }
size_t cuopx_gated_linear_workspace_size(const cuopx_linear_args*) { return 0; }

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
