// Layer norm over rows and its gradients.
//
//   forward   mean = avg(x), rstd = 1 / sqrt(avg((x - mean)^2) + eps),
//             y = (x - mean) rstd w + b
//   backward  h = (x - mean) rstd, t = dy w,
//             dx = rstd (t - avg(t) - h avg(t h)),
//             dw = sum over rows of dy h, db = sum over rows of dy
//
// The variance is summed from (x - mean), not from x^2: no cancellation when
// the mean is large.  All sums are fp32, in an order fixed by the launch
// shape, without atomics, so results do not change from run to run.
#include "common.cuh"
#include "dispatch.h"

namespace cuopx {

namespace {

struct NormParams {
  int64_t rows, cols;
  float eps;
  const void* x;
  int64_t ldx;
  const void* w;
  const void* b;
  void* y;
  int64_t ldy;
  float* mean;
  float* rstd;
  const void* dy;
  int64_t lddy;
  void* dx;
  int64_t lddx;
  void* dw;
  void* db;
  float* partial;  // [splits][2][cols]: sums of dy h, then of dy
  int splits;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA, the same value in every thread.  `buf` holds 32 floats.
__device__ __forceinline__ float block_sum(float v, float* buf) {
  v = warp_sum(v);
  __syncthreads();  // buf may still be read from the previous call
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = static_cast<int>(blockDim.x) >> 5;
  return warp_sum((threadIdx.x & 31) < warps ? buf[threadIdx.x & 31] : 0.f);
}

// ------------------------------------------------ any size, stride and alignment
// One CTA per row, three passes over it (the second and third from cache).
template <typename T, typename W>
__global__ void __launch_bounds__(256) layer_norm_any(const NormParams p) {
  __shared__ float buf[32];
  const float inv = 1.f / static_cast<float>(p.cols);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    T* y = static_cast<T*>(p.y) + row * p.ldy;
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) s += to_acc<T>(x[c]);
    const float mean = block_sum(s, buf) * inv;
    float v = 0.f;
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
      const float d = to_acc<T>(x[c]) - mean;
      v = fmaf(d, d, v);
    }
    const float rstd = 1.f / sqrtf(fmaf(block_sum(v, buf), inv, p.eps));
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
      const float w = p.w ? to_acc<W>(static_cast<const W*>(p.w)[c]) : 1.f;
      const float b = p.b ? to_acc<W>(static_cast<const W*>(p.b)[c]) : 0.f;
      y[c] = from_acc<T>(fmaf((to_acc<T>(x[c]) - mean) * rstd, w, b));
    }
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(256) layer_norm_dx_any(const NormParams p) {
  __shared__ float buf[32];
  const float inv = 1.f / static_cast<float>(p.cols);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    T* dx = static_cast<T*>(p.dx) + row * p.lddx;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s0 = 0.f, s1 = 0.f;
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
      const float t = to_acc<T>(dy[c]) * (p.w ? to_acc<W>(static_cast<const W*>(p.w)[c]) : 1.f);
      s0 += t;
      s1 = fmaf(t, (to_acc<T>(x[c]) - mean) * rstd, s1);
    }
    const float a0 = block_sum(s0, buf) * inv, a1 = block_sum(s1, buf) * inv;
    for (int64_t c = threadIdx.x; c < p.cols; c += blockDim.x) {
      const float t = to_acc<T>(dy[c]) * (p.w ? to_acc<W>(static_cast<const W*>(p.w)[c]) : 1.f);
      dx[c] = from_acc<T>(rstd * (t - a0 - (to_acc<T>(x[c]) - mean) * rstd * a1));
    }
  }
}

// Partial column sums: 32 columns per CTA, 8 row phases, blockIdx.y-th share of the rows.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_dw_any(const NormParams p) {
  __shared__ float sw[8][32], sb[8][32];
  const int lane = threadIdx.x & 31, phase = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  const int64_t r0 = p.rows * blockIdx.y / p.splits, r1 = p.rows * (blockIdx.y + 1) / p.splits;
  float aw = 0.f, ab = 0.f;
  if (c < p.cols) {
    for (int64_t r = r0 + phase; r < r1; r += 8) {
      const float g = to_acc<T>(static_cast<const T*>(p.dy)[r * p.lddy + c]);
      const float h = (to_acc<T>(static_cast<const T*>(p.x)[r * p.ldx + c]) - p.mean[r]) * p.rstd[r];
      aw = fmaf(g, h, aw);
      ab += g;
    }
  }
  sw[phase][lane] = aw;
  sb[phase][lane] = ab;
  __syncthreads();
  if (phase == 0 && c < p.cols) {
    for (int i = 1; i < 8; ++i) aw += sw[i][lane], ab += sb[i][lane];
    float* out = p.partial + (static_cast<int64_t>(blockIdx.y) * 2) * p.cols;
    out[c] = aw;
    out[p.cols + c] = ab;
  }
}

// Adds the partial sums in ascending order and rounds once.
template <typename W>
__global__ void __launch_bounds__(256) layer_norm_dw_finish(const NormParams p) {
  const int64_t c = blockIdx.x * 256ll + threadIdx.x;
  if (c >= p.cols) return;
  float aw = 0.f, ab = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float* in = p.partial + (static_cast<int64_t>(s) * 2) * p.cols;
    aw += in[c];
    ab += in[p.cols + c];
  }
  if (p.dw) static_cast<W*>(p.dw)[c] = from_acc<W>(aw);
  if (p.db) static_cast<W*>(p.db)[c] = from_acc<W>(ab);
}

// Shares of the rows that the column sums are split into.
int norm_splits(int64_t rows, int64_t cols) {
  const int64_t strips = (cols + 31) / 32;
  const int64_t want = (static_cast<int64_t>(device_sm_count()) * 8 + strips - 1) / strips;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, (rows + 31) / 32, 256})));
}

size_t norm_backward_workspace(const cuopx_layer_norm_args& a) {
  if (a.rows <= 0 || a.cols <= 0 || (!a.dweight && !a.dbias)) return 0;
  return static_cast<size_t>(norm_splits(a.rows, a.cols)) * 2 * static_cast<size_t>(a.cols) * sizeof(float);
}

int norm_types_ok(const cuopx_layer_norm_args& a) {
  if (a.dtype != CUOPX_F32 && a.dtype != CUOPX_F16 && a.dtype != CUOPX_BF16) return CUOPX_UNSUPPORTED_TYPE;
  if (a.wdtype != a.dtype && a.wdtype != CUOPX_F32) return CUOPX_UNSUPPORTED_TYPE;
  if (a.rows < 0 || a.cols < 0) return CUOPX_INVALID_ARGUMENT;
  return -1;
}

// Calls f(T{}, W{}) with the element types of the call.
template <typename F>
void with_norm_types(const cuopx_layer_norm_args& a, F&& f) {
  if (a.dtype == CUOPX_F32) return f(float{}, float{});
  if (a.dtype == CUOPX_F16) return a.wdtype == CUOPX_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
  return a.wdtype == CUOPX_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
}

NormParams norm_params(const cuopx_layer_norm_args& a) {
  NormParams p = {};
  p.rows = a.rows;
  p.cols = a.cols;
  p.eps = static_cast<float>(a.eps);
  p.x = a.X;
  p.ldx = a.ldx;
  p.w = a.weight;
  p.b = a.bias;
  p.y = a.Y;
  p.ldy = a.ldy;
  p.mean = a.mean;
  p.rstd = a.rstd;
  p.dy = a.dY;
  p.lddy = a.lddy;
  p.dx = a.dX;
  p.lddx = a.lddx;
  p.dw = a.dweight;
  p.db = a.dbias;
  return p;
}

unsigned norm_row_ctas(int64_t rows) {
  return static_cast<unsigned>(std::min<int64_t>(rows, static_cast<int64_t>(device_sm_count()) * 8));
}

int layer_norm_impl(const cuopx_layer_norm_args* a, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (const int v = norm_types_ok(*a); v >= 0) return v;
  if (!(a->eps >= 0.0 && a->eps <= 3.0e38)) return CUOPX_INVALID_ARGUMENT;
  if (a->rows == 0 || a->cols == 0) return CUOPX_SUCCESS;
  if (!a->X || !a->Y || a->ldx < a->cols || a->ldy < a->cols) return CUOPX_INVALID_ARGUMENT;
  const size_t es = dtype_size(a->dtype), ws = dtype_size(a->wdtype);
  const size_t yb = span_bytes(a->rows, a->cols, a->ldy, es), xb = span_bytes(a->rows, a->cols, a->ldx, es);
  const size_t wb = static_cast<size_t>(a->cols) * ws, sb = static_cast<size_t>(a->rows) * sizeof(float);
  if (!alias_ok(a->Y, a->ldy, a->X, a->ldx, a->rows, a->cols, es)) return CUOPX_INVALID_ARGUMENT;
  const void* outs[3] = {a->Y, a->mean, a->rstd};
  const size_t outb[3] = {yb, sb, sb};
  for (int i = 0; i < 3; ++i) {
    if (overlaps(outs[i], outb[i], a->weight, wb) || overlaps(outs[i], outb[i], a->bias, wb)) return CUOPX_INVALID_ARGUMENT;
    if (i > 0 && overlaps(outs[i], outb[i], a->X, xb)) return CUOPX_INVALID_ARGUMENT;
    for (int j = 0; j < i; ++j)
      if (overlaps(outs[i], outb[i], outs[j], outb[j])) return CUOPX_INVALID_ARGUMENT;
  }
  const NormParams p = norm_params(*a);
  with_norm_types(*a, [&](auto t, auto w) {
    layer_norm_any<decltype(t), decltype(w)><<<norm_row_ctas(p.rows), 256, 0, stream>>>(p);
  });
  note_launch("layer_norm_any");
  return check_launch();
}

int layer_norm_backward_impl(const cuopx_layer_norm_args* a, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (const int v = norm_types_ok(*a); v >= 0) return v;
  if (a->cols == 0 || (!a->dX && !a->dweight && !a->dbias)) return CUOPX_SUCCESS;
  const size_t es = dtype_size(a->dtype), ws = dtype_size(a->wdtype);
  const size_t wb = static_cast<size_t>(a->cols) * ws, sb = static_cast<size_t>(a->rows) * sizeof(float);
  if (a->rows > 0) {
    if (!a->X || !a->dY || !a->mean || !a->rstd || a->ldx < a->cols || a->lddy < a->cols) return CUOPX_INVALID_ARGUMENT;
    if (a->dX && a->lddx < a->cols) return CUOPX_INVALID_ARGUMENT;
  }
  const size_t need = norm_backward_workspace(*a);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need)) return CUOPX_RESOURCE_UNAVAILABLE;
  const size_t xb = span_bytes(a->rows, a->cols, a->ldx, es), gb = span_bytes(a->rows, a->cols, a->lddy, es);
  const void* outs[4] = {a->dX, a->dweight, a->dbias, need ? a->workspace : nullptr};
  const size_t outb[4] = {span_bytes(a->rows, a->cols, a->lddx, es), wb, wb, need};
  for (int i = 0; i < 4; ++i) {
    if (overlaps(outs[i], outb[i], a->X, xb) || overlaps(outs[i], outb[i], a->weight, wb) ||
        overlaps(outs[i], outb[i], a->mean, sb) || overlaps(outs[i], outb[i], a->rstd, sb))
      return CUOPX_INVALID_ARGUMENT;
    if (i == 0 ? a->dX && !alias_ok(a->dX, a->lddx, a->dY, a->lddy, a->rows, a->cols, es)
               : overlaps(outs[i], outb[i], a->dY, gb))
      return CUOPX_INVALID_ARGUMENT;
    for (int j = 0; j < i; ++j)
      if (overlaps(outs[i], outb[i], outs[j], outb[j])) return CUOPX_INVALID_ARGUMENT;
  }
  NormParams p = norm_params(*a);
  if (a->rows == 0) {  // sums over no rows
    if (a->dweight && cudaMemsetAsync(a->dweight, 0, wb, stream) != cudaSuccess) return cuda_failure(cudaGetLastError());
    if (a->dbias && cudaMemsetAsync(a->dbias, 0, wb, stream) != cudaSuccess) return cuda_failure(cudaGetLastError());
    return CUOPX_SUCCESS;
  }
  if (p.dw || p.db) {  // before dX, which may overwrite dY
    p.partial = static_cast<float*>(a->workspace);
    p.splits = norm_splits(p.rows, p.cols);
    const dim3 grid(static_cast<unsigned>((p.cols + 31) / 32), static_cast<unsigned>(p.splits));
    with_norm_types(*a, [&](auto t, auto w) {
      layer_norm_dw_any<decltype(t)><<<grid, 256, 0, stream>>>(p);
      note_launch("layer_norm_dw_any");
      layer_norm_dw_finish<decltype(w)><<<static_cast<unsigned>((p.cols + 255) / 256), 256, 0, stream>>>(p);
      note_launch("layer_norm_dw_finish");
    });
  }
  if (p.dx) {
    with_norm_types(*a, [&](auto t, auto w) {
      layer_norm_dx_any<decltype(t), decltype(w)><<<norm_row_ctas(p.rows), 256, 0, stream>>>(p);
    });
    note_launch("layer_norm_dx_any");
  }
  return check_launch();
}

}  // namespace

}  // namespace cuopx

extern "C" {

int cuopx_layer_norm(const cuopx_layer_norm_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_layer_norm", args ? args->rows : 0, args ? args->cols : 0, 1);
  return scope.done(cuopx::layer_norm_impl(args, static_cast<cudaStream_t>(stream)));
}

size_t cuopx_layer_norm_backward_workspace_size(const cuopx_layer_norm_args* args) {
  return args ? cuopx::norm_backward_workspace(*args) : 0;
}

int cuopx_layer_norm_backward(const cuopx_layer_norm_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_layer_norm_backward", args ? args->rows : 0, args ? args->cols : 0, 1);
  return scope.done(cuopx::layer_norm_backward_impl(args, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
