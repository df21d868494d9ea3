// Dropout with a counter-based generator: the mask is recomputed from (seed,
// offset, element index) wherever it is needed and never stored.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011): ten rounds over a 128-bit counter, two 32 x 32 -> 64
// products each, with a key that grows by a Weyl constant per round.  One
// counter gives the words of four consecutive elements.
#include <cmath>

#include "common.cuh"
#include "dispatch.h"

namespace cuopx {

namespace {

struct Philox4 {
  uint32_t w[4];
};

// The ten rounds' keys, the same for every element: computed on the host.
struct PhiloxKeys {
  uint32_t k0[10], k1[10];
};

PhiloxKeys philox_keys(uint64_t seed) {
  PhiloxKeys k;
  for (uint32_t r = 0; r < 10; ++r) {
    k.k0[r] = static_cast<uint32_t>(seed) + r * 0x9E3779B9u;
    k.k1[r] = static_cast<uint32_t>(seed >> 32) + r * 0xBB67AE85u;
  }
  return k;
}

__device__ __forceinline__ Philox4 philox4x32_10(const PhiloxKeys& keys, uint64_t counter) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32), c2 = 0, c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c0;
    const uint64_t p1 = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ keys.k0[r];
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ keys.k1[r];
    c1 = static_cast<uint32_t>(p1);
    c3 = static_cast<uint32_t>(p0);
  }
  return {{c0, c1, c2, c3}};
}

struct DropoutParams {
  int64_t rows, cols, n;
  bool keep_all;    // p rounds to 0
  uint32_t drop_max;  // otherwise a word up to this one drops its element
  PhiloxKeys keys;
  uint64_t offset;
  const uint64_t* offset_dev;
  float scale;
  const void* x;
  int64_t ldx;
  const void* r;
  int64_t ldr;
  void* y;
  int64_t ldy;
};

// One thread per counter, four elements; any strides and alignment.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutParams p) {
  const uint64_t offset = p.offset + (p.offset_dev ? *p.offset_dev : 0);
  const int64_t groups = (p.n + 3) / 4;
  const T* x = static_cast<const T*>(p.x);
  const T* r = static_cast<const T*>(p.r);
  T* y = static_cast<T*>(p.y);
  for (int64_t g = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; g < groups; g += (int64_t)gridDim.x * blockDim.x) {
    const Philox4 rnd = philox4x32_10(p.keys, offset + static_cast<uint64_t>(g));
    int64_t row = 4 * g / p.cols, col = 4 * g - row * p.cols;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (4 * g + j >= p.n) break;
      float v = p.keep_all || rnd.w[j] > p.drop_max ? to_acc<T>(x[row * p.ldx + col]) * p.scale : 0.f;
      if (r) v += to_acc<T>(r[row * p.ldr + col]);
      y[row * p.ldy + col] = from_acc<T>(v);
      if (++col == p.cols) col = 0, ++row;
    }
  }
}

// 16-byte groups (V elements, V / 4 counters) of rows that start on 16-byte
// boundaries.  In fp32 bound by HBM (one read or two, one write): 8192 x 8192 94
// us, with a residual 128 us (5.7 and 6.3 TB/s).  At 16 bits a group has two
// counters, whose ten rounds cost 5 wide multiplies and 5 three-way xors an
// element: 8192 x 4096 bf16 33.8 us, bound by those (ALU pipe 58 %, dispatch
// stalls); with a residual 42.5 us (4.7 TB/s), bound by latency (issue 59 %
// active, loads the longest stall): a thread has one group in flight.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_vec_kernel(const DropoutParams p) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  grid_dependency_wait();
  const uint64_t offset = p.offset + (p.offset_dev ? *p.offset_dev : 0);
  const int64_t per_row = (p.cols + V - 1) / V, groups = p.rows * per_row;
  // Kept out of the constant bank, from which each round loads them anew:
  // 44.4 -> 42.4 us for 8192 x 4096 bf16 with a residual (fp32 8192 x 8192: 137
  // -> 128), but 33.5 -> 37.1 without one.
  PhiloxKeys keys = p.keys;
  if constexpr (RES) {
#pragma unroll
    for (int r = 0; r < 10; ++r) asm volatile("" : "+r"(keys.k0[r]), "+r"(keys.k1[r]));
  }
  for (int64_t g = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; g < groups; g += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = p.rows == 1 ? 0 : g / per_row;
    const int64_t col = (g - row * per_row) * V;
    const T* xp = static_cast<const T*>(p.x) + row * p.ldx + col;
    const T* rp = static_cast<const T*>(p.r) + row * p.ldr + col;
    T* yp = static_cast<T*>(p.y) + row * p.ldy + col;
    const int64_t left = p.cols - col;  // below V only at the end of a single row
    uint4 xr = make_uint4(0, 0, 0, 0), rr = make_uint4(0, 0, 0, 0);
    if (left >= V) {
      xr = *reinterpret_cast<const uint4*>(xp);
      if constexpr (RES) rr = *reinterpret_cast<const uint4*>(rp);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {  // constant indices keep the groups in registers
        if (i >= left) continue;
        reinterpret_cast<T*>(&xr)[i] = xp[i];
        if constexpr (RES) reinterpret_cast<T*>(&rr)[i] = rp[i];
      }
    }
    const T* x = reinterpret_cast<const T*>(&xr);
    const T* r = reinterpret_cast<const T*>(&rr);
    uint4 yr;
    T* y = reinterpret_cast<T*>(&yr);
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const Philox4 rnd = philox4x32_10(keys, offset + static_cast<uint64_t>(g * (V / 4) + q));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 4 * q + j;
        float v = p.keep_all || rnd.w[j] > p.drop_max ? to_acc<T>(x[i]) * p.scale : 0.f;
        if constexpr (RES) v += to_acc<T>(r[i]);
        y[i] = from_acc<T>(v);
      }
    }
    if (left >= V) {
      *reinterpret_cast<uint4*>(yp) = yr;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < left) yp[i] = y[i];
    }
  }
  grid_launch_dependents();
}

template <typename T>
cudaError_t launch_dropout(const DropoutParams& p, cudaStream_t stream) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  auto ctas = [&](int64_t threads) {
    return static_cast<unsigned>(std::min<int64_t>((threads + 255) / 256, static_cast<int64_t>(device_sm_count()) * 32));
  };
  auto aligned = [&](const void* q, int64_t ld) {
    return reinterpret_cast<uintptr_t>(q) % 16 == 0 && (p.rows == 1 || ld % V == 0);
  };
  if ((p.rows == 1 || p.cols % V == 0) && aligned(p.x, p.ldx) && aligned(p.y, p.ldy) && (!p.r || aligned(p.r, p.ldr))) {
    note_launch("dropout_vec");
    return launch_pdl(p.r ? dropout_vec_kernel<T, true> : dropout_vec_kernel<T, false>,
                      dim3(ctas(p.rows * ((p.cols + V - 1) / V))), dim3(256), 0, stream, p);
  }
  dropout_kernel<T><<<ctas((p.n + 3) / 4), 256, 0, stream>>>(p);
  note_launch("dropout");
  return cudaSuccess;
}

int dropout_impl(const cuopx_dropout_args* a, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (a->dtype != CUOPX_F32 && a->dtype != CUOPX_F16 && a->dtype != CUOPX_BF16) return CUOPX_UNSUPPORTED_TYPE;
  if (a->rows < 0 || a->cols < 0 || !(a->p >= 0.0 && a->p <= 1.0)) return CUOPX_INVALID_ARGUMENT;
  if (a->cols > 0 && a->rows > INT64_MAX / 8 / a->cols) return CUOPX_INVALID_ARGUMENT;
  if (a->rows == 0 || a->cols == 0) return CUOPX_SUCCESS;
  if (!a->X || !a->Y || a->ldx < a->cols || a->ldy < a->cols || (a->residual && a->ldr < a->cols))
    return CUOPX_INVALID_ARGUMENT;
  if (!extent_ok(a->rows, a->ldx) || !extent_ok(a->rows, a->ldy) || (a->residual && !extent_ok(a->rows, a->ldr)))
    return CUOPX_INVALID_ARGUMENT;
  const size_t es = dtype_size(a->dtype);
  if (!starts_on(es, a->X, a->residual, a->Y) || !starts_on(8, a->offset_dev)) return CUOPX_INVALID_ARGUMENT;
  if (!alias_ok(a->Y, a->ldy, a->X, a->ldx, a->rows, a->cols, es)) return CUOPX_INVALID_ARGUMENT;
  if (a->residual && !alias_ok(a->Y, a->ldy, a->residual, a->ldr, a->rows, a->cols, es)) return CUOPX_INVALID_ARGUMENT;
  if (a->offset_dev && overlaps(a->Y, span_bytes(a->rows, a->cols, a->ldy, es), a->offset_dev, 8))
    return CUOPX_INVALID_ARGUMENT;
  DropoutParams p;
  p.rows = a->rows;
  p.cols = a->cols;
  p.n = a->rows * a->cols;
  const uint64_t threshold = static_cast<uint64_t>(std::nearbyint(a->p * 4294967296.0));  // 0 .. 2^32
  p.keep_all = threshold == 0;
  p.drop_max = static_cast<uint32_t>(threshold - 1);
  p.keys = philox_keys(a->seed);
  p.offset = a->offset;
  p.offset_dev = a->offset_dev;
  // Nothing is kept at 2^32; the factor is not used then.
  p.scale = a->p < 1.0 ? static_cast<float>(1.0 / (1.0 - a->p)) : 0.f;
  p.x = a->X;
  p.ldx = a->ldx;
  p.r = a->residual;
  p.ldr = a->ldr;
  p.y = a->Y;
  p.ldy = a->ldy;
  const cudaError_t e = a->dtype == CUOPX_F32   ? launch_dropout<float>(p, stream)
                        : a->dtype == CUOPX_F16 ? launch_dropout<__half>(p, stream)
                                                : launch_dropout<__nv_bfloat16>(p, stream);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(e);
  }
  return check_launch();
}

}  // namespace

}  // namespace cuopx

extern "C" int cuopx_dropout(const cuopx_dropout_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_dropout", args ? args->rows : 0, args ? args->cols : 0, 1);
  return scope.done(cuopx::dropout_impl(args, static_cast<cudaStream_t>(stream)));
}
