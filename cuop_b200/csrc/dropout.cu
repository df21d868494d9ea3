// Dropout with a counter-based generator: the mask is recomputed from (seed,
// offset, element index) wherever it is needed and never stored.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011): ten rounds over a 128-bit counter, two 32 x 32 -> 64
// products each, with a key that grows by a Weyl constant per round.  One
// counter gives the words of four consecutive elements.
#include "common.cuh"
#include "dispatch.h"

namespace cuopx {

namespace {

struct Philox4 {
  uint32_t w[4];
};

__device__ __forceinline__ Philox4 philox4x32_10(uint64_t key, uint64_t counter) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32), c2 = 0, c3 = 0;
  uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(0xD2511F53u) * c0;
    const uint64_t p1 = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c1 = static_cast<uint32_t>(p1);
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

struct DropoutParams {
  int64_t rows, cols, n;
  uint64_t threshold;  // a word below it drops its element; 2^32: all
  uint64_t seed, offset;
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
    const Philox4 rnd = philox4x32_10(p.seed, offset + static_cast<uint64_t>(g));
    int64_t row = 4 * g / p.cols, col = 4 * g - row * p.cols;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (4 * g + j >= p.n) break;
      float v = rnd.w[j] >= p.threshold ? to_acc<T>(x[row * p.ldx + col]) * p.scale : 0.f;
      if (r) v += to_acc<T>(r[row * p.ldr + col]);
      y[row * p.ldy + col] = from_acc<T>(v);
      if (++col == p.cols) col = 0, ++row;
    }
  }
}

template <typename T>
void launch_dropout(const DropoutParams& p, cudaStream_t stream) {
  const int64_t ctas = std::min<int64_t>(((p.n + 3) / 4 + 255) / 256, static_cast<int64_t>(device_sm_count()) * 16);
  dropout_kernel<T><<<static_cast<unsigned>(ctas), 256, 0, stream>>>(p);
  note_launch("dropout");
}

int dropout_impl(const cuopx_dropout_args* a, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (a->dtype != CUOPX_F32 && a->dtype != CUOPX_F16 && a->dtype != CUOPX_BF16) return CUOPX_UNSUPPORTED_TYPE;
  if (a->rows < 0 || a->cols < 0 || !(a->p >= 0.0 && a->p <= 1.0)) return CUOPX_INVALID_ARGUMENT;
  if (a->cols > 0 && a->rows > INT64_MAX / 8 / a->cols) return CUOPX_INVALID_ARGUMENT;
  if (a->rows == 0 || a->cols == 0) return CUOPX_SUCCESS;
  if (!a->X || !a->Y || a->ldx < a->cols || a->ldy < a->cols || (a->residual && a->ldr < a->cols))
    return CUOPX_INVALID_ARGUMENT;
  const size_t es = dtype_size(a->dtype);
  if (!alias_ok(a->Y, a->ldy, a->X, a->ldx, a->rows, a->cols, es)) return CUOPX_INVALID_ARGUMENT;
  if (a->residual && !alias_ok(a->Y, a->ldy, a->residual, a->ldr, a->rows, a->cols, es)) return CUOPX_INVALID_ARGUMENT;
  if (a->offset_dev && overlaps(a->Y, span_bytes(a->rows, a->cols, a->ldy, es), a->offset_dev, 8))
    return CUOPX_INVALID_ARGUMENT;
  DropoutParams p;
  p.rows = a->rows;
  p.cols = a->cols;
  p.n = a->rows * a->cols;
  p.threshold = static_cast<uint64_t>(std::nearbyint(a->p * 4294967296.0));
  p.seed = a->seed;
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
  switch (a->dtype) {
    case CUOPX_F32: launch_dropout<float>(p, stream); break;
    case CUOPX_F16: launch_dropout<__half>(p, stream); break;
    default: launch_dropout<__nv_bfloat16>(p, stream); break;
  }
  return check_launch();
}

}  // namespace

}  // namespace cuopx

extern "C" int cuopx_dropout(const cuopx_dropout_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_dropout", args ? args->rows : 0, args ? args->cols : 0, 1);
  return scope.done(cuopx::dropout_impl(args, static_cast<cudaStream_t>(stream)));
}
