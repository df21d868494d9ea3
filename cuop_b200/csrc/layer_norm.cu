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
//
// Bound by HBM: every element is read once and written once.  A warp or a CTA
// has a row, which stays packed in its threads' registers between the sums and
// the result.  Forward (layer_norm_rows), rows are loaded straight into
// registers, with a CTA, or a warp, for every row.  Backward, one kernel reads x
// and dy once for all three gradients: persistent groups of threads, each with
// the same columns of all its rows, whose two column sums stay in registers; one
// partial sum per CTA and column goes to the workspace, and a second small
// kernel adds those in CTA order.  Rows on 16-byte boundaries come through a
// ring of shared-memory stages filled by bulk copies (layer_norm_backward_ring),
// so that what is in flight costs no registers; others as single elements
// (layer_norm_backward_rows).  The *_any kernels take what neither does.
// Measured: fp32 16384 x 4096 forward 93 us (5.7 TB/s), backward 132 us (6.1);
// bf16 8192 x 8192 63 us (4.3 TB/s), bound by the instructions around each
// element, conversions first (issue 72 % active), and 92 us (4.4), bound by
// latency (issue 54 %): one CTA of 1024 threads per SM, whose warps meet at a
// barrier every two rows.
#include "common.cuh"
#include "dispatch.h"
#include "layer_epilogue.cuh"

namespace cuopx {

namespace {

struct NormParams {
  int64_t rows, cols;
  float eps;
  const void* x;
  int64_t ldx;
  const void* w;
  const void* b;
  bool vec_w, vec_b;  // weight, bias start on 16-byte boundaries
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

// ------------------------------------------------ ring of rows in shared memory
// One bulk copy of `bytes` (a multiple of 16, both addresses on 16-byte
// boundaries) from global to this CTA's shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The rows first, first + step, ... of up to two matrices, each stage one row
// of every matrix.  A group's leader thread issues the copies; every thread
// waits for a stage, and the stage is filled again once the whole group has
// read it (which the caller orders).
template <int NSRC>
struct RowRing {
  unsigned char* base;  // [stages][NSRC][bytes]
  uint64_t* full;       // [stages]
  int stages;
  uint32_t bytes;
  const unsigned char* src[NSRC];
  int64_t pitch[NSRC];  // bytes from row to row
  int64_t rows, step;
  volatile int* abort;

  __device__ __forceinline__ void fill(int stage, int64_t row) const {
    mbar_arrive_expect_tx(&full[stage], NSRC * bytes);
#pragma unroll
    for (int i = 0; i < NSRC; ++i) bulk_load(base + (stage * NSRC + i) * bytes, src[i] + row * pitch[i], bytes, &full[stage]);
  }
  // Fills the first stages; the number filled.
  __device__ __forceinline__ int64_t start(int64_t first) const {
    int s = 0;
    for (; s < stages && first + s * step < rows; ++s) fill(s, first + s * step);
    return s;
  }
  // After a timeout (recorded): let the copies in flight land, with a limit of their own.
  __device__ __forceinline__ void drain(int64_t filled) const {
    for (int s = 0; s < stages && s < filled; ++s) {
      const uint32_t parity = static_cast<uint32_t>((filled - s + stages - 1) / stages - 1) & 1u;
      const unsigned long long t0 = global_timer_ns();
      while (!mbar_try_wait(smem_u32(&full[s]), parity)) {
        if (global_timer_ns() - t0 > kWaitLimitNs) {
          record_device_error(kDevErrAbortDrain);
          break;
        }
      }
    }
  }
  __device__ __forceinline__ bool wait(int stage, uint32_t phase) const {
    return mbar_wait_bounded(&full[stage], phase, kDevErrWaitTimeoutFull, abort);
  }
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

// ------------------------------------------------ rows in registers
// A thread holds NV groups of V neighbouring columns: group g of thread t is
// columns [V (t + G g), ...), G threads per row.  V elements are one 16-byte
// load, or V = 1 where rows are not 16-byte aligned.
template <typename T, int V>
struct RowVec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ RowVec<T, V> load_vec(const T* p) {
  RowVec<T, V> r;
  if constexpr (V == 1) {
    r.e[0] = *p;
  } else {
    static_assert(sizeof(r) == 16, "16-byte groups");
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const RowVec<T, V>& r) {
  if constexpr (V == 1) *p = r.e[0];
  else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
}

// Elements 2i and 2i + 1 of a group widened, and two results rounded into it.
// Arithmetic is in packed pairs: at 16 bits an element HBM leaves about 22
// issue slots per element forward and 32 backward.
template <typename T, int V>
__device__ __forceinline__ float2 widen2(const RowVec<T, V>& r, int i) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    return unpack2_layer<T>(reinterpret_cast<const uint32_t*>(&r)[i]);
  } else {
    return make_float2(to_acc<T>(r.e[2 * i]), to_acc<T>(r.e[2 * i + 1]));
  }
}
template <typename T, int V>
__device__ __forceinline__ void round2(RowVec<T, V>& r, int i, float2 v) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    reinterpret_cast<uint32_t*>(&r)[i] = pack2_layer<T>(v.x, v.y);
  } else {
    r.e[2 * i] = from_acc<T>(v.x);
    r.e[2 * i + 1] = from_acc<T>(v.y);
  }
}

// V weights from column c on, in 16-byte loads where `vec` says that they start on such a boundary.
template <typename W, int V>
__device__ __forceinline__ void load_weights(const W* w, int64_t c, bool vec, float (&out)[V]) {
  constexpr int E = 16 / static_cast<int>(sizeof(W));
  if constexpr (V % E == 0) {
    if (vec) {
#pragma unroll
      for (int j = 0; j < V / E; ++j) {
        const RowVec<W, E> r = load_vec<W, E>(w + c + j * E);
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          const float2 f = widen2<W, E>(r, i);
          out[j * E + 2 * i] = f.x;
          out[j * E + 2 * i + 1] = f.y;
        }
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = to_acc<W>(w[c + i]);
}

// V weights from column c on, as pairs.
template <typename W, int V>
__device__ __forceinline__ void load_weights2(const W* w, int64_t c, bool vec, float2 (&out)[V / 2]) {
  float f[V];
  load_weights<W, V>(w, c, vec, f);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) out[i] = make_float2(f[2 * i], f[2 * i + 1]);
}

// Sums of two values over the threads of a row: the warp, or the CTA through
// one of two alternating buffers (one barrier: a thread writes a buffer again
// only after every thread has arrived at the barrier after its last reads).
template <bool WARP>
__device__ __forceinline__ float2 row_sum(float a, float b, float2 (*buf)[32], int& parity) {
  a = warp_sum(a);
  b = warp_sum(b);
  if constexpr (!WARP) {
    if ((threadIdx.x & 31) == 0) buf[parity][threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    const int warps = static_cast<int>(blockDim.x) >> 5;
    const float2 v = (threadIdx.x & 31) < warps ? buf[parity][threadIdx.x & 31] : make_float2(0.f, 0.f);
    a = warp_sum(v.x);
    b = warp_sum(v.y);
    parity ^= 1;
  }
  return make_float2(a, b);
}

// Four values at once: each exchange halves the number of values a lane still
// sums, so the warp's four totals take 6 shuffles instead of 20.  After it,
// lanes with (lane >> 3) == j hold the total of value j.
__device__ __forceinline__ float warp_sum4(float4 v) {
  const int lane = static_cast<int>(threadIdx.x & 31);
  const bool hi = lane & 16, mid = lane & 8;
  float a = hi ? v.z : v.x, b = hi ? v.w : v.y;  // kept
  a += __shfl_xor_sync(0xffffffffu, hi ? v.x : v.z, 16);
  b += __shfl_xor_sync(0xffffffffu, hi ? v.y : v.w, 16);
  float c = mid ? b : a;
  c += __shfl_xor_sync(0xffffffffu, mid ? a : b, 8);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  return c;
}

template <bool WARP>
__device__ __forceinline__ float4 row_sum4(float4 v, float4 (*buf)[32], int& parity) {
  float c = warp_sum4(v);
  if constexpr (!WARP) {
    const int lane = static_cast<int>(threadIdx.x & 31);
    if ((lane & 7) == 0) reinterpret_cast<float*>(&buf[parity][threadIdx.x >> 5])[lane >> 3] = c;
    __syncthreads();
    const int warps = static_cast<int>(blockDim.x) >> 5;
    c = warp_sum4(lane < warps ? buf[parity][lane] : make_float4(0.f, 0.f, 0.f, 0.f));
    parity ^= 1;
  }
  return make_float4(__shfl_sync(0xffffffffu, c, 0), __shfl_sync(0xffffffffu, c, 8), __shfl_sync(0xffffffffu, c, 16),
                     __shfl_sync(0xffffffffu, c, 24));
}

template <bool WARP>
__device__ __forceinline__ float row_sum1(float a, float2 (*buf)[32], int& parity) {
  a = warp_sum(a);
  if constexpr (!WARP) {
    if ((threadIdx.x & 31) == 0) buf[parity][threadIdx.x >> 5].x = a;
    __syncthreads();
    const int warps = static_cast<int>(blockDim.x) >> 5;
    a = warp_sum((threadIdx.x & 31) < warps ? buf[parity][threadIdx.x & 31].x : 0.f);
    parity ^= 1;
  }
  return a;
}

// Statistics and result of one row of 16-byte groups, kept packed and widened
// for each of the three passes: keeping it widened costs the registers of a
// third of the warps.
template <typename T, typename W, int V, int NV, bool WARP>
__device__ __forceinline__ void norm_one_row(const NormParams& p, int64_t row, const RowVec<T, V> (&raw)[NV], int t, int G,
                                             float2 (*buf)[32], int& parity) {
  const int cols = static_cast<int>(p.cols);
  const float inv = 1.f / static_cast<float>(cols);
  T* y = static_cast<T*>(p.y) + row * p.ldy;
  float2 s = both(0.f);
#pragma unroll
  for (int g = 0; g < NV; ++g)
    if (V * (t + G * g) < cols)
#pragma unroll
      for (int i = 0; i < V / 2; ++i) s = add2(s, widen2<T, V>(raw[g], i));
  const float mean = row_sum1<WARP>(s.x + s.y, buf, parity) * inv;
  float2 q = both(0.f);
#pragma unroll
  for (int g = 0; g < NV; ++g)
    if (V * (t + G * g) < cols)
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 d = add2(widen2<T, V>(raw[g], i), both(-mean));
        q = fma2(d, d, q);
      }
  const float rstd = 1.f / sqrtf(fmaf(row_sum1<WARP>(q.x + q.y, buf, parity), inv, p.eps));
  if (t == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    const int c = V * (t + G * g);
    if (c >= cols) continue;
    float2 w[V / 2], b[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = both(1.f), b[i] = both(0.f);
    if (p.w) load_weights2<W, V>(static_cast<const W*>(p.w), c, p.vec_w, w);
    if (p.b) load_weights2<W, V>(static_cast<const W*>(p.b), c, p.vec_b, b);
    RowVec<T, V> out;
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      round2<T, V>(out, i, fma2(mul2(add2(widen2<T, V>(raw[g], i), both(-mean)), both(rstd)), w[i], b[i]));
    store_vec<T, V>(y + c, out);
  }
}

// The same for rows that are not 16-byte aligned: single elements.
template <typename T, typename W, int NV, bool WARP>
__device__ __forceinline__ void norm_one_row(const NormParams& p, int64_t row, const RowVec<T, 1> (&raw)[NV], int t, int G,
                                             float2 (*buf)[32], int& parity) {
  const int cols = static_cast<int>(p.cols);
  const float inv = 1.f / static_cast<float>(cols);
  float v[NV], s = 0.f, q = 0.f;
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    v[g] = t + G * g < cols ? to_acc<T>(raw[g].e[0]) : 0.f;
    s += v[g];
  }
  const float mean = row_sum1<WARP>(s, buf, parity) * inv;
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    v[g] -= mean;
    if (t + G * g < cols) q = fmaf(v[g], v[g], q);
  }
  const float rstd = 1.f / sqrtf(fmaf(row_sum1<WARP>(q, buf, parity), inv, p.eps));
  if (t == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    const int c = t + G * g;
    if (c >= cols) continue;
    const float w = p.w ? to_acc<W>(static_cast<const W*>(p.w)[c]) : 1.f;
    const float b = p.b ? to_acc<W>(static_cast<const W*>(p.b)[c]) : 0.f;
    static_cast<T*>(p.y)[row * p.ldy + c] = from_acc<T>(fmaf(v[g] * rstd, w, b));
  }
}

// Forward: rows loaded straight into registers.  The ring of the backward
// kernel measured slower here (8192 x 8192 bf16: 80 us for a CTA per row, 216
// for a warp per row): with 64 registers a thread, four CTAs of eight warps
// per SM keep enough rows in flight and hide one another's barriers.
template <typename T, typename W, int V, int NV, bool WARP, int MAXT, int CTAS>
__global__ void __launch_bounds__(MAXT, CTAS) layer_norm_rows(const NormParams p) {
  __shared__ float2 buf[2][32];
  int parity = 0;
  const int G = WARP ? 32 : static_cast<int>(blockDim.x);
  const int t = WARP ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
  const int64_t first = WARP ? blockIdx.x * static_cast<int64_t>(blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = WARP ? gridDim.x * static_cast<int64_t>(blockDim.x >> 5) : gridDim.x;
  grid_dependency_wait();
  for (int64_t row = first; row < p.rows; row += step) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    RowVec<T, V> v[NV];
#pragma unroll
    for (int g = 0; g < NV; ++g)
      if (V * (t + G * g) < p.cols) v[g] = load_vec<T, V>(x + V * (t + G * g));
    if constexpr (V == 1) norm_one_row<T, W, NV, WARP>(p, row, v, t, G, buf, parity);
    else norm_one_row<T, W, V, NV, WARP>(p, row, v, t, G, buf, parity);
  }
  grid_launch_dependents();
}

// Backward for rows that are not 16-byte aligned: single elements, NV columns
// per thread, the next row's on their way while a row is worked on.
template <typename T, typename W, int NV, bool WARP, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) layer_norm_backward_rows(const NormParams p) {
  __shared__ float2 buf[2][32];
  extern __shared__ float warp_part[];  // WARP: [warps][2][32 NV]
  int parity = 0;
  const int G = WARP ? 32 : static_cast<int>(blockDim.x);
  const int t = WARP ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
  const int64_t first = WARP ? blockIdx.x * static_cast<int64_t>(blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = WARP ? gridDim.x * static_cast<int64_t>(blockDim.x >> 5) : gridDim.x;
  const int cols = static_cast<int>(p.cols);
  const float inv = 1.f / static_cast<float>(cols);
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  T* dx = static_cast<T*>(p.dx);
  float aw[NV] = {}, ab[NV] = {};
  grid_dependency_wait();
  T nx[NV], ng[NV];
  float nmean = 0.f, nrstd = 0.f;
  auto fetch = [&](int64_t row) {
    if (row >= p.rows) return;
    nmean = p.mean[row];
    nrstd = p.rstd[row];
#pragma unroll
    for (int g = 0; g < NV; ++g) {
      const int c = t + G * g;
      if (c < cols) nx[g] = x[row * p.ldx + c], ng[g] = dy[row * p.lddy + c];
    }
  };
  fetch(first);
  for (int64_t row = first; row < p.rows; row += step) {
    const float mean = nmean, rstd = nrstd;
    float h[NV], d[NV];  // normalised x; dy w
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int g = 0; g < NV; ++g) {
      const int c = t + G * g;
      h[g] = d[g] = 0.f;
      if (c >= cols) continue;
      h[g] = (to_acc<T>(nx[g]) - mean) * rstd;
      d[g] = to_acc<T>(ng[g]);
      aw[g] = fmaf(d[g], h[g], aw[g]);
      ab[g] += d[g];
      if (p.w) d[g] *= to_acc<W>(static_cast<const W*>(p.w)[c]);
      s0 += d[g];
      s1 = fmaf(d[g], h[g], s1);
    }
    fetch(row + step);
    if (dx) {
      const float2 sum = row_sum<WARP>(s0, s1, buf, parity);
      const float a0 = sum.x * inv, a1 = sum.y * inv;
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        const int c = t + G * g;
        if (c < cols) dx[row * p.lddx + c] = from_acc<T>(rstd * (d[g] - a0 - h[g] * a1));
      }
    }
  }
  if (p.partial) {
    float* out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.cols;
    if constexpr (WARP) {
      // Add the warps' sums in warp order.
      constexpr int COLS = 32 * NV;
      const int warps = static_cast<int>(blockDim.x >> 5);
      float* mine = warp_part + static_cast<int>(threadIdx.x >> 5) * 2 * COLS;
#pragma unroll
      for (int g = 0; g < NV; ++g) mine[t + 32 * g] = aw[g], mine[COLS + t + 32 * g] = ab[g];
      __syncthreads();
      for (int e = threadIdx.x; e < 2 * COLS; e += static_cast<int>(blockDim.x)) {
        const int c = e % COLS, which = e / COLS;
        if (c >= cols) continue;
        float s = 0.f;
        for (int i = 0; i < warps; ++i) s += warp_part[i * 2 * COLS + e];
        out[which * p.cols + c] = s;
      }
    } else {
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        const int c = t + G * g;
        if (c < cols) out[c] = aw[g], out[p.cols + c] = ab[g];
      }
    }
  }
  grid_launch_dependents();
}

// The same for rows on 16-byte boundaries, through the ring.  WARP: eight
// rings per CTA, one per warp.
template <typename T, typename W, int V, int NV, bool WARP, int MAXT, int CTAS, int ROWS>
__global__ void __launch_bounds__(MAXT, CTAS) layer_norm_backward_ring(const NormParams p, int stages) {
  extern __shared__ __align__(128) unsigned char ring_smem[];  // rings; WARP: afterwards [warps][2][32 V NV] sums
  __shared__ float4 buf[2][32];
  __shared__ uint64_t full[8 * 8];
  __shared__ int abort_flag;
  int parity = 0;
  const int G = WARP ? 32 : static_cast<int>(blockDim.x);
  const int t = WARP ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
  const int group = WARP ? static_cast<int>(threadIdx.x >> 5) : 0;
  const int groups = WARP ? static_cast<int>(blockDim.x >> 5) : 1;
  const int64_t first = blockIdx.x * static_cast<int64_t>(groups) + group;
  const int64_t step = gridDim.x * static_cast<int64_t>(groups);
  const int cols = static_cast<int>(p.cols);
  const float inv = 1.f / static_cast<float>(cols);
  RowRing<2> ring;
  ring.bytes = static_cast<uint32_t>(p.cols * static_cast<int64_t>(sizeof(T)));
  ring.base = ring_smem + static_cast<size_t>(group) * stages * 2 * ring.bytes;
  ring.full = full + group * stages;
  ring.stages = stages;
  ring.src[0] = static_cast<const unsigned char*>(p.x);
  ring.src[1] = static_cast<const unsigned char*>(p.dy);
  ring.pitch[0] = p.ldx * static_cast<int64_t>(sizeof(T));
  ring.pitch[1] = p.lddy * static_cast<int64_t>(sizeof(T));
  ring.rows = p.rows;
  ring.step = step;
  ring.abort = &abort_flag;
  if (threadIdx.x == 0) {
    for (int s = 0; s < groups * stages; ++s) mbar_init(&full[s], 1);
    abort_flag = 0;
    fence_mbarrier_init();
  }
  __syncthreads();
  grid_dependency_wait();
  int64_t filled = t == 0 ? ring.start(first) : 0;
  float2 aw[NV][V / 2], ab[NV][V / 2], ww[NV][V / 2];
#pragma unroll
  for (int g = 0; g < NV; ++g) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) aw[g][i] = ab[g][i] = both(0.f), ww[g][i] = both(1.f);
    if (p.w && V * (t + G * g) < cols) load_weights2<W, V>(static_cast<const W*>(p.w), V * (t + G * g), p.vec_w, ww[g]);
  }
  // ROWS (1 or 2) rows per step: one exchange of their sums.
  float nmean[ROWS] = {}, nrstd[ROWS] = {};
  auto statistics = [&](int64_t row) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (row + r * step < p.rows) nmean[r] = p.mean[row + r * step], nrstd[r] = p.rstd[row + r * step];
  };
  statistics(first);
  int stage = 0;
  uint32_t phase = 0;
  for (int64_t row = first; row < p.rows; row += ROWS * step) {
    float mean[ROWS], rstd[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) mean[r] = nmean[r], rstd[r] = nrstd[r];
    const bool two = ROWS == 2 && row + step < p.rows;
    if (row + ROWS * step < p.rows) statistics(row + ROWS * step);
    RowVec<T, V> vx[ROWS][NV], vg[ROWS][NV];
    float2 h[V / 2], u[V / 2];
    float2 s[2][2] = {{both(0.f), both(0.f)}, {both(0.f), both(0.f)}};
    // x and dy stay packed between the sums and the result and are widened twice.
    auto widen = [&](int r, int g, int i, float2& d) {
      h[i] = mul2(add2(widen2<T, V>(vx[r][g], i), both(-mean[r])), both(rstd[r]));
      d = widen2<T, V>(vg[r][g], i);
      u[i] = mul2(d, ww[g][i]);
    };
    int st[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      st[r] = stage;
      if (r == 1 && !two) break;
      ring.wait(stage, phase);  // after a timeout (recorded) the rest runs through on stale data
      const T* sx = reinterpret_cast<const T*>(ring.base + stage * 2 * ring.bytes);
      const T* sg = reinterpret_cast<const T*>(ring.base + (stage * 2 + 1) * ring.bytes);
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        const int c = V * (t + G * g);
        if (c >= cols) continue;
        vx[r][g] = load_vec<T, V>(sx + c);
        vg[r][g] = load_vec<T, V>(sg + c);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          float2 d;
          widen(r, g, i, d);
          aw[g][i] = fma2(d, h[i], aw[g][i]);
          ab[g][i] = add2(d, ab[g][i]);
          s[r][0] = add2(s[r][0], u[i]);
          s[r][1] = fma2(u[i], h[i], s[r][1]);
        }
      }
      if (++stage == stages) stage = 0, phase ^= 1u;
    }
    float4 sum;
    if constexpr (ROWS == 1) {
      const float2 one = row_sum<WARP>(s[0][0].x + s[0][0].y, s[0][1].x + s[0][1].y, reinterpret_cast<float2(*)[32]>(buf), parity);
      sum = make_float4(one.x, one.y, 0.f, 0.f);
    } else sum = row_sum4<WARP>(make_float4(s[0][0].x + s[0][0].y, s[0][1].x + s[0][1].y, s[1][0].x + s[1][0].y,
                                                  s[1][1].x + s[1][1].y), buf, parity);  // also: the group has read the stages
    if (t == 0 && !*ring.abort) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const int64_t ahead = row + (stages + r) * step;
        if (ahead < p.rows) ring.fill(st[r], ahead), ++filled;
      }
    }
    if (p.dx) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r == 1 && !two) break;
        const float a0 = (r ? sum.z : sum.x) * inv, a1 = (r ? sum.w : sum.y) * inv;
        T* dx = static_cast<T*>(p.dx) + (row + r * step) * p.lddx;
#pragma unroll
        for (int g = 0; g < NV; ++g) {
          const int c = V * (t + G * g);
          if (c >= cols) continue;
          RowVec<T, V> out;
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            float2 d;
            widen(r, g, i, d);
            round2<T, V>(out, i, mul2(both(rstd[r]), fma2(h[i], both(-a1), add2(u[i], both(-a0)))));
          }
          store_vec<T, V>(dx + c, out);
        }
      }
    }
  }
  if (t == 0 && *ring.abort) ring.drain(filled);
  if (p.partial) {
    float* out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.cols;
    if constexpr (WARP) {
      // Add the warps' sums in warp order; every copy has landed and been read.
      __syncthreads();
      constexpr int COLS = 32 * V * NV;
      float* part = reinterpret_cast<float*>(ring_smem);
      float* mine = part + group * 2 * COLS;
#pragma unroll
      for (int g = 0; g < NV; ++g)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          mine[V * (t + 32 * g) + i] = i % 2 ? aw[g][i / 2].y : aw[g][i / 2].x;
          mine[COLS + V * (t + 32 * g) + i] = i % 2 ? ab[g][i / 2].y : ab[g][i / 2].x;
        }
      __syncthreads();
      for (int e = threadIdx.x; e < 2 * COLS; e += static_cast<int>(blockDim.x)) {
        const int c = e % COLS, which = e / COLS;
        if (c >= cols) continue;
        float s = 0.f;
        for (int i = 0; i < groups; ++i) s += part[i * 2 * COLS + e];
        out[which * p.cols + c] = s;
      }
    } else {
#pragma unroll
      for (int g = 0; g < NV; ++g) {
        const int c = V * (t + G * g);
        if (c >= cols) continue;
#pragma unroll
        for (int i = 0; i < V; i += 4) {  // cols is a multiple of V: 16-byte boundaries
          const float2 w0 = aw[g][i / 2], w1 = aw[g][i / 2 + 1], b0 = ab[g][i / 2], b1 = ab[g][i / 2 + 1];
          *reinterpret_cast<float4*>(out + c + i) = make_float4(w0.x, w0.y, w1.x, w1.y);
          *reinterpret_cast<float4*>(out + p.cols + c + i) = make_float4(b0.x, b0.y, b1.x, b1.y);
        }
      }
    }
  }
  grid_launch_dependents();
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

// Adds the CTAs' partial sums: 32 columns of one of the two sums per CTA,
// every eighth partial per warp, then the eight warps' sums in order; one
// rounding.
template <typename W>
__global__ void __launch_bounds__(256) layer_norm_dw_finish(const NormParams p) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t strips = (p.cols + 31) / 32;
  const bool second = blockIdx.x >= strips;
  const int64_t c = (blockIdx.x - (second ? strips : 0)) * 32 + lane;
  void* out = second ? p.db : p.dw;
  if (!out) return;
  grid_dependency_wait();
  float s = 0.f;
  if (c < p.cols) {
    const float* in = p.partial + (second ? p.cols : 0) + c;
#pragma unroll 8
    for (int i = warp; i < p.splits; i += 8) s += in[static_cast<int64_t>(i) * 2 * p.cols];
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < p.cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][lane];
    static_cast<W*>(out)[c] = from_acc<W>(s);
  }
}

// How a call runs: rows in registers (a warp or a CTA per row, 16-byte groups
// or single elements), or the kernels for any size.
struct NormPlan {
  bool rows, warp;
  bool vec;
  int stages;   // of the ring; 0: no ring
  int nv;       // groups per thread
  int threads;  // per CTA
  int64_t ctas;
  int partials;  // backward: partial sums per column
};

bool norm_aligned(const void* p, int64_t ld, size_t es) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && static_cast<size_t>(ld) * es % 16 == 0;
}

NormPlan norm_forward_plan(const cuopx_layer_norm_args& a) {
  NormPlan q = {};
  const size_t es = dtype_size(a.dtype);
  const int v = static_cast<int>(16 / es);
  const int64_t sms = device_sm_count();
  q.vec = a.cols % v == 0 && norm_aligned(a.X, a.ldx, es) && norm_aligned(a.Y, a.ldy, es);
  const int per = q.vec ? v : 1;
  // Unaligned 16-bit rows of up to 1024 columns still go to a warp each (8192 x
  // 1001 bf16: 30.3 -> 25.0 us); fp32 ones are faster with a CTA per row from 512.
  const int alone = es == 2 ? 32 : 16;  // single elements per lane
  const int64_t warp_max = 32ll * (q.vec ? 4 * v : alone);
  if (a.cols <= warp_max && a.rows > sms) {
    q.rows = q.warp = true;
    q.nv = q.vec ? 4 : alone;
    q.threads = 256;
    q.ctas = std::min<int64_t>((a.rows + 7) / 8, int64_t(1) << 30);
    return q;
  }
  // Few rows: as many threads per row as there are groups, for the shortest
  // chain of loads; many rows: several groups per thread, several rows per SM.
  const int small = q.vec ? 1 : 4, large = q.vec ? 4 : 16;
  q.nv = a.rows <= 2 * sms && a.cols <= 1024ll * per * small ? small : large;
  const int64_t t = (a.cols + static_cast<int64_t>(per) * q.nv - 1) / (static_cast<int64_t>(per) * q.nv);
  q.threads = static_cast<int>((t + 31) / 32 * 32);
  q.rows = q.threads <= (q.nv == 16 ? 512 : 1024);
  q.ctas = std::min<int64_t>(a.rows, int64_t(1) << 30);
  return q;
}

NormPlan norm_backward_plan(const cuopx_layer_norm_args& a) {
  NormPlan q = {};
  const size_t es = dtype_size(a.dtype);
  const int v = static_cast<int>(16 / es);
  const int64_t sms = device_sm_count();
  q.vec = a.cols % v == 0 && norm_aligned(a.X, a.ldx, es) && norm_aligned(a.dY, a.lddy, es) &&
          (!a.dX || norm_aligned(a.dX, a.lddx, es));
  const int per = q.vec ? v : 1;
  const int64_t row_bytes = 2 * a.cols * static_cast<int64_t>(es);  // of x and dy
  const int64_t warp_max = 32ll * (q.vec ? 4 * v : 16);
  if (a.cols <= warp_max) {
    q.rows = q.warp = true;
    q.nv = q.vec ? (a.cols <= 32 * v ? 1 : 4) : 16;
    q.threads = 256;
    const int per_sm = q.nv == 4 ? 1 : 2;
    q.ctas = std::min<int64_t>((a.rows + 7) / 8, sms * per_sm);
    if (q.vec) q.stages = static_cast<int>(std::min<int64_t>(8, 200 * 1024 / per_sm / (8 * row_bytes)));
  } else {
    q.nv = !q.vec ? 16 : a.cols <= 1024 * v ? 1 : 4;
    const int64_t t = (a.cols + static_cast<int64_t>(per) * q.nv - 1) / (static_cast<int64_t>(per) * q.nv);
    q.threads = static_cast<int>(std::min<int64_t>(2048, (t + 31) / 32 * 32));
    q.rows = q.threads <= (q.nv == 1 ? 1024 : 512);
    const int per_sm = std::max(1, (q.nv == 1 ? 1024 : 512) / q.threads);
    // Two rows per CTA at least, four from 200 rows on: every CTA leaves a
    // partial sum per column for the second launch to read (300 x 4096 bf16:
    // 11.1 us with one row per CTA, 8.2 with four).
    const int64_t least = !a.dweight && !a.dbias ? 1 : a.rows < 200 ? 2 : 4;
    q.ctas = std::min<int64_t>((a.rows + least - 1) / least, sms * per_sm);
    if (q.vec) {
      q.stages = static_cast<int>(std::min<int64_t>(8, 200 * 1024 / per_sm / row_bytes));
      if (q.stages < 2) q.rows = false;
    }
  }
  if (!q.rows) {
    // Shares of the rows for the column sums of the any-size kernel.
    const int64_t strips = (a.cols + 31) / 32;
    q.partials = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(sms * 8 + strips - 1) / strips, (a.rows + 31) / 32, 256})));
  } else {
    q.partials = static_cast<int>(q.ctas);
  }
  return q;
}

size_t norm_backward_workspace(const cuopx_layer_norm_args& a) {
  if (a.rows <= 0 || a.cols <= 0 || (!a.dweight && !a.dbias) || dtype_size(a.dtype) == 0) return 0;
  return static_cast<size_t>(norm_backward_plan(a).partials) * 2 * static_cast<size_t>(a.cols) * sizeof(float);
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
  p.vec_w = reinterpret_cast<uintptr_t>(a.weight) % 16 == 0;
  p.vec_b = reinterpret_cast<uintptr_t>(a.bias) % 16 == 0;
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
  if (!extent_ok(a->rows, a->ldx) || !extent_ok(a->rows, a->ldy)) return CUOPX_INVALID_ARGUMENT;
  if (!starts_on(es, a->X, a->Y) || !starts_on(ws, a->weight, a->bias) || !starts_on(4, a->mean, a->rstd))
    return CUOPX_INVALID_ARGUMENT;
  const size_t wb = static_cast<size_t>(a->cols) * ws, sb = static_cast<size_t>(a->rows) * sizeof(float);
  if (!alias_ok(a->Y, a->ldy, a->X, a->ldx, a->rows, a->cols, es)) return CUOPX_INVALID_ARGUMENT;
  const Extent x{a->X, a->rows, a->cols, a->ldx, es};
  const Extent weight = vector_extent(a->weight, wb), bias = vector_extent(a->bias, wb);
  const Extent outs[3] = {{a->Y, a->rows, a->cols, a->ldy, es}, vector_extent(a->mean, sb), vector_extent(a->rstd, sb)};
  for (int i = 0; i < 3; ++i) {
    if (overlaps(outs[i], weight) || overlaps(outs[i], bias)) return CUOPX_INVALID_ARGUMENT;
    if (i > 0 && overlaps(outs[i], x)) return CUOPX_INVALID_ARGUMENT;
    for (int j = 0; j < i; ++j)
      if (overlaps(outs[i], outs[j])) return CUOPX_INVALID_ARGUMENT;
  }
  const NormParams p = norm_params(*a);
  const NormPlan q = norm_forward_plan(*a);
  if (q.rows) {
    cudaError_t e = cudaSuccess;
    with_norm_types(*a, [&](auto t, auto w) {
      using T = decltype(t);
      using W = decltype(w);
      constexpr int V = 16 / static_cast<int>(sizeof(T));
      auto go = [&](auto kern) {
        e = launch_pdl(kern, dim3(static_cast<unsigned>(q.ctas)), dim3(static_cast<unsigned>(q.threads)), 0, stream, p);
      };
      constexpr bool kHalf = sizeof(T) == 2;
      if (q.warp && q.vec) go(layer_norm_rows<T, W, V, 4, true, 256, 4>);
      else if (q.warp) go(layer_norm_rows<T, W, 1, kHalf ? 32 : 16, true, 256, kHalf ? 2 : 3>);
      else if (q.vec) q.nv == 1 ? go(layer_norm_rows<T, W, V, 1, false, 1024, 1>) : go(layer_norm_rows<T, W, V, 4, false, 1024, 1>);
      else q.nv == 4 ? go(layer_norm_rows<T, W, 1, 4, false, 1024, 1>) : go(layer_norm_rows<T, W, 1, 16, false, 512, 2>);
    });
    if (e != cudaSuccess) {
      cudaGetLastError();
      return cuda_failure(e);
    }
    note_launch("layer_norm_rows");
    return check_launch();
  }
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
    if (!extent_ok(a->rows, a->ldx) || !extent_ok(a->rows, a->lddy) || (a->dX && !extent_ok(a->rows, a->lddx)))
      return CUOPX_INVALID_ARGUMENT;
  }
  if (!starts_on(es, a->X, a->dY, a->dX) || !starts_on(ws, a->weight, a->dweight, a->dbias) ||
      !starts_on(4, a->mean, a->rstd) || !starts_on(256, a->workspace))
    return CUOPX_INVALID_ARGUMENT;
  const size_t need = norm_backward_workspace(*a);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need)) return CUOPX_RESOURCE_UNAVAILABLE;
  const Extent ins[4] = {{a->X, a->rows, a->cols, a->ldx, es}, vector_extent(a->weight, wb), vector_extent(a->mean, sb),
                         vector_extent(a->rstd, sb)};
  const Extent grad{a->dY, a->rows, a->cols, a->lddy, es};
  const Extent outs[4] = {{a->dX, a->rows, a->cols, a->lddx, es}, vector_extent(a->dweight, wb), vector_extent(a->dbias, wb),
                          vector_extent(need ? a->workspace : nullptr, need)};
  for (int i = 0; i < 4; ++i) {
    for (const Extent& in : ins)
      if (overlaps(outs[i], in)) return CUOPX_INVALID_ARGUMENT;
    if (i == 0 ? a->dX && !alias_ok(a->dX, a->lddx, a->dY, a->lddy, a->rows, a->cols, es) : overlaps(outs[i], grad))
      return CUOPX_INVALID_ARGUMENT;
    for (int j = 0; j < i; ++j)
      if (overlaps(outs[i], outs[j])) return CUOPX_INVALID_ARGUMENT;
  }
  NormParams p = norm_params(*a);
  if (a->rows == 0) {  // sums over no rows
    if (a->dweight && cudaMemsetAsync(a->dweight, 0, wb, stream) != cudaSuccess) return cuda_failure(cudaGetLastError());
    if (a->dbias && cudaMemsetAsync(a->dbias, 0, wb, stream) != cudaSuccess) return cuda_failure(cudaGetLastError());
    return CUOPX_SUCCESS;
  }
  const NormPlan q = norm_backward_plan(*a);
  const bool sums = p.dw || p.db;
  p.splits = q.partials;
  if (sums) p.partial = static_cast<float*>(a->workspace);
  cudaError_t e = cudaSuccess;
  with_norm_types(*a, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    constexpr int NV = sizeof(T) == 4 ? 4 : 2;
    if (q.rows && q.vec) {
      auto go = [&](auto kern, int cols) {
        size_t smem = static_cast<size_t>(q.stages) * 2 * static_cast<size_t>(p.cols) * sizeof(T);
        if (q.warp) smem = std::max(smem * 8, static_cast<size_t>(8 * 2 * cols) * sizeof(float));
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 211 * 1024);
        if (e == cudaSuccess)
          e = launch_pdl(kern, dim3(static_cast<unsigned>(q.ctas)), dim3(static_cast<unsigned>(q.threads)), smem, stream, p,
                         q.stages);
        note_launch("layer_norm_backward_ring");
      };
      constexpr int ROWS = sizeof(T) == 2 ? 2 : 1;
      if (q.warp && q.nv == 1) go(layer_norm_backward_ring<T, W, V, 1, true, 256, 2, 2>, 32 * V);
      else if (q.warp) go(layer_norm_backward_ring<T, W, V, 4, true, 256, 1, 2>, 32 * V * 4);
      else if (q.nv == 1) go(layer_norm_backward_ring<T, W, V, 1, false, 1024, 1, ROWS>, 0);
      else go(layer_norm_backward_ring<T, W, V, 4, false, 512, 1, 1>, 0);
    } else if (q.rows) {
      const size_t smem = q.warp ? static_cast<size_t>(q.threads / 32) * 2 * 32 * 16 * sizeof(float) : 0;
      e = launch_pdl(q.warp ? layer_norm_backward_rows<T, W, 16, true, 256> : layer_norm_backward_rows<T, W, 16, false, 512>,
                     dim3(static_cast<unsigned>(q.ctas)), dim3(static_cast<unsigned>(q.threads)), smem, stream, p);
      note_launch("layer_norm_backward_rows");
    } else {
      if (sums) {  // before dX, which may overwrite dY
        layer_norm_dw_any<T><<<dim3(static_cast<unsigned>((p.cols + 31) / 32), static_cast<unsigned>(q.partials)), 256, 0, stream>>>(p);
        note_launch("layer_norm_dw_any");
      }
      if (p.dx) {
        layer_norm_dx_any<T, W><<<norm_row_ctas(p.rows), 256, 0, stream>>>(p);
        note_launch("layer_norm_dx_any");
      }
    }
    if (e == cudaSuccess && sums) {
      const unsigned strips = static_cast<unsigned>((p.cols + 31) / 32);
      e = launch_pdl(layer_norm_dw_finish<W>, dim3(2 * strips), dim3(256), 0, stream, p);
      note_launch("layer_norm_dw_finish");
    }
  });
  if (e != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(e);
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
