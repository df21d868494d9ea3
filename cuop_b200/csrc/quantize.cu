// Symmetric int8 quantisation with one scale for each row (activations: for
// each token) or for each column of a transposed result (weights stored
// [K][columns]):
//   a = max |x| (at least 2^-100),  scale = a / 127,  q = rint(x * (127 / a)).
// The three fp32 operations are IEEE's, so a result can be reproduced bit by
// bit; |x * (127 / a)| is at most 127 (1 + 2^-23), so nothing is clamped.  The
// lower limit on a keeps 127 / a and the scale in fp32's normal range, for
// rows of zeros too.
#include "common.cuh"
#include "dispatch.h"

namespace cuopx {

namespace {

constexpr float kQuantMin = 0x1p-100f;

// Magnitudes are compared as integers: a NaN's bits are above infinity's, and
// infinity's above every number's, so one maximum finds all three.
template <typename T>
struct Magnitude;
template <>
struct Magnitude<float> {
  static constexpr int V = 4;  // elements of 16 bytes
  static __device__ __forceinline__ uint32_t word(uint32_t m, uint32_t w) { return max(m, w & 0x7fffffffu); }
  static __device__ __forceinline__ uint32_t one(float v) { return __float_as_uint(v) & 0x7fffffffu; }
  static __device__ __forceinline__ uint32_t fold(uint32_t m) { return m; }
  static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m); }
};
template <typename T>
struct Magnitude {  // 16 bits, two to a word
  static constexpr int V = 8;
  static __device__ __forceinline__ uint32_t word(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }
  static __device__ __forceinline__ uint32_t one(T v) { return *reinterpret_cast<unsigned short*>(&v) & 0x7fffu; }
  static __device__ __forceinline__ uint32_t fold(uint32_t m) { return max(m & 0xffffu, m >> 16); }
  static __device__ __forceinline__ float value(uint32_t m) {
    const unsigned short b = static_cast<unsigned short>(m);
    return to_acc<T>(*reinterpret_cast<const T*>(&b));
  }
};

// 127 / a and the scale; `keep` is 0 where a is not finite.
struct RowScale {
  float r, scale;
  uint32_t keep;
};
__device__ __forceinline__ RowScale row_scale(float a) {
  a = a < kQuantMin ? kQuantMin : a;  // NaN stays
  return {__fdiv_rn(127.f, a), __fdiv_rn(a, 127.f), a < __int_as_float(0x7f800000) ? ~0u : 0u};
}

// Adding 1.5 * 2^23 leaves rint(v) in the low bits of the sum (|v| < 2^22), which
// saves the conversion to integer, at a quarter of the rate.  The product is
// rounded before: in packed form (f32x2) the two operations came out fused, and ties
// such as x = a / 2 (63.5) fell the wrong way.
__device__ __forceinline__ uint32_t quantized(float v, const RowScale& s) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, s.r), 12582912.f));
}
__device__ __forceinline__ uint32_t quantize4(float2 a, float2 b, const RowScale& s) {
  const uint32_t lo = __byte_perm(quantized(a.x, s), quantized(a.y, s), 0x0040);
  const uint32_t hi = __byte_perm(quantized(b.x, s), quantized(b.y, s), 0x0040);
  return __byte_perm(lo, hi, 0x5410) & s.keep;
}
__device__ __forceinline__ int8_t quantize1(float a, const RowScale& s) { return static_cast<int8_t>(quantized(a, s) & s.keep); }

template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

struct QuantParams {
  int64_t rows, cols;
  const void* X;
  int64_t ldx;
  int8_t* Q;
  int64_t ldq;
  float* scale;
};

// The row's largest magnitude from every thread's; `tpr` threads (whole warps)
// to a row, `part` one word per warp of the CTA.
__device__ __forceinline__ uint32_t row_max(uint32_t m, int tpr, uint32_t* part) {
  m = __reduce_max_sync(0xffffffffu, m);
  if (tpr == 32) return m;
  // Two of these arrays in turn: a barrier lies between a warp's last reads of one and the next writes.
  const int warp = threadIdx.x >> 5, first = warp - warp % (tpr >> 5);
  if ((threadIdx.x & 31) == 0) part[warp] = m;
  __syncthreads();
  for (int w = 0; w < tpr >> 5; ++w) m = max(m, part[first + w]);
  return m;
}

// Rows on 16-byte boundaries (Q's on 8, or 4 for fp32): `tpr` threads hold a row in G
// groups of 16 bytes each, so that X is read once, and a CTA loads its next rows
// before it works on the present ones.  HBM-bound: 8192 x 8192 bf16 36.9 us, 5.5 TB/s (without
// rows ahead 40.4).
template <typename T, int G>
__device__ __forceinline__ void load_row(const QuantParams& p, int64_t row, int t, int tpr, uint4 (&v)[G]) {
  constexpr int V = Magnitude<T>::V;
  const T* x = static_cast<const T*>(p.X) + row * p.ldx;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int64_t c = (g * static_cast<int64_t>(tpr) + t) * V;
    v[g] = make_uint4(0, 0, 0, 0);
    if (row < p.rows && c < p.cols) {
      if (c + V <= p.cols) {
        v[g] = __ldcs(reinterpret_cast<const uint4*>(x + c));
      } else {
        alignas(16) T some[V] = {};
        for (int i = 0; i < V; ++i)
          if (c + i < p.cols) some[i] = x[c + i];
        v[g] = *reinterpret_cast<const uint4*>(some);
      }
    }
  }
}

template <typename T, int G>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const QuantParams p, int tpr) {
  using Mag = Magnitude<T>;
  constexpr int V = Mag::V;
  __shared__ uint32_t part[2][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int t = threadIdx.x % tpr, each = blockDim.x / tpr;
  const int64_t step = static_cast<int64_t>(gridDim.x) * each;
  int64_t row = blockIdx.x * static_cast<int64_t>(each) + threadIdx.x / tpr;
  const int64_t first = blockIdx.x * static_cast<int64_t>(each);
  uint4 next[G];
  load_row<T, G>(p, row, t, tpr, next);
  int turn = 0;
  for (int64_t at = first; at < p.rows; at += step, row += step, turn ^= 1) {
    uint4 v[G];
    uint32_t m = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) v[g] = next[g];
    if (at + step < p.rows) load_row<T, G>(p, row + step, t, tpr, next);
#pragma unroll
    for (int g = 0; g < G; ++g) m = Mag::word(Mag::word(Mag::word(Mag::word(m, v[g].x), v[g].y), v[g].z), v[g].w);
    m = row_max(Mag::fold(m), tpr, part[turn]);
    if (row >= p.rows) continue;
    const RowScale s = row_scale(Mag::value(m));
    if (t == 0) p.scale[row] = s.scale;
    int8_t* q = p.Q + row * p.ldq;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int64_t c = (g * static_cast<int64_t>(tpr) + t) * V;
      if (c >= p.cols) break;
      uint32_t w[V / 4];
      if constexpr (V == 8) {
        w[0] = quantize4(pair_of<T>(v[g].x), pair_of<T>(v[g].y), s);
        w[V / 4 - 1] = quantize4(pair_of<T>(v[g].z), pair_of<T>(v[g].w), s);
      } else {
        w[0] = quantize4(make_float2(__uint_as_float(v[g].x), __uint_as_float(v[g].y)),
                         make_float2(__uint_as_float(v[g].z), __uint_as_float(v[g].w)), s);
      }
      if (c + V <= p.cols) {
        if constexpr (V == 8) *reinterpret_cast<uint2*>(q + c) = make_uint2(w[0], w[V / 4 - 1]);
        else *reinterpret_cast<uint32_t*>(q + c) = w[0];
      } else {
        for (int i = 0; i < V; ++i)
          if (c + i < p.cols) q[c + i] = static_cast<int8_t>(w[i / 4] >> (8 * (i % 4)));
      }
    }
  }
}

// Any alignment and any length: a CTA to a row, elements, the row read twice (the second time from
// L2).  8192 x 8192 bf16 off 16-byte boundaries 65 us (aligned 37), 1024 x 40000 100 us.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const QuantParams p) {
  using Mag = Magnitude<T>;
  __shared__ uint32_t part[32];
  grid_dependency_wait();
  grid_launch_dependents();
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.X) + row * p.ldx;
    uint32_t m = 0;
#pragma unroll 8
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) m = max(m, Mag::one(x[c]));
    m = row_max(m, 256, part);
    const RowScale s = row_scale(Mag::value(m));
    if (threadIdx.x == 0) p.scale[row] = s.scale;
    int8_t* q = p.Q + row * p.ldq;
#pragma unroll 8
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) q[c] = quantize1(to_acc<T>(x[c]), s);
    __syncthreads();  // `part` is free
  }
}

// Columns, with Q transposed: a cluster holds a strip of X of 128 bytes' width in the shared
// memory of its CTAs, a share of the rows each, so that X is read once.  The
// strip's column maxima meet through distributed shared memory; every CTA then quantises its
// rows in place, four of a column to a word, and writes them out along Q's rows.
// A CTA's four phases, which other CTAs of the SM overlap only in part, bound it: 4096 x 10240 bf16
// 47 us, rows off 4-byte boundaries as in 4095 x 10001 fp16 (WORD false: single elements) 57;
// two passes over X took 141.  Half the threads: 52 and 73.  Loads by 4-byte cp.async, all of
// a share at once: 76 and 89.
constexpr int QC_PITCH = 33;  // words of a row in shared memory
constexpr int QC_MAX_SHARE = 1536;

template <typename T, bool WORD>
__global__ void __maxnreg__(WORD ? 64 : 40) quantize_columns_kernel(const QuantParams p, int cs, int share) {
  using Mag = Magnitude<T>;
  constexpr int PER = 4 / sizeof(T);  // columns to a word
  extern __shared__ uint32_t qc_rows[];
  __shared__ uint32_t part[32][32], top[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rank = static_cast<int>(blockIdx.x) % cs;
  const int64_t c0 = static_cast<int64_t>(blockIdx.x / cs) * (32 * PER), c = c0 + lane * PER, r0 = static_cast<int64_t>(rank) * share;
  const int64_t left = p.rows - r0;
  const int rows = left <= 0 ? 0 : left < share ? static_cast<int>(left) : share;
  grid_dependency_wait();
  uint32_t m = 0;
  if (rows > 0) {
    // Sixteen loads of a warp on their way at once, from rows next to the other warps'.  Lanes
    // beyond the last column read one that exists; it does not reach Q.
    const T* x = static_cast<const T*>(p.X) + r0 * p.ldx;
    const int64_t last = p.cols - 1;
    uint32_t* dst = qc_rows + warp * QC_PITCH + lane;
    // A row's word, or its two halves, `step` elements from one of the warp's rows to the next.
    // Registers decide the order of the loads and how many CTAs share an SM: whole groups
    // apart from the last one and 64 registers are best for words (40: 52 us instead of 47), one
    // form and 40 for elements (with whole groups apart 79 instead of 55).
    auto read = [&](const auto* at, int64_t step, int second) {
      constexpr int AHEAD = WORD ? 16 : 8;
      auto group = [&](auto whole, int n) {
        uint32_t lo[AHEAD], hi[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const auto* row = at + (decltype(whole)::value ? i : min(i, n - 1)) * step;
          lo[i] = __ldcs(row);
          if constexpr (!WORD) hi[i] = __ldcs(row + second);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const uint32_t w = WORD ? lo[i] : __byte_perm(lo[i], hi[i], 0x5410);
          m = Mag::word(m, w);
          if (decltype(whole)::value || i < n) dst[i * warps * QC_PITCH] = w;
        }
        at += AHEAD * step;
        dst += AHEAD * warps * QC_PITCH;
      };
      int n = (rows - warp + warps - 1) / warps;  // this warp's rows
      if constexpr (WORD)
        for (; n >= AHEAD; n -= AHEAD) group(std::true_type{}, n);
      for (; n > 0; n -= AHEAD) group(std::false_type{}, n);
    };
    if constexpr (WORD)
      read(reinterpret_cast<const uint32_t*>(x + warp * p.ldx + (c < p.cols ? c : 0)), warps * p.ldx / PER, 0);
    else
      read(reinterpret_cast<const unsigned short*>(x + warp * p.ldx) + min(c, last), warps * p.ldx, c < last ? 1 : 0);
  }
  part[warp][lane] = m;
  __syncthreads();
  if (warp == 0) {
    for (int i = 1; i < warps; ++i) m = Mag::word(m, part[i][lane]);
    top[lane] = m;
  }
  if (cs > 1) {
    cluster_sync_all();  // every CTA's maxima are in place
    if (warp == 0) {
      m = 0;
      for (int i = 0; i < cs; ++i) {
        uint32_t w;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(map_to_rank(&top[lane], static_cast<uint32_t>(i))) : "memory");
        m = Mag::word(m, w);
      }
      part[0][lane] = m;
    }
    __syncthreads();
    m = part[0][lane];
    // Has read the others': the release of the warp that did keeps its reads before the arrival, after which
    // another CTA may leave, one without rows at once.  (Every warp reading, and releasing here: 4096 x
    // 10240 12 us more; releasing behind the next phase: 7.)
    if (warp == 0) cluster_arrive();
    else cluster_arrive_relaxed();
  } else {
    __syncthreads();
    m = top[lane];
  }
  RowScale s[PER];
  if constexpr (PER == 2) {
    s[0] = row_scale(Mag::value(m & 0xffffu));
    s[PER - 1] = row_scale(Mag::value(m >> 16));
  } else {
    s[0] = row_scale(Mag::value(m));
  }
  if (rank == 0 && warp == 0) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (c + k < p.cols) p.scale[c + k] = s[k].scale;
  }
  // Four rows of a lane's columns to a word for each column, in the rows' own places: group g's
  // words lie in its row (g / 8 + column) % 4, so that 32 groups of a column lie in 32 banks.
  for (int r = 4 * warp; r < rows; r += 4 * warps) {
    uint32_t w[4];
    uint32_t* at = qc_rows + r * QC_PITCH + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = at[i * QC_PITCH];
    if constexpr (PER == 2) {
      float2 f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = pair_of<T>(w[i]);
      at[(r >> 5 & 3) * QC_PITCH] = quantize4(make_float2(f[0].x, f[1].x), make_float2(f[2].x, f[3].x), s[0]);
      at[((r >> 5) + 1 & 3) * QC_PITCH] = quantize4(make_float2(f[0].y, f[1].y), make_float2(f[2].y, f[3].y), s[PER - 1]);
    } else {
      at[(r >> 5 & 3) * QC_PITCH] = quantize4(make_float2(__uint_as_float(w[0]), __uint_as_float(w[1])),
                                              make_float2(__uint_as_float(w[2]), __uint_as_float(w[3])), s[0]);
    }
  }
  __syncthreads();
  // Q's rows in whole words wherever they start; what lies before the first and behind the last in bytes.
  for (int k = warp; k < 32 * PER; k += warps) {
    if (c0 + k >= p.cols) break;
    int8_t* q = p.Q + (c0 + k) * p.ldq + r0;
    auto group = [&](int g) { return qc_rows[(4 * g + ((g >> 3) + k % PER & 3)) * QC_PITCH + k / PER]; };
    const int head = min(rows, static_cast<int>(-reinterpret_cast<uintptr_t>(q) & 3)), n = (rows - head) >> 2;
    for (int g = lane; g < n; g += 32) {
      uint32_t w = group(g);
      if (head > 0) w = __funnelshift_r(w, group(g + 1), 8 * head);
      *reinterpret_cast<uint32_t*>(q + head + 4 * g) = w;
    }
    if (lane < rows - 4 * n) {
      const int e = lane < head ? lane : lane + 4 * n;
      q[e] = static_cast<int8_t>(group(e >> 2) >> (8 * (e & 3)));
    }
  }
  if (cs > 1) cluster_wait();  // the others have read this CTA's maxima
}

// More rows than a cluster holds: maxima first, then a second pass, single elements in both: 28672 x 8192
// bf16 650 us, 109 being its floor.
// Largest magnitudes of columns, as bits, in `top` (zeroed before): a thread
// to a column, 8 row phases and a share of the rows to a CTA.
template <typename T>
__global__ void __launch_bounds__(256) quantize_column_max_kernel(const QuantParams p, uint32_t* top, int64_t share) {
  using Mag = Magnitude<T>;
  __shared__ uint32_t part[8][32];
  const int lane = threadIdx.x & 31, phase = threadIdx.x >> 5;
  const int64_t c = blockIdx.x * 32ll + lane;
  const int64_t r0 = blockIdx.y * share, r1 = min(p.rows, r0 + share);
  uint32_t m = 0;
  if (c < p.cols) {
    const T* x = static_cast<const T*>(p.X) + c;
#pragma unroll 8
    for (int64_t r = r0 + phase; r < r1; r += 8) m = max(m, Mag::one(x[r * p.ldx]));
  }
  part[phase][lane] = m;
  __syncthreads();
  if (phase == 0 && c < p.cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, part[i][lane]);
    atomicMax(top + c, m);
  }
}

// 128 rows x 32 columns of X to 32 rows of Q.
template <typename T>
__global__ void __launch_bounds__(256) quantize_transpose_kernel(const QuantParams p, const uint32_t* top) {
  using Mag = Magnitude<T>;
  __shared__ int8_t tile[32][128 + 4];
  const int lane = threadIdx.x & 31, phase = threadIdx.x >> 5;
  const int64_t c0 = blockIdx.x * 32ll, r0 = blockIdx.y * 128ll, c = c0 + lane;
  if (c < p.cols) {
    const RowScale s = row_scale(Mag::value(top[c]));
    if (blockIdx.y == 0 && phase == 0) p.scale[c] = s.scale;
    const T* x = static_cast<const T*>(p.X) + c;
#pragma unroll 8
    for (int r = phase; r < 128; r += 8)
      if (r0 + r < p.rows) tile[lane][r] = quantize1(to_acc<T>(x[(r0 + r) * p.ldx]), s);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 32 * 128; e += 256) {
    const int r = e & 127, k = e >> 7;
    if (c0 + k < p.cols && r0 + r < p.rows) p.Q[(c0 + k) * p.ldq + r0 + r] = tile[k][r];
  }
}

template <typename T, int G>
cudaError_t launch_quantize_rows(const QuantParams& p, int tpr, cudaStream_t stream) {
  const int rows = std::max(1, 256 / tpr);
  const int64_t resident = static_cast<int64_t>(device_sm_count()) * (1024 / std::max(256, tpr));
  return launch_pdl(quantize_rows_kernel<T, G>, dim3(static_cast<unsigned>(std::min((p.rows + rows - 1) / rows, resident))),
                    dim3(static_cast<unsigned>(rows * tpr)), 0, stream, p, tpr);
}

template <typename T>
int quantize_rows_typed(const QuantParams& p, cudaStream_t stream) {
  constexpr int V = Magnitude<T>::V;
  cudaError_t err;
  const bool aligned = reinterpret_cast<uintptr_t>(p.X) % 16 == 0 && (p.rows == 1 || p.ldx % V == 0) &&
                       reinterpret_cast<uintptr_t>(p.Q) % V == 0 && (p.rows == 1 || p.ldq % V == 0);
  const int64_t groups = (p.cols + V - 1) / V;
  if (aligned && groups <= 4096) {
    // Four groups a thread, whole warps, a power of two of them.
    int tpr = 32;
    while (tpr * 4 < groups) tpr *= 2;
    err = launch_quantize_rows<T, 4>(p, tpr, stream);
    note_launch("quantize_rows");
  } else {
    err = launch_pdl(quantize_rows_any_kernel<T>, dim3(static_cast<unsigned>(std::min<int64_t>(p.rows, 1 << 30))), dim3(256), 0,
                     stream, p);
    note_launch("quantize_rows_any");
  }
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  return check_launch();
}

// CTAs of a cluster and their shares of the rows: 256 rows or more each, up to eight CTAs.
int quantize_cluster(int64_t rows, int64_t& share) {
  int cs = 1;
  while (cs < 8 && rows > 256ll * cs) cs *= 2;
  share = ((rows + cs - 1) / cs + 31) / 32 * 32;
  return cs;
}

template <typename T>
int quantize_columns_typed(const QuantParams& p, uint32_t* top, cudaStream_t stream) {
  int64_t share = 0;
  const int cs = quantize_cluster(p.rows, share);
  if (share <= QC_MAX_SHARE) {
    constexpr int PER = 4 / sizeof(T);
    const bool words = sizeof(T) == 4 || (reinterpret_cast<uintptr_t>(p.X) % 4 == 0 && (p.rows == 1 || p.ldx % PER == 0) && p.cols % PER == 0);
    auto kern = quantize_columns_kernel<T, true>;
    if constexpr (PER == 2)
      if (!words) kern = quantize_columns_kernel<T, false>;
    static std::atomic<bool> attr_set[64][2] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return CUOPX_CUDA_ERROR;
    if (!attr_set[dev][words].load(std::memory_order_relaxed)) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, QC_MAX_SHARE * QC_PITCH * 4) != cudaSuccess)
        return CUOPX_CUDA_ERROR;
      attr_set[dev][words].store(true, std::memory_order_relaxed);
    }
    const int64_t strips = (p.cols + 32 * PER - 1) / (32 * PER);
    const unsigned threads = share <= 640 ? 512 : 1024;
    const cudaError_t err =
        launch_pdl_cluster(kern, dim3(static_cast<unsigned>(strips * cs)), dim3(threads), static_cast<size_t>(share) * QC_PITCH * 4,
                           stream, static_cast<unsigned>(cs), p, cs, static_cast<int>(share));
    if (err != cudaSuccess) {
      cudaGetLastError();
      return cuda_failure(err);
    }
    note_launch("quantize_columns");
    return check_launch();
  }
  if (const cudaError_t e = cudaMemsetAsync(top, 0, static_cast<size_t>(p.cols) * 4, stream); e != cudaSuccess)
    return cuda_failure(e);
  const int64_t strips = (p.cols + 31) / 32;
  const int64_t want = std::max<int64_t>(1, device_sm_count() * 16 / strips);
  share = std::max<int64_t>(64, (p.rows + want - 1) / want);
  quantize_column_max_kernel<T><<<dim3(static_cast<unsigned>(strips), static_cast<unsigned>((p.rows + share - 1) / share)), 256, 0,
                                  stream>>>(p, top, share);
  note_launch("quantize_column_max");
  quantize_transpose_kernel<T><<<dim3(static_cast<unsigned>(strips), static_cast<unsigned>((p.rows + 127) / 128)), 256, 0, stream>>>(
      p, top);
  note_launch("quantize_transpose");
  return check_launch();
}

int quantize_rows(int dtype, const QuantParams& p, cudaStream_t stream) {
  switch (dtype) {
    case CUOPX_F32: return quantize_rows_typed<float>(p, stream);
    case CUOPX_F16: return quantize_rows_typed<__half>(p, stream);
    default: return quantize_rows_typed<__nv_bfloat16>(p, stream);
  }
}

size_t quantize_workspace(const cuopx_quantize_args& a) {
  int64_t share = 0;
  if (!a.trans || a.rows <= 0 || a.cols <= 0) return 0;
  quantize_cluster(a.rows, share);
  return share > QC_MAX_SHARE ? static_cast<size_t>(a.cols) * 4 : 0;
}

int validate_quantize(const cuopx_quantize_args& a) {
  if (a.dtype != CUOPX_F32 && a.dtype != CUOPX_F16 && a.dtype != CUOPX_BF16) return CUOPX_UNSUPPORTED_TYPE;
  if (a.trans != 0 && a.trans != 1) return CUOPX_INVALID_ARGUMENT;
  if (a.rows < 0 || a.cols < 0) return CUOPX_INVALID_ARGUMENT;
  const int64_t q_rows = a.trans ? a.cols : a.rows, q_cols = a.trans ? a.rows : a.cols;
  if (q_rows == 0) return CUOPX_SUCCESS;
  const size_t es = dtype_size(a.dtype);
  if (!a.scale || !starts_on(4, a.scale) || !starts_on(es, a.X) || !starts_on(256, a.workspace)) return CUOPX_INVALID_ARGUMENT;
  if (q_cols > 0 && (!a.X || !a.Q || a.ldx < a.cols || a.ldq < q_cols)) return CUOPX_INVALID_ARGUMENT;
  if (q_cols > 0 && (!extent_ok(a.rows, a.ldx) || !extent_ok(q_rows, a.ldq))) return CUOPX_INVALID_ARGUMENT;
  if (a.rows >= (int64_t(1) << 31) || a.cols >= (int64_t(1) << 31)) return CUOPX_INVALID_ARGUMENT;
  // The column kernels' grid holds 65535 groups of 128 rows.
  if (a.trans && a.rows > 65535ll * 128) return CUOPX_INVALID_ARGUMENT;
  const size_t need = quantize_workspace(a);
  if (need > 0 && (!a.workspace || a.workspace_bytes < need)) return CUOPX_RESOURCE_UNAVAILABLE;
  const Extent x{a.X, a.rows, a.cols, a.ldx, es}, q{a.Q, q_rows, q_cols, a.ldq, 1};
  const Extent scale = vector_extent(a.scale, static_cast<size_t>(q_rows) * 4);
  const Extent scratch = vector_extent(need ? a.workspace : nullptr, need);
  if (overlaps(q, x) || overlaps(scale, x) || overlaps(scale, q)) return CUOPX_INVALID_ARGUMENT;
  if (overlaps(scratch, x) || overlaps(scratch, q) || overlaps(scratch, scale)) return CUOPX_INVALID_ARGUMENT;
  return -1;
}

// Scales of rows without elements.
__global__ void __launch_bounds__(256) quantize_empty_kernel(float* scale, int64_t n) {
  const int64_t i = blockIdx.x * 256ll + threadIdx.x;
  if (i < n) scale[i] = row_scale(0.f).scale;
}

int quantize(const cuopx_quantize_args* a, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (const int v = validate_quantize(*a); v >= 0) return v;
  const QuantParams p{a->rows, a->cols, a->X, a->ldx, a->Q, a->ldq, a->scale};
  if ((a->trans ? a->rows : a->cols) == 0) {
    const int64_t n = a->trans ? a->cols : a->rows;
    quantize_empty_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, stream>>>(a->scale, n);
    note_launch("quantize_empty");
    return check_launch();
  }
  if (!a->trans) return quantize_rows(a->dtype, p, stream);
  uint32_t* top = static_cast<uint32_t*>(a->workspace);
  switch (a->dtype) {
    case CUOPX_F32: return quantize_columns_typed<float>(p, top, stream);
    case CUOPX_F16: return quantize_columns_typed<__half>(p, top, stream);
    default: return quantize_columns_typed<__nv_bfloat16>(p, top, stream);
  }
}

}  // namespace

}  // namespace cuopx

extern "C" {

size_t cuopx_quantize_workspace_size(const cuopx_quantize_args* args) { return args ? cuopx::quantize_workspace(*args) : 0; }

int cuopx_quantize(const cuopx_quantize_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_quantize", args ? args->rows : 0, args ? args->cols : 0, 0);
  return scope.done(cuopx::quantize(args, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
