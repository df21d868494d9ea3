// Linear and gated linear layers on int8 operands (cuopx_int8_linear,
// cuopx_int8_gated_linear):
//   S = Xq Wq^T (int32, exact),  Z = S * x_scale[row] * w_scale[column] + b,
//   Y = act(Z) + R,  or with [G | U] = Z  Y = act(G) * U.
// The products run on the layers' tcgen05 kernels (gemm_tc2.cu, linear_pair.cu,
// linear_split.cu) with kind::i8, whose K blocks of 128 bytes hold twice the
// elements, at twice the rate; the scales go into their epilogue.  16-bit
// activations are quantised by one pass before (quantize.cu).
#include "activation.cuh"
#include "common.cuh"
#include "dispatch.h"

namespace cuopx {

namespace {

constexpr int64_t kInt8MaxK = 131071;  // 2^14 K < 2^31

// ---------------------------------------------------------------- any size and alignment
// 64 x 64 outputs per CTA, 32-deep steps through shared memory, 4 x 4 outputs
// per thread (of both projections when gated), four products per instruction.
constexpr int I8S_T = 64, I8S_K = 32;

template <typename T, bool GATED>
__global__ void __launch_bounds__(256) int8_linear_simt_kernel(const LinearProblem p) {
  constexpr int NB = GATED ? 2 : 1;
  __shared__ int xs[I8S_T][I8S_K / 4 + 1];
  __shared__ int ws[NB][I8S_T][I8S_K / 4 + 1];
  const int8_t* X = static_cast<const int8_t*>(p.X);
  const int8_t* W = static_cast<const int8_t*>(p.W);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t tiles_n = (p.N + I8S_T - 1) / I8S_T, tiles = tiles_n * ((p.M + I8S_T - 1) / I8S_T);
  grid_dependency_wait();
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t m0 = t / tiles_n * I8S_T, n0 = t % tiles_n * I8S_T;
    int acc[NB][4][4] = {};
    for (int64_t k0 = 0; k0 < p.K; k0 += I8S_K) {
      __syncthreads();
      for (int e = threadIdx.x; e < I8S_T * I8S_K; e += 256) {
        const int r = e / I8S_K, k = e % I8S_K;
        const bool in = k0 + k < p.K;
        reinterpret_cast<int8_t*>(xs[r])[k] = in && m0 + r < p.M ? X[(m0 + r) * p.ldx + k0 + k] : int8_t(0);
#pragma unroll
        for (int h = 0; h < NB; ++h)
          reinterpret_cast<int8_t*>(ws[h][r])[k] = in && n0 + r < p.N ? W[(h * p.w_up + n0 + r) * p.ldw + k0 + k] : int8_t(0);
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < I8S_K / 4; ++k)
#pragma unroll
        for (int h = 0; h < NB; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[h][i][j] = __dp4a(xs[ty + 16 * i][k], ws[h][tx + 16 * j][k], acc[h][i][j]);
    }
    with_activation(p.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty + 16 * i;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t n = n0 + tx + 16 * j;
          if (n >= p.N) continue;
          float z[NB];
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            z[h] = p.K > 0 ? __int2float_rn(acc[h][i][j]) * p.xs[m] * p.ws[h * p.N + n] : 0.f;
            if (p.bias) z[h] += to_acc<T>(static_cast<const T*>(p.bias)[h * p.N + n]);
          }
          float y = act_value<act.value>(z[0]);
          if constexpr (GATED) y *= z[NB - 1];
          if (p.R) y += to_acc<T>(static_cast<const T*>(p.R)[m * p.ldr + n]);
          static_cast<T*>(p.Y)[m * p.ldy + n] = from_acc<T>(y);
        }
      }
    });
  }
}

template <typename T>
cudaError_t launch_int8_simt(const LinearProblem& p, cudaStream_t stream) {
  const int64_t tiles = ((p.N + I8S_T - 1) / I8S_T) * ((p.M + I8S_T - 1) / I8S_T);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(tiles, 1 << 30)));
  return p.gated ? launch_pdl(int8_linear_simt_kernel<T, true>, grid, dim3(256), 0, stream, p)
                 : launch_pdl(int8_linear_simt_kernel<T, false>, grid, dim3(256), 0, stream, p);
}

int int8_linear_simt(const LinearProblem& p, cudaStream_t stream) {
  const cudaError_t err =
      p.dtype == CUOPX_BF16 ? launch_int8_simt<__nv_bfloat16>(p, stream) : launch_int8_simt<__half>(p, stream);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  note_launch(p.gated ? "int8_gated_linear_simt" : "int8_linear_simt");
  return check_launch();
}

// ---------------------------------------------------------------- copies on 16-byte boundaries
// Rows of bytes to rows that start on 16-byte boundaries, for TMA: five
// aligned words around the sixteen bytes where all lie inside the row.
__global__ void __launch_bounds__(256)
    int8_repack_kernel(const int8_t* src, int64_t rows, int64_t cols, int64_t ld, int8_t* dst, int64_t ldd) {
  const int64_t groups = (cols + 15) / 16;
  grid_dependency_wait();
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < rows * groups; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = e / groups, c = (e - row * groups) * 16;
    const int8_t* s = src + row * ld + c;
    uint32_t w[4];
    if (c > 0 && c + 20 <= cols) {
      const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s) & 3u);
      const uint32_t* a = reinterpret_cast<const uint32_t*>(s - shift);
      uint32_t v[5];
#pragma unroll
      for (int i = 0; i < 5; ++i) v[i] = a[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], 8 * shift);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (c + 4 * i + b < cols) w[i] |= static_cast<uint32_t>(static_cast<uint8_t>(s[4 * i + b])) << (8 * b);
      }
    }
    *reinterpret_cast<uint4*>(dst + row * ldd + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

int int8_repack(const void* src, int64_t rows, int64_t cols, int64_t ld, void* dst, cudaStream_t stream) {
  const int64_t n = rows * (round16(cols) / 16);
  const unsigned ctas = static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, static_cast<int64_t>(device_sm_count()) * 32));
  const cudaError_t err = launch_pdl(int8_repack_kernel, dim3(ctas), dim3(256), 0, stream, static_cast<const int8_t*>(src), rows,
                                     cols, ld, static_cast<int8_t*>(dst), round16(cols));
  if (err != cudaSuccess) {
    cudaGetLastError();
    return cuda_failure(err);
  }
  note_launch("int8_repack");
  return check_launch();
}

// ---------------------------------------------------------------- entry points
LinearProblem int8_problem(const cuopx_int8_linear_args& a, bool gated) {
  LinearProblem p{a.dtype, true, a.activation, gated, a.M,   a.N, a.K,   a.X,     a.ldx, a.W,
                  a.ldw,   a.bias, a.residual, a.ldr, a.Y, a.ldy, nullptr, 0};
  p.w_up = a.N;
  p.int8 = true;
  p.xs = a.x_scale;
  p.ws = a.w_scale;
  return p;
}

// What the workspace holds: the quantised X with its scales, or X's aligned
// copy, and W's.
struct Int8Plan {
  bool fused;  // the product's kernel quantises X
  bool quantise, copy_x, copy_w;
  size_t x_off, scale_off, w_off, bytes;
};

Int8Plan int8_plan(const cuopx_int8_linear_args& a, bool gated) {
  Int8Plan q = {};
  if (a.M <= 0 || a.N <= 0 || a.K <= 0) return q;
  const int64_t wide = gated ? 2 * a.N : a.N;
  const LinearProblem p = int8_problem(a, gated);
  q.quantise = a.x_scale == nullptr;
  // Unaligned int8 operands are copied where the tensor cores pay for it: up to kRepackMinWork
  // multiplications the kernel for any alignment is one launch instead of two or three, but takes 2 us
  // for 32 of K (8 x 130 x 503: 36 us, 9 with copies).
  const bool tensor = a.K > 64 || static_cast<double>(a.M) * static_cast<double>(wide) * static_cast<double>(a.K) >= kRepackMinWork;
  q.copy_x = a.x_scale && tensor && !operand_aligned16(p, a.X, a.M == 1 ? 0 : a.ldx);
  q.copy_w = tensor && !operand_aligned16(p, a.W, a.ldw);
  if (q.quantise && split_quantises(a.M, a.N, a.K, gated) && (q.copy_w || operand_aligned16(p, a.W, a.ldw))) {
    q.fused = true;
    q.quantise = false;
  }
  size_t off = 0;
  q.x_off = off;
  if (q.quantise || q.copy_x) off += round256(static_cast<size_t>(a.M) * round16(a.K));
  q.scale_off = off;
  if (q.quantise) off += round256(static_cast<size_t>(a.M) * 4);
  q.w_off = off;
  if (q.copy_w) off += round256(static_cast<size_t>(wide) * round16(a.K));
  q.bytes = off;
  return q;
}

int validate_int8(const cuopx_int8_linear_args& a, bool gated) {
  if (a.dtype != CUOPX_F16 && a.dtype != CUOPX_BF16) return CUOPX_UNSUPPORTED_TYPE;
  if (!activation_ok(a.activation)) return CUOPX_INVALID_ARGUMENT;
  if (a.M < 0 || a.N < 0 || a.K < 0 || a.N > INT64_MAX / 4 || a.K > kInt8MaxK) return CUOPX_INVALID_ARGUMENT;
  if (gated && a.residual) return CUOPX_INVALID_ARGUMENT;
  if (a.M == 0 || a.N == 0) return CUOPX_SUCCESS;
  const int64_t wide = gated ? 2 * a.N : a.N;
  const size_t es = 2, xes = a.x_scale ? 1 : 2;
  if (!starts_on(2, a.bias, a.residual, a.Y) || !starts_on(xes, a.X) || !starts_on(4, a.x_scale, a.w_scale) ||
      !starts_on(256, a.workspace))
    return CUOPX_INVALID_ARGUMENT;
  if (!extent_ok(a.M, a.ldy) || (a.K > 0 && (!extent_ok(a.M, a.ldx) || !extent_ok(wide, a.ldw))) ||
      (a.residual && !extent_ok(a.M, a.ldr)))
    return CUOPX_INVALID_ARGUMENT;
  if (!a.Y || a.ldy < a.N || !a.w_scale || (a.residual && a.ldr < a.N)) return CUOPX_INVALID_ARGUMENT;
  if (a.K > 0 && (!a.X || !a.W || a.ldx < a.K || a.ldw < a.K)) return CUOPX_INVALID_ARGUMENT;
  if (!extent_ok(a.M, round16(a.K)) || !extent_ok(wide, round16(a.K))) return CUOPX_INVALID_ARGUMENT;
  const size_t need = int8_plan(a, gated).bytes;
  if (need > 0 && (!a.workspace || a.workspace_bytes < need)) return CUOPX_RESOURCE_UNAVAILABLE;
  const Extent x{a.X, a.M, a.K, a.ldx, xes}, w{a.W, wide, a.K, a.ldw, 1}, r{a.residual, a.M, a.N, a.ldr, es};
  const Extent y{a.Y, a.M, a.N, a.ldy, es}, bias = vector_extent(a.bias, static_cast<size_t>(wide) * es);
  const Extent xs = vector_extent(a.x_scale, static_cast<size_t>(a.M) * 4);
  const Extent ws = vector_extent(a.w_scale, static_cast<size_t>(wide) * 4);
  const Extent scratch = vector_extent(need ? a.workspace : nullptr, need);
  for (const Extent& e : {x, w, bias, xs, ws})
    if (overlaps(y, e) || overlaps(scratch, e)) return CUOPX_INVALID_ARGUMENT;
  if (overlaps(scratch, r) || overlaps(scratch, y)) return CUOPX_INVALID_ARGUMENT;
  if (a.residual && !alias_ok(a.Y, a.ldy, a.residual, a.ldr, a.M, a.N, es)) return CUOPX_INVALID_ARGUMENT;
  return -1;
}

int int8_forward(const cuopx_int8_linear_args* a, bool gated, cudaStream_t stream) {
  if (a == nullptr) return CUOPX_INVALID_ARGUMENT;
  if (const int v = validate_int8(*a, gated); v >= 0) return v;
  const Int8Plan q = int8_plan(*a, gated);
  LinearProblem p = int8_problem(*a, gated);
  char* ws = static_cast<char*>(a->workspace);
  if (a->K == 0) return int8_linear_simt(p, stream);  // no sums: no scales are read
  if (q.quantise) {
    const QuantParams quant{a->M, a->K, a->X, a->ldx, reinterpret_cast<int8_t*>(ws + q.x_off), round16(a->K),
                            reinterpret_cast<float*>(ws + q.scale_off)};
    if (const int rc = quantize_rows(a->dtype, quant, stream); rc != CUOPX_SUCCESS) return rc;
    p.xs = quant.scale;
    p.early_w = !q.copy_w;
  } else if (q.copy_x) {
    if (const int rc = int8_repack(a->X, a->M, a->K, a->ldx, ws + q.x_off, stream); rc != CUOPX_SUCCESS) return rc;
  }
  if (q.quantise || q.copy_x) {
    p.X = ws + q.x_off;
    p.ldx = round16(a->K);
  }
  if (q.copy_w) {
    if (const int rc = int8_repack(a->W, p.wide(), a->K, a->ldw, ws + q.w_off, stream); rc != CUOPX_SUCCESS) return rc;
    p.W = ws + q.w_off;
    p.ldw = round16(a->K);
  }
  p.quant_x = q.fused;
  if (linear_split_supported(p) && few_rows(p)) return linear_split(p, stream);
  if (linear_tc2_supported(p)) {
    const int ks = pair_split(p);
    return ks > 1 ? linear_pair(p, ks, stream) : linear_tc2(p, stream);
  }
  return int8_linear_simt(p, stream);
}

}  // namespace

}  // namespace cuopx

extern "C" {

size_t cuopx_int8_linear_workspace_size(const cuopx_int8_linear_args* args) {
  return args ? cuopx::int8_plan(*args, false).bytes : 0;
}
size_t cuopx_int8_gated_linear_workspace_size(const cuopx_int8_linear_args* args) {
  return args ? cuopx::int8_plan(*args, true).bytes : 0;
}

int cuopx_int8_linear(const cuopx_int8_linear_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_int8_linear", args ? args->M : 0, args ? args->N : 0, args ? args->K : 0);
  return scope.done(cuopx::int8_forward(args, false, static_cast<cudaStream_t>(stream)));
}

int cuopx_int8_gated_linear(const cuopx_int8_linear_args* args, void* stream) {
  cuopx::ApiScope scope("cuopx_int8_gated_linear", args ? args->M : 0, args ? args->N : 0, args ? args->K : 0);
  return scope.done(cuopx::int8_forward(args, true, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
