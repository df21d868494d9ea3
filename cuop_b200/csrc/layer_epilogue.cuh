// Epilogue of the tcgen05 layer kernels: bias, kept pre-activation,
// activation, product of the two projections, residual, one rounding, TMA
// stores.  A warp drains its 32 accumulator rows in 64-column chunks (the box
// of a TMA store), each in two halves of 32 columns.
#pragma once

#include <cuda.h>

#include "activation.cuh"
#include "common.cuh"
#include "dispatch.h"

namespace cuopx {

struct LayerEpi {
  const void* bias;  // NULL: none.  Gated: the gate's N, then the other projection's N
  const void* R;     // residual or NULL
  int64_t ldr;
  int act;
  int has_z;     // store the pre-activation
  int vec_bias;  // bias can be read in 16-byte groups
  int vec_res;   // so can the residual's rows
  void* Y;
  int64_t ldy;
  void* Z;
  int64_t ldz;
  // 64-column chunks that end at or before this column go out by TMA, the
  // others in plain 2-byte stores, 64 columns of a row per two of a warp's: 0
  // where rows do not start on 16-byte boundaries, N where they do not end on one.
  int tma_y, tma_z;
};

inline LayerEpi layer_epi(const LinearProblem& p) {
  LayerEpi e;
  e.bias = p.bias;
  e.R = p.R;
  e.ldr = p.ldr;
  e.act = p.act;
  e.has_z = p.Z != nullptr;
  e.vec_bias = p.N % 8 == 0 && row_aligned16(p.bias, 0);
  e.vec_res = p.N % 8 == 0 && row_aligned16(p.R, p.ldr);
  e.Y = p.Y;
  e.ldy = p.ldy;
  e.Z = p.Z;
  e.ldz = p.ldz;
  const int inside = tma_store_cols<2>(p.N);
  e.tma_y = row_aligned16(p.Y, p.ldy) ? inside : 0;
  e.tma_z = p.Z && row_aligned16(p.Z, p.ldz) && (!p.gated || p.N % 8 == 0) ? inside : 0;  // gated: U starts at column N
  return e;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2_layer(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

template <typename T>
__device__ __forceinline__ float2 unpack2_layer(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    // bf16 is the upper half of a float.
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<__half2*>(&w));
  }
}

// 32 elements of a row from column `col` on, zeros past column N.
template <typename T>
__device__ __forceinline__ void load_row32(const T* row, int64_t col, int64_t N, bool vec, uint4 (&raw)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    raw[j] = make_uint4(0, 0, 0, 0);
    if (vec) {  // N is a multiple of 8: a group is inside or outside
      if (col + 8 * j < N) raw[j] = *reinterpret_cast<const uint4*>(row + col + 8 * j);
    } else {
      uint32_t* w = &raw[j].x;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + 8 * j + i < N)
          w[i / 2] |= static_cast<uint32_t>(*reinterpret_cast<const unsigned short*>(row + col + 8 * j + i)) << (16 * (i & 1));
    }
  }
}

template <typename T>
__device__ __forceinline__ void add_row32(float (&v)[32], const uint4 (&raw)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2_layer<T>(w[i]);
      v[8 * j + 2 * i] += f.x;
      v[8 * j + 2 * i + 1] += f.y;
    }
  }
}

// Rounds 32 values into half `h` of this lane's 128-byte staging row
// (128-byte swizzle: 16-byte group j of row r at j ^ (r & 7)).
template <typename T>
__device__ __forceinline__ void stage_row32(unsigned char* buf, int lane, int h, const float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 w;
    w.x = pack2_layer<T>(v[8 * j + 0], v[8 * j + 1]);
    w.y = pack2_layer<T>(v[8 * j + 2], v[8 * j + 3]);
    w.z = pack2_layer<T>(v[8 * j + 4], v[8 * j + 5]);
    w.w = pack2_layer<T>(v[8 * j + 6], v[8 * j + 7]);
    *reinterpret_cast<uint4*>(buf + lane * 128 + (((4 * h + j) ^ (lane & 7)) << 4)) = w;
  }
}

// One warp's rows of PART columns of one tile.  t_row: TMEM address of the
// first of them in this warp's lane quarter; the second projection's (GATED)
// are COLS further on.  `stage`: 3 (GATED) or 2
// staging buffers of 4 KB.  wait() returns once the accumulator is complete (false: give up),
// release() is called once it has been read, partial() adds what other CTAs
// have summed.  (n0, m0): output column and first row of this warp's box.
struct NoPartialSums {
  template <typename... A>
  __device__ __forceinline__ void operator()(A&&...) const {}
};

template <typename T, bool GATED, int COLS, int PART, typename Wait, typename Release, typename Partial = NoPartialSums>
__device__ __forceinline__ bool layer_epilogue_tile(uint32_t t_row, int n0, int m0, int M, int N, const LayerEpi& e,
                                                    const CUtensorMap* tmY, const CUtensorMap* tmZ,
                                                    const CUtensorMap* tmZ2, unsigned char* stage, int lane, int& ybuf,
                                                    Wait&& wait, Release&& release, Partial&& partial = Partial{}) {
  constexpr int BUF = 32 * 64 * 2;
  constexpr int NBUF = GATED ? 3 : 2;
  const int64_t grow = static_cast<int64_t>(m0) + lane;
  const bool has_res = !GATED && e.R != nullptr && grow < M;
  const T* rrow = static_cast<const T*>(e.R) + grow * e.ldr;
  const T* bias = static_cast<const T*>(e.bias);
  // Bias and residual of the first half are on their way before the products
  // are done, those of every other one while the one before it is worked on.
  uint4 nbias[GATED ? 2 : 1][4], nres[GATED ? 1 : 4];
  auto fetch = [&](int64_t col) {
    if (bias) {
      load_row32<T>(bias, col, N, e.vec_bias, nbias[0]);
      if constexpr (GATED) load_row32<T>(bias + N, col, N, e.vec_bias, nbias[1]);
    }
    if constexpr (!GATED) {
      if (has_res) load_row32<T>(rrow, col, N, e.vec_res, nres);
    }
  };
  fetch(n0);
  if (!wait()) return false;
#pragma unroll 1
  for (int half = 0; half < PART / 32; ++half) {
    const int h = half & 1;
    const int64_t col = static_cast<int64_t>(n0) + 32 * half;
    uint32_t ra[32], rb[GATED ? 32 : 1];
    tmem_ld_32x32b_x32(t_row + 32 * half, ra);
    if constexpr (GATED) tmem_ld_32x32b_x32(t_row + COLS + 32 * half, rb);
    tmem_wait_ld();
    if (half == PART / 32 - 1) release();
    float a[32], b[GATED ? 32 : 1];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      a[i] = __uint_as_float(ra[i]);
      if constexpr (GATED) b[i] = __uint_as_float(rb[i]);
    }
    partial(half, a, b);
    if (bias) {
      add_row32<T>(a, nbias[0]);
      if constexpr (GATED) add_row32<T>(b, nbias[1]);
    }
    uint4 res[GATED ? 1 : 4];
    if constexpr (!GATED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) res[i] = nres[i];
    }
    if (half + 1 < PART / 32) fetch(col + 32);
    if (h == 0) {
      // The buffers this chunk fills: with a kept pre-activation all of them,
      // else one, the stores of the previous chunk having the other.
      if (lane == 0) {
        if (e.has_z) bulk_wait_group_read<0>();
        else bulk_wait_group_read<1>();
      }
      __syncwarp();
      if (e.has_z) ybuf = NBUF - 1;
      else ybuf = ybuf == 0 ? 1 : 0;
    }
    if (e.has_z) {
      stage_row32<T>(stage, lane, h, a);
      if constexpr (GATED) stage_row32<T>(stage + BUF, lane, h, b);
    }
    with_activation(e.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        float2 y = act_value2<act.value>(make_float2(a[i], a[i + 1]));
        if constexpr (GATED) y = mul2(y, make_float2(b[i], b[i + 1]));
        a[i] = y.x, a[i + 1] = y.y;
      }
    });
    if constexpr (!GATED) {
      if (has_res) add_row32<T>(a, res);
    }
    stage_row32<T>(stage + ybuf * BUF, lane, h, a);
    if (h == 1) {
      fence_proxy_async_shared();
      __syncwarp();
      const int c = n0 + 32 * (half - 1);
      if (lane == 0) {
        if (e.has_z && c + 64 <= e.tma_z) {
          tma_store_3d(tmZ, stage, c, m0, 0);
          if constexpr (GATED) tma_store_3d(tmZ2, stage + BUF, c, m0, 0);
        }
        if (c + 64 <= e.tma_y) tma_store_3d(tmY, stage + ybuf * BUF, c, m0, 0);
        bulk_commit_group();
      }
      if (e.has_z && c + 64 > e.tma_z) {
        store_staged_chunk<2>(stage, e.Z, e.ldz, c, m0, M, N, lane);
        if constexpr (GATED) store_staged_chunk<2>(stage + BUF, static_cast<T*>(e.Z) + N, e.ldz, c, m0, M, N, lane);
      }
      if (c + 64 > e.tma_y) store_staged_chunk<2>(stage + ybuf * BUF, e.Y, e.ldy, c, m0, M, N, lane);
    }
  }
  return true;
}

}  // namespace cuopx
