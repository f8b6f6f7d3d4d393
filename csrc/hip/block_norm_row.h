// What the forward and backward kernels of the gated residual norm share
// (block_norm.hip, block_norm_bwd_*.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "block_ops.h"

namespace pbx {
namespace {

// 8 elements at any element's address
template <typename E>
using Vec8 = E __attribute__((ext_vector_type(8), aligned(sizeof(E))));


template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// sum over 16 lanes, in each of them, and over the wave: lane moves within the
// vector pipe (a shuffle through LDS costs ten times the latency)
__device__ __forceinline__ float sum16(float v) {
  v += dpp<0xB1>(v);   // quad: 1 0 3 2
  v += dpp<0x4E>(v);   // quad: 2 3 0 1
  v += dpp<0x141>(v);  // half row mirrored
  v += dpp<0x140>(v);  // row mirrored
  return v;
}
__device__ __forceinline__ float sum64(float v) {
  const int s = __builtin_bit_cast(int, sum16(v));
  auto lane = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(s, l)); };
  return (lane(0) + lane(16)) + (lane(32) + lane(48));
}

// sums of K values over the L threads that share a row; red: LDS of K floats a
// wave, its own for each call of a row (so one barrier a call suffices)
template <int L, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float* red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = L == 16 ? sum16(v[k]) : sum64(v[k]);
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) red[(threadIdx.x >> 6) * K + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < L / 64; ++w) v[k] += red[w * K + k];
    }
  }
}
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
  float a[1] = {v};
  row_sums<L>(a, red);
  return a[0];
}

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + expf(-v)); }

struct Seed {
  uint64_t seed, offset;
};
__device__ __forceinline__ Seed mask_seed(const MaskArgs& m) {
  if (m.seed) return {(uint64_t)m.seed[0], (uint64_t)m.seed[1]};
  return {(uint64_t)m.seed_v, (uint64_t)m.offset_v};
}
__device__ __forceinline__ void keep_seed(const MaskArgs& m, const Seed& s) {
  if (m.seed_out && blockIdx.x == 0 && threadIdx.x == 0) {
    m.seed_out[0] = (int64_t)s.seed;
    m.seed_out[1] = (int64_t)s.offset;
  }
}

// The columns of one thread: C chunks of 8, chunk c of lane l from column
// min((c L + l) 8, D - 8).  In a row whose width is no multiple of 8 the last
// chunk thus begins inside the one before: loads and stores are whole vectors
// everywhere (what two lanes store twice is the same value), and the first
// `skip` columns, which the other lane counts, stay out of the row's sums.
// skip = 8: no chunk.  NARROW: rows of less than 8 columns, lane 0 alone.
template <int L, int C, bool NARROW>
struct Columns {
  int col[C], skip[C], width;
  float per;  // 1 / width
  __device__ __forceinline__ Columns(int lane, int D) : width(D), per(1.f / (float)D) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = (c * L + lane) * 8;
      col[c] = NARROW ? 0 : max(0, min(at, D - 8));
      skip[c] = at < D ? at - col[c] : 8;
    }
  }
  __device__ __forceinline__ bool any(int c) const { return skip[c] < 8; }
  __device__ __forceinline__ bool counts(int c, int j) const { return NARROW ? skip[c] == 0 && j < width : j >= skip[c]; }
  // sum of f(j) over the columns of chunk c that count; the rare chunk with others takes a branch of its own
  template <typename F>
  __device__ __forceinline__ float sum(int c, F f) const {
    float s = 0.f;
    if (NARROW) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s += counts(c, j) ? f(j) : 0.f;
      return s;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s += f(j);
    if (skip[c]) {
      s = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += j >= skip[c] ? f(j) : 0.f;
    }
    return s;
  }
  template <typename E>
  __device__ __forceinline__ Vec8<E> load(int c, const E* row) const {
    Vec8<E> v;
    if (NARROW) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < width ? row[j] : (E)0.f;
    } else {
      v = *reinterpret_cast<const Vec8<E>*>(row + col[c]);
    }
    return v;
  }
  template <typename E>
  __device__ __forceinline__ void store(int c, E* row, const float v[8]) const {
    if (!any(c)) return;
    Vec8<E> x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (E)v[j];
    if (NARROW) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < width) row[j] = x[j];
    } else {
      *reinterpret_cast<Vec8<E>*>(row + col[c]) = x;
    }
  }
};

// normalises v in place; returns (mean, 1/dev)
template <int L, int C, bool N>
__device__ __forceinline__ float2 normalise(float v[C][8], const Columns<L, C, N>& at, int kind, float eps, float* red) {
  float mean = 0.f;
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) s += at.sum(c, [&](int j) { return v[c][j]; });
    mean = row_sum<L>(s, red) * at.per;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] -= mean;
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) q += at.sum(c, [&](int j) { return v[c][j] * v[c][j]; });
  const float inv = 1.f / sqrtf(row_sum<L>(q, red + 16) * at.per + eps);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[c][j] *= inv;
  return {mean, inv};
}

template <int L, int C, bool N>
__device__ __forceinline__ void affine(float v[C][8], const Columns<L, C, N>& at, const float* w, const float* b) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const Vec8<float> wv = at.load(c, w);
    if (b) {
      const Vec8<float> bv = at.load(c, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = v[c][j] * wv[j] + bv[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] *= wv[j];
    }
  }
}

// threads a row by its width: one chunk of 8 columns a thread
template <typename F>
void by_width(int D, F f) {
  using std::integral_constant;
  if (D < 8) f(integral_constant<int, 16>{}, integral_constant<int, 1>{}, integral_constant<bool, true>{});
  else if (D <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 1>{}, integral_constant<bool, false>{});
  else if (D <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 1>{}, integral_constant<bool, false>{});
  else if (D <= 2048) f(integral_constant<int, 256>{}, integral_constant<int, 1>{}, integral_constant<bool, false>{});
  else if (D <= 4096) f(integral_constant<int, 512>{}, integral_constant<int, 1>{}, integral_constant<bool, false>{});
  else if (D <= 8192) f(integral_constant<int, 1024>{}, integral_constant<int, 1>{}, integral_constant<bool, false>{});
  else f(integral_constant<int, 1024>{}, integral_constant<int, 2>{}, integral_constant<bool, false>{});
}

}  // namespace
}  // namespace pbx
