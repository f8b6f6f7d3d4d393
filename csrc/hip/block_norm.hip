// Gated residual norm and counter-based dropout, hand-written for gfx950.
//
//   u = norm_post(y)                              none | rms | layer
//   r = x_scale x + y_scale g keep(u) up          g: none | [D] | [M] | [M, D], raw or sigmoid
//   h = norm_pre(r)                               none | rms | layer
//
// Memory bound: forward reads x, y (and a full gate) and writes r and h once;
// backward reads dr, dh, x, y (and a full gate) and writes dx, dy (and dgate).
// A row stays in registers between its statistics and its output, 8
// consecutive columns a thread and chunk; statistics are fp32, the variance is
// taken around the mean (two passes over the registers, none over memory).
// h is the norm of r before r is rounded to the stream's type (one rounding
// from the inputs), and the backward makes that same r again from x and y: it
// costs the bytes that a saved r would (x in its place), and a gradient of a
// weight, held in 32 bits, does not take on the rounding of a 16-bit stream.
// The dropout mask is drawn again in the backward, never stored.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "block_ops.h"

namespace pbx {
namespace {

// sum over the L threads that share a row; red: LDS of one float a wave, its
// own for each call of a row (so one barrier a call suffices)
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 1; o < (L < 64 ? L : 64); o <<= 1) v += __shfl_xor(v, o);
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < L / 64; ++w) v += red[w];
  }
  return v;
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

// normalises v (C chunks of 8, `valid` columns each) in place; returns (mean, 1/dev)
template <int L, int C>
__device__ __forceinline__ float2 normalise(float v[C][8], const int valid[C], int D, int kind, float eps, float* red) {
  float mean = 0.f;
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[c][j];
    mean = row_sum<L>(s, red) / (float)D;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = j < valid[c] ? v[c][j] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) q += v[c][j] * v[c][j];
  const float inv = 1.f / sqrtf(row_sum<L>(q, red + 16) / (float)D + eps);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[c][j] *= inv;
  return {mean, inv};
}

template <int L, int C>
__device__ __forceinline__ void affine(float v[C][8], const int valid[C], const int col[C], const float* w, const float* b) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float wv[8], bv[8];
    load8(w + col[c], valid[c], wv);
    if (b) load8(b + col[c], valid[c], bv);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[c][j] = b ? v[c][j] * wv[j] + bv[j] : v[c][j] * wv[j];
  }
}

// L threads a row, C chunks of 8 columns a thread: column (c L + lane) 8 + j
template <int TR, int TT, int L, int C>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_residual_fwd(ResidualArgs a) {
  using R = typename BlockElem<TR>::type;
  using E = typename BlockElem<TT>::type;
  constexpr int kRows = L < 256 ? 256 / L : 1;
  __shared__ float red[64];
  const Seed sd = mask_seed(a.mask);
  keep_seed(a.mask, sd);
  const int lane = threadIdx.x % L;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / L;
  if (row >= a.M) return;  // the same for every thread of a row
  int col[C], valid[C];
  float u[C][8], x[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    col[c] = (c * L + lane) * 8;
    valid[c] = max(0, min(8, a.D - col[c]));
    if (!valid[c]) col[c] = 0;
    load8((const E*)a.y + row * a.ldy + col[c], valid[c], u[c]);
    load8((const R*)a.x + row * a.ldx + col[c], valid[c], x[c]);
  }
  float2 ps{0.f, 1.f}, qs{0.f, 1.f};
  if (a.post) {
    ps = normalise<L, C>(u, valid, a.D, a.post, a.eps, red);
    affine<L, C>(u, valid, col, a.post_w, a.post_b);
  }
  float grow = 1.f;
  if (a.gate_kind == kGateRow) {
    grow = ((const float*)a.gate)[row];
    if (a.sigmoid) grow = sigmoid(grow);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t keep = a.mask.thr && valid[c] ? keep8(row * a.D + col[c], sd.seed, sd.offset, a.mask.thr) : 0xffu;
    float g[8];
    if (a.gate_kind == kGateChannel) load8((const float*)a.gate + col[c], valid[c], g);
    else if (a.gate_kind == kGateFull) load8((const E*)a.gate + row * a.ldg + col[c], valid[c], g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float gv = grow;
      if (a.gate_kind == kGateChannel || a.gate_kind == kGateFull) gv = a.sigmoid ? sigmoid(g[j]) : g[j];
      const float d = (keep >> j & 1) ? u[c][j] * a.mask.up : 0.f;
      u[c][j] = j < valid[c] ? a.x_scale * x[c][j] + a.y_scale * (gv * d) : 0.f;
    }
    store8((R*)a.r + row * a.D + col[c], valid[c], u[c]);
  }
  if (a.pre) {
    qs = normalise<L, C>(u, valid, a.D, a.pre, a.eps, red + 32);
    affine<L, C>(u, valid, col, a.pre_w, a.pre_b);
#pragma unroll
    for (int c = 0; c < C; ++c) store8((E*)a.h + row * a.D + col[c], valid[c], u[c]);
  }
  if (a.stats && lane == 0) {
    float4 st{ps.x, ps.y, qs.x, qs.y};
    reinterpret_cast<float4*>(a.stats)[row] = st;
  }
}

// gradient of a norm's input from g = d(out) * w and the normalised n, in place in g
template <int L, int C>
__device__ __forceinline__ void norm_back(float g[C][8], float n[C][8], const int valid[C], int D, int kind, float inv,
                                          float* red) {
  float sgn = 0.f, sg = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sgn += g[c][j] * n[c][j];
      sg += g[c][j];
    }
  sgn = row_sum<L>(sgn, red) / (float)D;
  sg = kind == kNormLayer ? row_sum<L>(sg, red + 16) / (float)D : 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) g[c][j] = j < valid[c] ? inv * (g[c][j] - n[c][j] * sgn - sg) : 0.f;
}

// Column sums (weights, biases, channel gate) stay in registers over the rows
// a group walks, are added over the groups of a workgroup in order and leave
// as one slab row; k_block_cols adds the slab rows in order: no atomics, the
// same bits every time.
template <int TR, int TT, int L, int C>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_residual_bwd(ResidualArgs a) {
  using R = typename BlockElem<TR>::type;
  using E = typename BlockElem<TT>::type;
  constexpr int kRows = L < 256 ? 256 / L : 1;
  __shared__ float red[2][128];
  __shared__ float part[kRows > 1 ? kRows : 1][kRows > 1 ? L * 8 : 1];
  const Seed sd = mask_seed(a.mask);
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  int col[C], valid[C];
  float s_prew[C][8], s_preb[C][8], s_gate[C][8], s_postw[C][8], s_postb[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    col[c] = (c * L + lane) * 8;
    valid[c] = max(0, min(8, a.D - col[c]));
    if (!valid[c]) col[c] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) s_prew[c][j] = s_preb[c][j] = s_gate[c][j] = s_postw[c][j] = s_postb[c][j] = 0.f;
  }
  int it = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + grp; row < a.M; row += (int64_t)gridDim.x * kRows, it ^= 1) {
    float* rd = red[it];  // two sets in turn: a wave may be one row ahead of another, never two
    const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
    float grow = 1.f;
    if (a.gate_kind == kGateRow) {
      grow = ((const float*)a.gate)[row];
      if (a.sigmoid) grow = sigmoid(grow);
    }
    // the forward again: un = normalised y, d = keep(u) up, c = y_scale g (so r = x_scale x + c d), n = normalised r
    float un[C][8], d[C][8], gv[C][8], n[C][8], t[C][8];
    uint32_t keep[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float w[8], b[8], x[8];
      load8((const E*)a.y + row * a.ldy + col[c], valid[c], un[c]);
      if (a.gate_kind == kGateChannel) load8((const float*)a.gate + col[c], valid[c], gv[c]);
      else if (a.gate_kind == kGateFull) load8((const E*)a.gate + row * a.ldg + col[c], valid[c], gv[c]);
      const bool pre = a.pre && a.dh;
      if (pre) {
        load8((const R*)a.x + row * a.ldx + col[c], valid[c], x);
        load8((const E*)a.dh + row * a.lddh + col[c], valid[c], t[c]);
      }
      if (a.post) {
        load8(a.post_w + col[c], valid[c], w);
        if (a.post_b) load8(a.post_b + col[c], valid[c], b);
      }
      keep[c] = a.mask.thr && valid[c] ? keep8(row * a.D + col[c], sd.seed, sd.offset, a.mask.thr) : 0xffu;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float u = un[c][j];
        if (a.post) {
          un[c][j] = j < valid[c] ? (un[c][j] - st.x) * st.y : 0.f;
          u = a.post_b ? un[c][j] * w[j] + b[j] : un[c][j] * w[j];
        }
        d[c][j] = (keep[c] >> j & 1) ? u * a.mask.up : 0.f;
        if (a.gate_kind == kGateChannel || a.gate_kind == kGateFull) {
          if (a.sigmoid) gv[c][j] = sigmoid(gv[c][j]);
        } else {
          gv[c][j] = grow;
        }
      }
      if (pre) {
        load8(a.pre_w + col[c], valid[c], w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float r = a.x_scale * x[j] + a.y_scale * (gv[c][j] * d[c][j]);
          n[c][j] = j < valid[c] ? (r - st.z) * st.w : 0.f;
          s_prew[c][j] += t[c][j] * n[c][j];
          s_preb[c][j] += t[c][j];
          t[c][j] *= w[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[c][j] = 0.f;
      }
    }
    // t = dr + norm_pre'(dh)
    if (a.pre && a.dh) norm_back<L, C>(t, n, valid, a.D, a.pre, st.w, rd);
    float gdot = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float g[8], w[8];
      if (a.dr) {
        load8((const R*)a.dr + row * a.lddr + col[c], valid[c], g);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[c][j] += g[j];
      }
      if (a.dx) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = a.x_scale * t[c][j];
        store8((R*)a.dx + row * a.D + col[c], valid[c], g);
      }
      if (a.post) load8(a.post_w + col[c], valid[c], w);
      // dgate = y_scale t d slope, du = y_scale t g keep up
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float tg = a.y_scale * t[c][j];
        g[j] = tg * d[c][j];
        if (a.sigmoid && a.gate_kind != kGateRow) g[j] *= gv[c][j] * (1.f - gv[c][j]);
        s_gate[c][j] += g[j];
        gdot += g[j];
        const float du = (keep[c] >> j & 1) ? tg * gv[c][j] * a.mask.up : 0.f;
        s_postw[c][j] += du * un[c][j];
        s_postb[c][j] += du;
        t[c][j] = a.post ? du * w[j] : du;
      }
      if (a.gate_kind == kGateFull && a.dgate) store8((E*)a.dgate + row * a.D + col[c], valid[c], g);
    }
    if (a.gate_kind == kGateRow && a.dgate) {
      gdot = row_sum<L>(gdot, rd + 32);
      if (lane == 0) ((float*)a.dgate)[row] = a.sigmoid ? gdot * grow * (1.f - grow) : gdot;
    }
    if (a.dy) {
      if (a.post) norm_back<L, C>(t, un, valid, a.D, a.post, st.y, rd + 64);
#pragma unroll
      for (int c = 0; c < C; ++c) store8((E*)a.dy + row * a.D + col[c], valid[c], t[c]);
    }
  }
  // slab row blockIdx.x: the wanted sums in the order of residual_nvec
  int v = 0;
  auto leave = [&](float s[C][8], bool wanted) {
    if (!wanted) return;
    float* out = a.slab + ((int64_t)blockIdx.x * residual_nvec(a) + v) * a.D;
    ++v;
    if constexpr (kRows == 1) {
#pragma unroll
      for (int c = 0; c < C; ++c) store8(out + col[c], valid[c], s[c]);
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) part[grp][lane * 8 + j] = s[c][j];
        __syncthreads();
        for (int i = threadIdx.x; i < L * 8; i += 256) {
          const int cc = c * L * 8 + i;
          if (cc >= a.D) continue;
          float q = 0.f;
          for (int g = 0; g < kRows; ++g) q += part[g][i];
          out[cc] = q;
        }
      }
    }
  };
  leave(s_prew, a.dpre_w != nullptr);
  leave(s_preb, a.dpre_b != nullptr);
  leave(s_gate, a.gate_kind == kGateChannel && a.dgate != nullptr);
  leave(s_postw, a.dpost_w != nullptr);
  leave(s_postb, a.dpost_b != nullptr);
}

struct ColOut {
  float* p[5];
};
// out[v][c] = sum over the slab's rows, in an order of their number alone: 64
// columns a workgroup, 16 waves take every 16th row, eight loads in flight.
__global__ __launch_bounds__(1024) void k_block_cols(const float* __restrict__ slab, int64_t rows, int64_t W, int64_t D,
                                                     ColOut o) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s[8] = {};
  if (c < W) {
    int64_t r = w;
    for (; r + 112 < rows; r += 128)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += slab[(r + 16 * i) * W + c];
    for (; r < rows; r += 16) s[0] += slab[r * W + c];
  }
  red[w][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (w == 0 && c < W) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) q += red[i][lane];
    const int v = (int)(c / D);
    float* p = v == 0 ? o.p[0] : v == 1 ? o.p[1] : v == 2 ? o.p[2] : v == 3 ? o.p[3] : o.p[4];
    p[c - (int64_t)v * D] = q;
  }
}

template <typename E>
__global__ __launch_bounds__(256) void k_dropout(const E* __restrict__ x, E* __restrict__ y, int64_t n, MaskArgs m) {
  const Seed sd = mask_seed(m);
  keep_seed(m, sd);
  const int64_t step = (int64_t)gridDim.x * 256 * 8;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += step) {
    const int valid = n - i < 8 ? (int)(n - i) : 8;
    float v[8];
    load8(x + i, valid, v);
    const uint32_t keep = m.thr ? keep8(i, sd.seed, sd.offset, m.thr) : 0xffu;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (keep >> j & 1) ? v[j] * m.up : 0.f;
    store8(y + i, valid, v);
  }
}

template <int L, int C, typename F>
void by_types(const ResidualArgs& a, F f) {
  if (a.stream_t == kF32) {
    if (a.t == kF32) f(std::integral_constant<int, kF32>{}, std::integral_constant<int, kF32>{});
    else if (a.t == kBF16) f(std::integral_constant<int, kF32>{}, std::integral_constant<int, kBF16>{});
    else f(std::integral_constant<int, kF32>{}, std::integral_constant<int, kF16>{});
  } else if (a.stream_t == kBF16) {
    f(std::integral_constant<int, kBF16>{}, std::integral_constant<int, kBF16>{});
  } else {
    f(std::integral_constant<int, kF16>{}, std::integral_constant<int, kF16>{});
  }
}

// threads a row by its width: one chunk of 8 columns a thread
template <typename F>
void by_width(int D, F f) {
  if (D <= 128) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  else if (D <= 512) f(std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
  else if (D <= 2048) f(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
  else if (D <= 4096) f(std::integral_constant<int, 512>{}, std::integral_constant<int, 1>{});
  else if (D <= 8192) f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 1>{});
  else f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 2>{});
}

}  // namespace

int residual_slab_rows(int64_t M, int D) {
  const int rows = D <= 128 ? 16 : D <= 512 ? 4 : 1;
  const int64_t need = (M + rows - 1) / rows;
  return (int)(need < 1024 ? need : 1024);
}

void launch_residual_fwd(const ResidualArgs& a, hipStream_t s) {
  if (a.M == 0 || a.D == 0) return;
  by_width(a.D, [&](auto l, auto c) {
    constexpr int L = decltype(l)::value, C = decltype(c)::value, rows = L < 256 ? 256 / L : 1;
    by_types<L, C>(a, [&](auto tr, auto tt) {
      hipLaunchKernelGGL((k_residual_fwd<decltype(tr)::value, decltype(tt)::value, L, C>),
                         dim3((unsigned)((a.M + rows - 1) / rows)), dim3(L < 256 ? 256 : L), 0, s, a);
    });
  });
}

void launch_residual_bwd(const ResidualArgs& a, hipStream_t s) {
  if (a.M == 0 || a.D == 0) return;
  const int grid = residual_slab_rows(a.M, a.D);
  by_width(a.D, [&](auto l, auto c) {
    constexpr int L = decltype(l)::value, C = decltype(c)::value;
    by_types<L, C>(a, [&](auto tr, auto tt) {
      hipLaunchKernelGGL((k_residual_bwd<decltype(tr)::value, decltype(tt)::value, L, C>), dim3(grid),
                         dim3(L < 256 ? 256 : L), 0, s, a);
    });
  });
  const int nvec = residual_nvec(a);
  if (!nvec) return;
  float* out[5];
  int v = 0;
  if (a.dpre_w) out[v++] = a.dpre_w;
  if (a.dpre_b) out[v++] = a.dpre_b;
  if (a.gate_kind == kGateChannel && a.dgate) out[v++] = (float*)a.dgate;
  if (a.dpost_w) out[v++] = a.dpost_w;
  if (a.dpost_b) out[v++] = a.dpost_b;
  launch_block_cols(a.slab, grid, (int64_t)nvec * a.D, out, nvec, a.D, s);
}

void launch_block_cols(const float* slab, int64_t rows, int64_t W, float* const* out, int nout, int64_t D, hipStream_t s) {
  ColOut o{};
  for (int i = 0; i < nout; ++i) o.p[i] = out[i];
  hipLaunchKernelGGL(k_block_cols, dim3((unsigned)((W + 63) / 64)), dim3(1024), 0, s, slab, rows, W, D, o);
}

void launch_dropout(const void* x, void* y, int64_t n, BlockType t, const MaskArgs& m, hipStream_t s) {
  if (n <= 0) return;
  const int64_t need = (n + 2047) / 2048;
  const dim3 g((unsigned)(need < 8192 ? need : 8192));
  if (t == kF32) hipLaunchKernelGGL(k_dropout<float>, g, dim3(256), 0, s, (const float*)x, (float*)y, n, m);
  else if (t == kBF16) hipLaunchKernelGGL(k_dropout<__bf16>, g, dim3(256), 0, s, (const __bf16*)x, (__bf16*)y, n, m);
  else hipLaunchKernelGGL(k_dropout<_Float16>, g, dim3(256), 0, s, (const _Float16*)x, (_Float16*)y, n, m);
}

}  // namespace pbx
