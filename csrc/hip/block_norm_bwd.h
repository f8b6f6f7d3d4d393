// Backward kernel of the gated residual norm.  One source a pair of types
// (block_norm_bwd_*.hip) includes this, so that they build side by side.
#pragma once
#include <hip/hip_runtime.h>

#include "block_norm_row.h"

namespace pbx {
namespace {

// gradient of a norm's input from g = d(out) * w and the normalised n, in place in g
template <int L, int C, bool N>
__device__ __forceinline__ void norm_back(float g[C][8], const float n[C][8], const Columns<L, C, N>& at, int kind, float inv,
                                          float* red) {
  float sgn = 0.f, sg = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sgn += at.counts(c, j) ? g[c][j] * n[c][j] : 0.f;
      if (kind == kNormLayer) sg += at.counts(c, j) ? g[c][j] : 0.f;
    }
  sgn = row_sum<L>(sgn, red) / (float)at.width;
  if (kind == kNormLayer) sg = row_sum<L>(sg, red + 16) / (float)at.width;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) g[c][j] = inv * (g[c][j] - n[c][j] * sgn - sg);
}

// Column sums (weights, biases, channel gate) stay in registers over the rows
// a group walks, are added over the groups of a workgroup in order and leave
// as one slab row; k_block_cols adds the slab rows in order: no atomics, the
// same bits every time.
//
// LAYER: either norm has a bias, GATE: the gate is one of channels: which sums
// there are to hold.  With those that are not needed held as well the kernel
// took 180 registers a lane, one workgroup a CU, and twice the time.
template <int TR, int TT, int L, int C, bool N, bool LAYER, bool GATE>
__global__ __launch_bounds__(L < 256 ? 256 : L, L < 512 ? 2 : L == 512 && !LAYER ? 4 : 1) void k_residual_bwd(ResidualArgs a) {
  using R = typename BlockElem<TR>::type;
  using E = typename BlockElem<TT>::type;
  constexpr int kRows = L < 256 ? 256 / L : 1;
  __shared__ float red[2][128];
  __shared__ float part[kRows > 1 ? kRows : 1][kRows > 1 ? L * 8 : 1];
  const Seed sd = mask_seed(a.mask);
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  const Columns<L, C, N> at(lane, a.D);
  float s_prew[C][8], s_postw[C][8];
  float s_preb[LAYER ? C : 1][8], s_postb[LAYER ? C : 1][8], s_gate[GATE ? C : 1][8];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s_prew[c][j] = s_postw[c][j] = 0.f;
      if (LAYER) s_preb[c][j] = s_postb[c][j] = 0.f;
      if (GATE) s_gate[c][j] = 0.f;
    }
  const bool pre = a.pre && a.dh;
  int it = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + grp; row < a.M; row += (int64_t)gridDim.x * kRows, it ^= 1) {
    float* rd = red[it];  // two sets in turn: a wave may be one row ahead of another, never two
    Vec8<E> y[C], dh[C], gf[C];
    Vec8<R> x[C], dr[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      y[c] = at.load(c, (const E*)a.y + row * a.ldy);
      if (pre) {
        x[c] = at.load(c, (const R*)a.x + row * a.ldx);
        dh[c] = at.load(c, (const E*)a.dh + row * a.lddh);
      }
      if (a.dr) dr[c] = at.load(c, (const R*)a.dr + row * a.lddr);
      if (!GATE && a.gate_kind == kGateFull) gf[c] = at.load(c, (const E*)a.gate + row * a.ldg);
    }
    const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
    float grow = 1.f;
    if (!GATE && a.gate_kind == kGateRow) {
      grow = ((const float*)a.gate)[row];
      if (a.sigmoid) grow = sigmoid(grow);
    }
    // the forward again: un = normalised y, d = keep(u) up, r = x_scale x + y_scale gv d, n = normalised r
    float un[C][8], gv[C][8], d[C][8], t[C][8];
    uint32_t keep[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      keep[c] = a.mask.thr ? keep8(row * a.D + at.col[c], sd.seed, sd.offset, a.mask.thr) : 0xffu;
#pragma unroll
      for (int j = 0; j < 8; ++j) un[c][j] = d[c][j] = (float)y[c][j];
      if (a.post) {
        const Vec8<float> w = at.load(c, a.post_w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          un[c][j] = (un[c][j] - st.x) * st.y;
          d[c][j] = un[c][j] * w[j];
        }
        if (LAYER && a.post_b) {
          const Vec8<float> b = at.load(c, a.post_b);
#pragma unroll
          for (int j = 0; j < 8; ++j) d[c][j] += b[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) d[c][j] = (keep[c] >> j & 1) ? d[c][j] * a.mask.up : 0.f;
      if (GATE) {
        const Vec8<float> g = at.load(c, (const float*)a.gate);
#pragma unroll
        for (int j = 0; j < 8; ++j) gv[c][j] = a.sigmoid ? sigmoid(g[j]) : g[j];
      } else if (a.gate_kind == kGateFull) {
#pragma unroll
        for (int j = 0; j < 8; ++j) gv[c][j] = a.sigmoid ? sigmoid((float)gf[c][j]) : (float)gf[c][j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) gv[c][j] = grow;
      }
    }
    // t = dr + norm_pre'(dh)
    if (pre) {
      float n[C][8];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const Vec8<float> w = at.load(c, a.pre_w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float r = a.x_scale * (float)x[c][j] + a.y_scale * (gv[c][j] * d[c][j]), g = (float)dh[c][j];
          n[c][j] = (r - st.z) * st.w;
          s_prew[c][j] += g * n[c][j];
          if (LAYER) s_preb[c][j] += g;
          t[c][j] = g * w[j];
        }
      }
      norm_back<L, C, N>(t, n, at, a.pre, st.w, rd);
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) t[c][j] = 0.f;
    }
    float gdot = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float g[8];
      if (a.dr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[c][j] += (float)dr[c][j];
      }
      if (a.dx) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = a.x_scale * t[c][j];
        at.store(c, (R*)a.dx + row * a.D, g);
      }
      // dgate = y_scale t d slope, du = y_scale t gv keep up
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        t[c][j] *= a.y_scale;
        g[j] = t[c][j] * d[c][j];
        if (a.sigmoid && (GATE || a.gate_kind != kGateRow)) g[j] *= gv[c][j] * (1.f - gv[c][j]);
        if (GATE) s_gate[c][j] += g[j];
        gdot += at.counts(c, j) ? g[j] : 0.f;
        t[c][j] = (keep[c] >> j & 1) ? t[c][j] * gv[c][j] * a.mask.up : 0.f;
        s_postw[c][j] += t[c][j] * un[c][j];
        if (LAYER) s_postb[c][j] += t[c][j];
      }
      if (!GATE && a.gate_kind == kGateFull && a.dgate) at.store(c, (E*)a.dgate + row * a.D, g);
      if (a.post) {
        const Vec8<float> w = at.load(c, a.post_w);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[c][j] *= w[j];
      }
    }
    if (!GATE && a.gate_kind == kGateRow && a.dgate) {
      gdot = row_sum<L>(gdot, rd + 32);
      if (lane == 0) ((float*)a.dgate)[row] = a.sigmoid ? gdot * grow * (1.f - grow) : gdot;
    }
    if (a.dy) {
      if (a.post) norm_back<L, C, N>(t, un, at, a.post, st.y, rd + 64);
#pragma unroll
      for (int c = 0; c < C; ++c) at.store(c, (E*)a.dy + row * a.D, t[c]);
    }
  }
  // slab row blockIdx.x: the wanted sums in the order of residual_nvec
  int v = 0;
  auto leave = [&](float (*s)[8], bool wanted) {
    if (!wanted) return;
    float* out = a.slab + ((int64_t)blockIdx.x * residual_nvec(a) + v) * a.D;
    ++v;
    if constexpr (kRows == 1) {
#pragma unroll
      for (int c = 0; c < C; ++c) at.store(c, out, s[c]);
    } else {
      static_assert(C == 1, "one chunk a thread");
      __syncthreads();
      if (at.any(0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) part[grp][at.col[0] + j] = s[0][j];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < L * 8 && i < a.D; i += 256) {
        float q = 0.f;
        for (int g = 0; g < kRows; ++g) q += part[g][i];
        out[i] = q;
      }
    }
  };
  leave(s_prew, a.dpre_w != nullptr);
  if (LAYER) leave(s_preb, a.dpre_b != nullptr);
  if (GATE) leave(s_gate, a.dgate != nullptr);
  leave(s_postw, a.dpost_w != nullptr);
  if (LAYER) leave(s_postb, a.dpost_b != nullptr);
}

template <int TR, int TT>
void residual_bwd(const ResidualArgs& a, int grid, hipStream_t s) {
  const bool layer = a.post == kNormLayer || a.pre == kNormLayer, gate = a.gate_kind == kGateChannel;
  by_width(a.D, [&](auto l, auto c, auto n) {
    constexpr int L = decltype(l)::value, C = decltype(c)::value;
    constexpr bool N = decltype(n)::value;
    const dim3 g(grid), b(L < 256 ? 256 : L);
    if (layer && gate) hipLaunchKernelGGL((k_residual_bwd<TR, TT, L, C, N, true, true>), g, b, 0, s, a);
    else if (layer) hipLaunchKernelGGL((k_residual_bwd<TR, TT, L, C, N, true, false>), g, b, 0, s, a);
    else if (gate) hipLaunchKernelGGL((k_residual_bwd<TR, TT, L, C, N, false, true>), g, b, 0, s, a);
    else hipLaunchKernelGGL((k_residual_bwd<TR, TT, L, C, N, false, false>), g, b, 0, s, a);
  });
}

}  // namespace
}  // namespace pbx
