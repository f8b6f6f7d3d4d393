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
  float s[2] = {0.f, 0.f};  // of g n and, for the layer norm, of g
#pragma unroll
  for (int c = 0; c < C; ++c) {
    s[0] += at.sum(c, [&](int j) { return g[c][j] * n[c][j]; });
    if (kind == kNormLayer) s[1] += at.sum(c, [&](int j) { return g[c][j]; });
  }
  if (kind == kNormLayer) row_sums<L>(s, red);
  else s[0] = row_sum<L>(s[0], red);
  const float sgn = s[0] * at.per, sg = s[1] * at.per;
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
// took 180 registers a lane, one workgroup a CU, and twice the time.  ALL: both
// norms are there, all of dr, dh, dx and dy wanted: the conditions on them
// otherwise fill the scalar registers (32768 x 4096 bf16 with a channel gate:
// with ALL 455 us, without 525).
//
// Without a gate, 2^27 elements (us, TB/s of the 6 tensors that are read and
// written; a large copy 4.8, and up to 8 where some of it lies in the cache):
//                post rms, pre rms  none, rms       layer, layer    none, layer
//   bf16  2048   430 (3.8)          355 (4.5)       508 (3.2)       378 (4.3)
//         4096   359 (4.5)          341 (4.7)       516 (3.1)       391 (4.1)
//         5120   515 (3.1)          433 (3.7)       793 (2.0)      1043 (1.5)
//         8192   373 (4.3)          321 (5.0)       566 (2.9)       737 (2.2)
//        16384  1012 (1.6)         1127 (1.4)      2126 (0.8)      1520 (1.1)
//   fp32  4096   613 (5.3)          656 (4.9)       680 (4.7)       593 (5.4)
//         8192   616 (5.2)          589 (5.5)       936 (3.4)      1094 (2.9)
//        16384  1864 (1.7)         1621 (2.0)      2580 (1.3)      2338 (1.4)
// and 8192 x 400 fp32 with all inputs and a full gate 30.5 for 105 MB.
// Up to 4096 columns, and to 8192 without a layer norm, memory bounds it; the
// row's two reductions and their barriers cost the rest.  At 2049 to 4096
// columns rms norms alone fit two workgroups of 512 a CU (1 to 15 registers
// spilled); with a layer norm's bias sums there is one (154 to 173 registers).
// At 4097 to 8192 columns a layer norm spills 17 to 70 registers, over 8192, two
// chunks a lane of 1024 threads, every form 85 to 238: what they write and read
// again is the larger part of the time there.
template <int TR, int TT, int L, int C, bool N, bool LAYER, bool GATE, bool ALL>
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
  const bool pre = ALL || (a.pre && a.dh), post = ALL || a.post, has_dr = ALL || a.dr;
  const int pre_kind = LAYER ? a.pre : kNormRms, post_kind = LAYER ? a.post : kNormRms;  // where there is one
  // all loads of a row in one place, in front of its arithmetic
  struct Raw {
    Vec8<E> y[C], dh[C], gf[C];
    Vec8<R> x[C], dr[C];
    float4 st;
  };
  auto fetch = [&](Raw& v, int64_t row) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      v.y[c] = at.load(c, (const E*)a.y + row * a.ldy);
      if (pre) {
        v.x[c] = at.load(c, (const R*)a.x + row * a.ldx);
        v.dh[c] = at.load(c, (const E*)a.dh + row * a.lddh);
      }
      if (has_dr) v.dr[c] = at.load(c, (const R*)a.dr + row * a.lddr);
      if (!GATE && a.gate_kind == kGateFull) v.gf[c] = at.load(c, (const E*)a.gate + row * a.ldg);
    }
    v.st = reinterpret_cast<const float4*>(a.stats)[row];
  };
  const int64_t first = (int64_t)blockIdx.x * kRows + grp, step = (int64_t)gridDim.x * kRows;
  int it = 0;
  for (int64_t row = first; row < a.M; row += step, it ^= 1) {
    float* rd = red[it];  // two sets in turn: a wave may be one row ahead of another, never two
    Raw raw;
    fetch(raw, row);
    const auto &y = raw.y, &dh = raw.dh, &gf = raw.gf;
    const auto &x = raw.x, &dr = raw.dr;
    const float4 st = raw.st;
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
      if (post) {
        const Vec8<float> w = at.load(c, a.post_w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          un[c][j] = LAYER ? (un[c][j] - st.x) * st.y : un[c][j] * st.y;
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
          n[c][j] = LAYER ? (r - st.z) * st.w : r * st.w;
          s_prew[c][j] += g * n[c][j];
          if (LAYER) s_preb[c][j] += g;
          t[c][j] = g * w[j];
        }
      }
      norm_back<L, C, N>(t, n, at, pre_kind, st.w, rd);
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
      if (has_dr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[c][j] += (float)dr[c][j];
      }
      if (ALL || a.dx) {
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
        t[c][j] = (keep[c] >> j & 1) ? t[c][j] * gv[c][j] * a.mask.up : 0.f;
        s_postw[c][j] += t[c][j] * un[c][j];
        if (LAYER) s_postb[c][j] += t[c][j];
      }
      if (!GATE && a.gate_kind == kGateRow) gdot += at.sum(c, [&](int j) { return g[j]; });
      if (!GATE && a.gate_kind == kGateFull && a.dgate) at.store(c, (E*)a.dgate + row * a.D, g);
      if (post) {
        const Vec8<float> w = at.load(c, a.post_w);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[c][j] *= w[j];
      }
    }
    if (!GATE && a.gate_kind == kGateRow && a.dgate) {
      gdot = row_sum<L>(gdot, rd + 32);
      if (lane == 0) ((float*)a.dgate)[row] = a.sigmoid ? gdot * grow * (1.f - grow) : gdot;
    }
    if (ALL || a.dy) {
      if (post) norm_back<L, C, N>(t, un, at, post_kind, st.y, rd + 64);
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
  const bool all = a.post && a.pre && a.dr && a.dh && a.dx && a.dy;
  by_width(a.D, [&](auto l, auto c, auto n) {
    constexpr int L = decltype(l)::value, C = decltype(c)::value;
    constexpr bool N = decltype(n)::value;
    const dim3 g(grid), b(L < 256 ? 256 : L);
    auto go = [&](auto layer_t, auto gate_t) {
      constexpr bool LA = decltype(layer_t)::value, GA = decltype(gate_t)::value;
      if (all) hipLaunchKernelGGL((k_residual_bwd<TR, TT, L, C, N, LA, GA, true>), g, b, 0, s, a);
      else hipLaunchKernelGGL((k_residual_bwd<TR, TT, L, C, N, LA, GA, false>), g, b, 0, s, a);
    };
    if (layer && gate) go(std::true_type{}, std::true_type{});
    else if (layer) go(std::true_type{}, std::false_type{});
    else if (gate) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
  });
}

}  // namespace
}  // namespace pbx
