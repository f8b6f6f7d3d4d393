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

#include "block_norm_row.h"

namespace pbx {
namespace {

// One row to the L lanes that hold it, 8 columns each; nothing is shared
// between rows.  32768 x 4096 bf16: 1.07 GB in 236 to 262 us (4.1 to 4.5 TB/s,
// a large copy 4.8); 8192 x 400 fp32 with a full gate, a sigmoid, two layer
// norms and dropout: 66 MB in 18 us.
template <int TR, int TT, int L, int C, bool N>
__global__ __launch_bounds__(L < 256 ? 256 : L) void k_residual_fwd(ResidualArgs a) {
  using R = typename BlockElem<TR>::type;
  using E = typename BlockElem<TT>::type;
  constexpr int kRows = L < 256 ? 256 / L : 1;
  __shared__ float red[64];
  const Seed sd = mask_seed(a.mask);
  keep_seed(a.mask, sd);
  const int lane = threadIdx.x % L;
  const int64_t row = grid_piece() * kRows + threadIdx.x / L;
  if (row >= a.M) return;  // the same for every thread of a row
  const Columns<L, C, N> at(lane, a.D);
  Vec8<E> y[C];
  Vec8<R> x[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    y[c] = at.load(c, (const E*)a.y + row * a.ldy);
    x[c] = at.load(c, (const R*)a.x + row * a.ldx);
  }
  float u[C][8];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) u[c][j] = (float)y[c][j];
  float2 ps{0.f, 1.f}, qs{0.f, 1.f};
  if (a.post) {
    ps = normalise<L, C, N>(u, at, a.post, a.eps, red);
    affine<L, C, N>(u, at, a.post_w, a.post_b);
  }
  float grow = 1.f;
  if (a.gate_kind == kGateRow) {
    grow = ((const float*)a.gate)[row];
    if (a.sigmoid) grow = sigmoid(grow);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const uint32_t keep = a.mask.thr ? keep8(row * a.D + at.col[c], sd.seed, sd.offset, a.mask.thr) : 0xffu;
    float g[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = grow;
    if (a.gate_kind == kGateChannel) {
      const Vec8<float> v = at.load(c, (const float*)a.gate);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = a.sigmoid ? sigmoid(v[j]) : v[j];
    } else if (a.gate_kind == kGateFull) {
      const Vec8<E> v = at.load(c, (const E*)a.gate + row * a.ldg);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = a.sigmoid ? sigmoid((float)v[j]) : (float)v[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = (keep >> j & 1) ? u[c][j] * a.mask.up : 0.f;
      u[c][j] = a.x_scale * (float)x[c][j] + a.y_scale * (g[j] * d);
    }
    at.store(c, (R*)a.r + row * a.D, u[c]);
  }
  if (a.pre) {
    qs = normalise<L, C, N>(u, at, a.pre, a.eps, red + 32);
    affine<L, C, N>(u, at, a.pre_w, a.pre_b);
#pragma unroll
    for (int c = 0; c < C; ++c) at.store(c, (E*)a.h + row * a.D, u[c]);
  }
  if (a.stats && lane == 0) reinterpret_cast<float4*>(a.stats)[row] = float4{ps.x, ps.y, qs.x, qs.y};
}

struct ColOut {
  float* p[5];
};
// out[v][c] = sum over the slab's rows, in an order of their number alone: 64
// columns a workgroup, 16 waves take every 16th row, eight loads in flight
// (512 rows of 4096 x 3: 6 us; 4 waves with one load each took 22).
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

// 8 values a thread and step.  Reads and writes bound it, the mask's integer
// products run beside them: 32768 x 8192 bf16, 1.07 GB, in 215 to 222 us (4.8
// to 5.0 TB/s); 8192 x 400 fp32 in 8 us.
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

template <typename F>
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

}  // namespace

int residual_slab_rows(int64_t M, int D) {
  const int rows = D <= 128 ? 16 : D <= 512 ? 4 : 1;
  const int64_t need = (M + rows - 1) / rows;
  return (int)(need < 512 ? need : 512);  // two workgroups a CU
}

void launch_residual_fwd(const ResidualArgs& a, hipStream_t s) {
  if (a.M == 0 || a.D == 0) return;
  by_width(a.D, [&](auto l, auto c, auto n) {
    constexpr int L = decltype(l)::value, C = decltype(c)::value, rows = L < 256 ? 256 / L : 1;
    by_types(a, [&](auto tr, auto tt) {
      hipLaunchKernelGGL((k_residual_fwd<decltype(tr)::value, decltype(tt)::value, L, C, decltype(n)::value>),
                         grid_of((a.M + rows - 1) / rows), dim3(L < 256 ? 256 : L), 0, s, a);
    });
  });
}

void launch_residual_bwd(const ResidualArgs& a, hipStream_t s) {
  if (a.M == 0 || a.D == 0) return;
  const int grid = residual_slab_rows(a.M, a.D);
  if (a.stream_t != a.t) a.t == kBF16 ? launch_residual_bwd_f32_bf16(a, grid, s) : launch_residual_bwd_f32_f16(a, grid, s);
  else if (a.t == kF32) launch_residual_bwd_f32(a, grid, s);
  else if (a.t == kBF16) launch_residual_bwd_bf16(a, grid, s);
  else launch_residual_bwd_f16(a, grid, s);
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
