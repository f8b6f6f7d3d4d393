// Launcher API and device helpers of the dense-block operators: the 8-bit
// block-scaled fc (block_fp8.hip), the gated residual norm and the
// counter-based dropout (block_norm.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#define PBX_FP8_HD __host__ __device__ inline

namespace pbx {

// element types of the dense-block operators
enum BlockType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// ---------------------------------------------------------------- counter-based mask
// Element i of a tensor (row-major, logical order) takes 16 bits of
// Philox4x32-10(counter = (i / 8, offset), key = seed): half-word i % 8, the
// low half of a word first.  It is dropped iff they are < thr = round(p 2^16);
// a kept value is scaled by 2^16 / (2^16 - thr).  16 bits an element: one
// block serves 8 elements, and p is a multiple of 2^-16.
struct MaskArgs {
  uint32_t thr = 0;               // 0: no dropout
  float up = 1.f;                 // scale of a kept value
  const int64_t* seed = nullptr;  // device (seed, offset), or null: the two values below
  int64_t seed_v = 0, offset_v = 0;
  int64_t* seed_out = nullptr;  // [2] the values used, for the backward pass (null: not wanted)
};

// y[i] = keep(i) ? x[i] * up : 0, n elements of one type
void launch_dropout(const void* x, void* y, int64_t n, BlockType t, const MaskArgs& m, hipStream_t s);

// out[v][c] = sum of slab[r][v D + c] over rows, v < nout <= 5, W = nout D
void launch_block_cols(const float* slab, int64_t rows, int64_t W, float* const* out, int nout, int64_t D, hipStream_t s);

// ---------------------------------------------------------------- gated residual norm
enum NormKind : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };
enum GateKind : int { kGateNone = 0, kGateChannel = 1, kGateRow = 2, kGateFull = 3 };

// A workgroup for each of `wgs` pieces, in two dimensions where one would pass
// the 2^32 threads that a launch may have there; surplus ones find no piece.
constexpr int64_t kGridX = 1 << 20;
inline dim3 grid_of(int64_t wgs) {
  return wgs <= kGridX ? dim3((unsigned)wgs) : dim3((unsigned)kGridX, (unsigned)((wgs + kGridX - 1) / kGridX));
}
#ifdef __HIPCC__
__device__ __forceinline__ int64_t grid_piece() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
#endif

struct ResidualArgs {
  int64_t M = 0;
  int D = 0;
  BlockType stream_t = kF32, t = kF32;  // x, r, dr, dx / y, h, dy, dh, full gate
  int post = 0, pre = 0, gate_kind = 0, sigmoid = 0;
  float x_scale = 1.f, y_scale = 1.f, eps = 0.f;
  MaskArgs mask;
  // row strides (elements) of the tensors that come from outside
  int64_t ldx = 0, ldy = 0, ldg = 0, lddr = 0, lddh = 0;
  const void* x = nullptr;
  const void* y = nullptr;
  const void* gate = nullptr;  // fp32 [D] / fp32 [M] / t [M, D]
  const float *post_w = nullptr, *post_b = nullptr, *pre_w = nullptr, *pre_b = nullptr;
  // forward
  void* r = nullptr;       // stream_t [M, D]
  void* h = nullptr;       // t [M, D], null without a pre norm
  float* stats = nullptr;  // [M][4]: post mean, post 1/dev, pre mean, pre 1/dev (null: not wanted)
  // backward
  const void* dr = nullptr;  // may be null: zero
  const void* dh = nullptr;  // may be null: zero
  void* dx = nullptr;        // any of the gradients may be null: not wanted
  void* dy = nullptr;
  void* dgate = nullptr;  // fp32 [D] / fp32 [M] / t [M, D]
  float *dpost_w = nullptr, *dpost_b = nullptr, *dpre_w = nullptr, *dpre_b = nullptr;
  float* slab = nullptr;  // [residual_slab_rows][nvec][D] partial column sums
};
// column sums the backward takes through the slab: pre weight, pre bias,
// channel gate, post weight, post bias, those of them that are wanted
__host__ __device__ inline int residual_nvec(const ResidualArgs& a) {
  return (a.dpre_w != nullptr) + (a.dpre_b != nullptr) + (a.gate_kind == kGateChannel && a.dgate != nullptr) +
         (a.dpost_w != nullptr) + (a.dpost_b != nullptr);
}
int residual_slab_rows(int64_t M, int D);
constexpr int kResidualMaxD = 16384;
void launch_residual_fwd(const ResidualArgs& a, hipStream_t s);
void launch_residual_bwd(const ResidualArgs& a, hipStream_t s);
// its kernel by types (stream and, where it differs, the rest)
void launch_residual_bwd_f32(const ResidualArgs& a, int grid, hipStream_t s);
void launch_residual_bwd_bf16(const ResidualArgs& a, int grid, hipStream_t s);
void launch_residual_bwd_f16(const ResidualArgs& a, int grid, hipStream_t s);
void launch_residual_bwd_f32_bf16(const ResidualArgs& a, int grid, hipStream_t s);
void launch_residual_bwd_f32_f16(const ResidualArgs& a, int grid, hipStream_t s);

// ---------------------------------------------------------------- 8-bit blocks
// A matrix [rows, K] held in e4m3 with one power-of-two scale for each block
// of 128 along K: codes [rows][Kp], Kp = K up to a multiple of 128 (padding
// zero), exponent bytes [rows][Sp], Sp = Kp / 128 up to a multiple of 4; byte
// e stands for 2^(e - 127).  A block scaled over 128 rows as well repeats its
// byte in each of them.
PBX_FP8_HD int64_t fp8_kp(int64_t K) { return (K + 127) / 128 * 128; }
PBX_FP8_HD int64_t fp8_sp(int64_t K) { return (fp8_kp(K) / 128 + 3) / 4 * 4; }

struct Fp8QuantArgs {
  const void* x = nullptr;  // [M, K], row stride ld
  BlockType t = kF32;
  int64_t M = 0, K = 0, ld = 0;
  int tile = 0;  // one scale for 128 x 128, both outputs alike
  uint8_t *row_codes = nullptr, *row_scales = nullptr;  // x in blocks along K: [M][fp8_kp(K)], [M][fp8_sp(K)]
  uint8_t *col_codes = nullptr, *col_scales = nullptr;  // x^T in blocks along M: [K][fp8_kp(M)], [K][fp8_sp(M)]
  float* slab = nullptr;    // [ceil(M / 128)][K]: column sums of x by tiles of rows
  float* colsum = nullptr;  // [K] fp32: their sums (null: the caller adds the slab up)
};
void launch_fp8_quant(const Fp8QuantArgs& a, hipStream_t s);
// activations and weight (in 128 x 128 blocks) of one layer, in one launch where their kernel is the same
void launch_fp8_quant_two(const Fp8QuantArgs& a, const Fp8QuantArgs& w, hipStream_t s);

struct Fp8GemmArgs {  // c [M, N] = a [M, K] b [N, K]^T (+ bias [N])
  const uint8_t *a = nullptr, *b = nullptr, *sa = nullptr, *sb = nullptr;
  int M = 0, N = 0;
  int64_t K = 0;  // logical: strides are fp8_kp(K), fp8_sp(K)
  const float* bias = nullptr;
  void* c = nullptr;
  BlockType ct = kF32;
  int ksplit = 1;         // slices of K; more than one goes through the slab
  float* slab = nullptr;  // [ksplit][M][N]
};
// blocks of a slice: a multiple of 4, as the exponent bytes' dwords are
PBX_FP8_HD int fp8_slice(int blocks, int ksplit) { return ((blocks + ksplit - 1) / ksplit + 3) / 4 * 4; }
int fp8_gemm_ksplit(int M, int N, int64_t K);
void launch_fp8_gemm(const Fp8GemmArgs& a, hipStream_t s);
// Two products of one layer's backward (dx, dW) in one launch, and a second one that joins their slices and sums db
// [K] from the quantiser's slab.  _split says whether they go together, and into how many slices each.
bool fp8_gemm_two_split(Fp8GemmArgs& g, Fp8GemmArgs& h);
void launch_fp8_gemm_two(const Fp8GemmArgs& g, const Fp8GemmArgs& h, const float* slab, int64_t rows, int64_t K, float* db,
                         hipStream_t s);

#ifdef __HIPCC__
// ---------------------------------------------------------------- device helpers
template <int T>
struct BlockElem;
template <>
struct BlockElem<kF32> {
  using type = float;
};
template <>
struct BlockElem<kBF16> {
  using type = __bf16;
};
template <>
struct BlockElem<kF16> {
  using type = _Float16;
};

// 8 consecutive elements; the address need only be aligned to the element
// (rows of odd width), and elements at and past `valid` read as 0 / stay
// unwritten.
template <typename E>
__device__ __forceinline__ void load8(const E* p, int valid, float v[8]) {
  typedef E vec __attribute__((ext_vector_type(8), aligned(sizeof(E))));
  if (valid >= 8) {
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)x[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < valid ? (float)p[j] : 0.f;
  }
}
template <typename E>
__device__ __forceinline__ void store8(E* p, int valid, const float v[8]) {
  typedef E vec __attribute__((ext_vector_type(8), aligned(sizeof(E))));
  if (valid >= 8) {
    vec x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (E)v[j];
    *reinterpret_cast<vec*>(p) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < valid) p[j] = (E)v[j];
  }
}

// Philox4x32-10: the counter-based generator of Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3" (2011).
__device__ __forceinline__ void philox4x32(uint64_t block, uint64_t offset, uint64_t seed, uint32_t w[4]) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}
// keep bits of elements i0 .. i0 + 7 (bit j: element i0 + j stays)
__device__ __forceinline__ uint32_t keep8(int64_t i0, uint64_t seed, uint64_t offset, uint32_t thr) {
  uint32_t w[4];
  philox4x32((uint64_t)i0 >> 3, offset, seed, w);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m |= ((w[j] & 0xffffu) >= thr ? 1u : 0u) << (2 * j);
    m |= ((w[j] >> 16) >= thr ? 1u : 0u) << (2 * j + 1);
  }
  const int sh = (int)(i0 & 7);
  if (sh) {  // rows of odd width: the elements straddle two blocks
    philox4x32(((uint64_t)i0 >> 3) + 1, offset, seed, w);
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      n |= ((w[j] & 0xffffu) >= thr ? 1u : 0u) << (2 * j);
      n |= ((w[j] >> 16) >= thr ? 1u : 0u) << (2 * j + 1);
    }
    m = (m | n << 8) >> sh;
  }
  return m & 0xffu;
}
#endif

}  // namespace pbx
