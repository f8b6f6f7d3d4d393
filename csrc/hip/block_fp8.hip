// 8-bit fc: e4m3 operands with one power-of-two scale for each block of 128,
// hand-written for gfx950.
//
// Quantisation: a = largest finite |v| of the block, e the least exponent with
// a <= 448 * 2^e, code = e4m3(v * 2^-e) rounded to the nearest, halves to
// even.  The scale is a power of two, so v * 2^-e is exact and the code holds
// the one rounding there is (half a step, 2^-4 of the value); what it costs
// against a free scale is at most one bit at the small end of the block's
// range, never precision.  Values that are not finite become NaN codes.
//
// Product, bfloat16 results: v_mfma_scale_f32_16x16x128_f8f6f4 (few rows) and
// 32x32x64 (tiles) take an exponent byte for each 32 values of either operand;
// equal bytes are one block of 128, so the instruction applies the scales with
// no vector work beside it, and a block is one or two of them deep.  Inside the
// instruction each run of 8 products is aligned to its largest and what lies
// more than 13 bits below that is dropped (measured; runs are added in full
// fp32).  So each of a run's seven other products loses less than 2^-13 of the
// largest, and a sum at most 7 * 2^-13 = 2^-10.2 of the sum of its runs' largest
// products: under bfloat16's half step (2^-9 to 2^-8 of a value) unless the sum
// cancels, and far under the 2^-4 that the codes themselves are rounded by.
// That is 4.2 PFLOP/s from registers.
// float32 and float16 results: float16's half step (2^-12 to 2^-11) is smaller
// than that loss.  The codes become bf16 with their scale in registers
// (v_cvt_scalef32_pk_bf16_fp8; 4 significant bits fit) and go through
// the bf16 instructions of the same tiles, which drop nothing above 2^-23 (2.3
// PFLOP/s).
// A scale holds for all 128 values of its block, so any order of them within
// the instructions is right as long as both operands use the same.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "block_ops.h"

namespace pbx {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------- quantisation
// |v| as an integer that orders like it; 0 where v is not finite
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// exponent byte of a block whose largest finite |v| has these bits: with
// |v| = 1.f * 2^(E - 127), the least e such that 1.f * 2^(E-127) <= 1.75 * 2^(8+e)
__device__ __forceinline__ int scale_byte(uint32_t bits) {
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 0 ? 0 : e;
}
// 2^(127 - byte): bytes are 0 .. 247, so this is a normal number
__device__ __forceinline__ float inverse_scale(int byte) { return __builtin_bit_cast(float, (uint32_t)(254 - byte) << 23); }
__device__ __forceinline__ float scaled(float v, float inv) {
  return finite_bits(v) || v == 0.f ? v * inv : __builtin_bit_cast(float, 0x7fc00000u);
}
// four codes, the first in the low byte
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// Blocks along a row only: 16 lanes a block, 8 values a lane, every load and
// store whole.  One row of 1024 takes 2 us, a launch.
template <typename E>
__global__ __launch_bounds__(256) void k_fp8_quant_rows(Fp8QuantArgs a) {
  const int64_t nb = fp8_kp(a.K) / 128, sp = fp8_sp(a.K);
  const int64_t blk = grid_piece() * 16 + (threadIdx.x >> 4);
  if (blk >= a.M * nb) return;  // the same for the 16 lanes of a block
  const int lane = threadIdx.x & 15;
  const int64_t row = blk / nb, kb = blk % nb, col = kb * 128 + lane * 8;
  const int64_t left = a.K - col;
  float v[8];
  load8((const E*)a.x + row * a.ld + (left > 0 ? col : 0), left >= 8 ? 8 : left > 0 ? (int)left : 0, v);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, finite_bits(v[j]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
  const int byte = scale_byte(m);
  const float inv = inverse_scale(byte);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = scaled(v[j], inv);
  uint2 c{codes4(v[0], v[1], v[2], v[3]), codes4(v[4], v[5], v[6], v[7])};
  *reinterpret_cast<uint2*>(a.row_codes + row * nb * 128 + col) = c;
  if (lane == 0) {
    uint8_t* s = a.row_scales + row * sp;
    s[kb] = (uint8_t)byte;
    if (kb == nb - 1)
      for (int64_t i = nb; i < sp; ++i) s[i] = 127;
  }
}

// Eight consecutive values of a row as they lie in memory (16-bit types two to
// a dword), and what the tile kernel does with them: magnitudes as integers
// that order like them, and codes straight from the stored type, with the
// scale in the conversion (v_cvt_scalef32_pk_fp8_*: v / scale, rounded to the
// nearest, halves to even; what is not finite becomes NaN).
template <typename E>
struct Eight {
  typedef E vec8 __attribute__((ext_vector_type(8), aligned(sizeof(E))));
  typedef E pair __attribute__((ext_vector_type(2)));
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  static constexpr bool WIDE = sizeof(E) == 4;
  static constexpr int NM = WIDE ? 8 : 4;  // dwords
  typedef uint32_t dwords __attribute__((ext_vector_type(NM)));
  dwords d;
  __device__ __forceinline__ void load(const E* p) { d = __builtin_bit_cast(dwords, *reinterpret_cast<const vec8*>(p)); }
  // `valid` values of them; the others come from the first address and count as 0
  __device__ __forceinline__ void load(const E* p, int valid) {
#pragma unroll
    for (int k = 0; k < NM; ++k) {
      if constexpr (WIDE) {
        const uint32_t x = __builtin_bit_cast(uint32_t, p[k < valid ? k : 0]);
        d[k] = k < valid ? x : 0u;
      } else {
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
        const uint32_t lo = q[2 * k < valid ? 2 * k : 0], hi = q[2 * k + 1 < valid ? 2 * k + 1 : 0];
        d[k] = (2 * k < valid ? lo : 0u) | (2 * k + 1 < valid ? hi << 16 : 0u);
      }
    }
  }
  __device__ __forceinline__ void only_if(bool keep) {
#pragma unroll
    for (int k = 0; k < NM; ++k) d[k] = keep ? d[k] : 0u;
  }
  __device__ __forceinline__ float value(int j) const {
    if constexpr (WIDE) return __builtin_bit_cast(float, (uint32_t)d[j]);
    else return (float)__builtin_bit_cast(pair, (uint32_t)d[j / 2])[j & 1];
  }
  __device__ __forceinline__ uint32_t mag(int k) const { return d[k] & (WIDE ? 0x7fffffffu : 0x7fff7fffu); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    if constexpr (WIDE) {
      return max(a, b);
    } else {
      const u16x2 x = __builtin_bit_cast(u16x2, a), y = __builtin_bit_cast(u16x2, b);
      return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
    }
  }
  // the larger half of a dword of magnitudes, and its bits as fp32
  static __device__ __forceinline__ uint32_t top(uint32_t m) { return WIDE ? m : max(m & 0xffffu, m >> 16); }
  static constexpr uint32_t kInf = WIDE ? 0x7f800000u : std::is_same<E, __bf16>::value ? 0x7f80u : 0x7c00u;
  static __device__ __forceinline__ uint32_t bits(uint32_t m) {
    if constexpr (WIDE) return m;
    else if constexpr (std::is_same<E, __bf16>::value) return m << 16;
    else return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, (unsigned short)m));
  }
  // a dword of magnitudes without those that are not finite
  static __device__ __forceinline__ uint32_t finite(uint32_t m) {
    if constexpr (WIDE) return m < kInf ? m : 0u;
    else return ((m & 0xffffu) < kInf ? m & 0xffffu : 0u) | ((m >> 16) < kInf ? m & 0xffff0000u : 0u);
  }
  // codes of two pairs of values, a pair as two dwords of fp32 or the halves of one
  static __device__ __forceinline__ uint32_t codes(uint32_t a, uint32_t b, uint32_t c, uint32_t e, float scale) {
    s16x2 r{0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __builtin_bit_cast(float, a), __builtin_bit_cast(float, b), scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, __builtin_bit_cast(float, c), __builtin_bit_cast(float, e), scale, true);
    return __builtin_bit_cast(uint32_t, r);
  }
  static __device__ __forceinline__ uint32_t codes(uint32_t ab, uint32_t ce, float scale) {
    s16x2 r{0, 0};
    if constexpr (std::is_same<E, __bf16>::value) {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(pair, ab), scale, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(pair, ce), scale, true);
    } else {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(pair, ab), scale, false);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(pair, ce), scale, true);
    }
    return __builtin_bit_cast(uint32_t, r);
  }
  __device__ __forceinline__ uint2 row_codes(float scale) const {
    if constexpr (WIDE) return make_uint2(codes(d[0], d[1], d[2], d[3], scale), codes(d[4], d[5], d[6], d[7], scale));
    else return make_uint2(codes(d[0], d[1], scale), codes(d[2], d[3], scale));
  }
  // of column j of the four rows x[0 .. 3]
  static __device__ __forceinline__ uint32_t col_codes(const Eight* x, int j, float scale) {
    if constexpr (WIDE) {
      return codes(x[0].d[j], x[1].d[j], x[2].d[j], x[3].d[j], scale);
    } else {
      const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;  // the high or the low halves of two dwords
      return codes(__builtin_amdgcn_perm(x[1].d[j / 2], x[0].d[j / 2], sel),
                   __builtin_amdgcn_perm(x[3].d[j / 2], x[2].d[j / 2], sel), scale);
    }
  }
};
__device__ __forceinline__ float scale_of(int byte) { return __builtin_bit_cast(float, (uint32_t)byte << 23); }

// the largest over the 16 lanes of a row of the wave
__device__ __forceinline__ uint32_t max16(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));   // quad: 1 0 3 2
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));   // quad: 2 3 0 1
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, true));  // half row mirrored
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xf, 0xf, true));  // row mirrored
  return m;
}

// One 128 x 128 tile a workgroup, read once: codes in blocks along the rows
// and, transposed, along the columns, and partial column sums.  Thread t holds
// columns 8 (t % 16) .. + 7 of rows 8 (t / 16) .. + 7 as they were stored: a
// row's block is 16 lanes, and 8 rows of a column are 8 bytes of the
// transposed codes, put together through LDS so that whole 128-byte lines are
// written.  Bound by memory: 16384 x 4096 bf16 to both forms, 268 MB, takes
// 66 us (4.0 TB/s); 8192 x 400 fp32, one tile a CU, 11 us, the latency of its
// two trips through memory.
template <typename E>
__device__ __forceinline__ void quant_tile(const Fp8QuantArgs& a, int tile) {
  using X = Eight<E>;
  __shared__ __attribute__((aligned(16))) uint8_t cols[128 * 128];
  __shared__ __attribute__((aligned(16))) uint32_t red[4][X::NM * 16];
  __shared__ uint32_t wave_max[4];
  const int kbs = (int)(fp8_kp(a.K) / 128), mbs = (int)(fp8_kp(a.M) / 128), bx = tile % kbs, by = tile / kbs;
  const int64_t k0 = (int64_t)bx * 128, m0 = (int64_t)by * 128;
  const int t = threadIdx.x, cl = t & 15, g = t >> 4, c0 = cl * 8, wave = t >> 6;
  const int64_t rows = a.M - m0, width = a.K - k0;
  const int64_t kp = fp8_kp(a.K), ksp = fp8_sp(a.K), mp = fp8_kp(a.M), msp = fp8_sp(a.M);
  const int valid = width - c0 >= 8 ? 8 : width - c0 > 0 ? (int)(width - c0) : 0;
  X x[8];
  // loads without a branch between them; rows and columns past the end read the last row and the first column
  const E* from = (const E*)a.x + m0 * a.ld + k0 + (valid ? c0 : 0);
  if (width >= 128 || width % 8 == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i].load(from + min((int64_t)(g * 8 + i), rows - 1) * a.ld);
    if (rows < 128 || width < 128) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i].only_if(g * 8 + i < rows && valid);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i].load(from + min((int64_t)(g * 8 + i), rows - 1) * a.ld, g * 8 + i < rows ? valid : 0);
  }
  if (a.slab) {
    float* part = reinterpret_cast<float*>(cols);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += x[i].value(j);
      part[g * 128 + c0 + j] = s;
    }
    __syncthreads();
    if (t < 128 && t < width) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += part[i * 128 + t];
      a.slab[(int64_t)by * a.K + k0 + t] = s;
    }
    __syncthreads();
  }
  // largest magnitudes of this thread's rows and columns; once more without what is not finite, where there is any
  uint32_t rm[8], cm[X::NM];
  auto largest = [&](auto f) {
#pragma unroll
    for (int k = 0; k < X::NM; ++k) cm[k] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < X::NM; ++k) {
        const uint32_t q = f(x[i].mag(k));
        m = X::larger(m, q);
        cm[k] = X::larger(cm[k], q);
      }
      rm[i] = X::top(m);
    }
  };
  largest([](uint32_t m) { return m; });
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) all = max(all, rm[i]);
  if (__any(all >= X::kInf)) {
    largest([](uint32_t m) { return X::finite(m); });
    all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) all = max(all, rm[i]);
  }
  int tile_byte = 0;
  if (a.tile) {
    uint32_t m = max16(all);
    m = max(m, (uint32_t)__shfl_xor((int)m, 16));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32));
    if ((t & 63) == 0) wave_max[wave] = m;
    __syncthreads();
    tile_byte = scale_byte(X::bits(max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]))));
  }
  if (a.row_codes) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int byte = a.tile ? tile_byte : scale_byte(X::bits(max16(rm[i])));
      const int r = g * 8 + i;
      if (r >= rows) continue;  // the same for the 16 lanes of a row
      const float scale = scale_of(byte);
      *reinterpret_cast<uint2*>(a.row_codes + (m0 + r) * kp + k0 + c0) = x[i].row_codes(scale);
      if (cl == 0) {
        uint8_t* s = a.row_scales + (m0 + r) * ksp;
        s[bx] = (uint8_t)byte;
        if (bx == kbs - 1)
          for (int64_t q = kbs; q < ksp; ++q) s[q] = 127;
      }
    }
  }
  if (a.col_codes) {
    if (!a.tile) {
#pragma unroll
      for (int k = 0; k < X::NM; ++k) {
        cm[k] = X::larger(cm[k], (uint32_t)__shfl_xor((int)cm[k], 16));
        cm[k] = X::larger(cm[k], (uint32_t)__shfl_xor((int)cm[k], 32));
      }
      if ((t & 63) < 16) {
#pragma unroll
        for (int k = 0; k < X::NM; ++k) red[wave][cl * X::NM + k] = cm[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < X::NM; ++k) {
        const int q = cl * X::NM + k;
        cm[k] = X::larger(X::larger(red[0][q], red[1][q]), X::larger(red[2][q], red[3][q]));
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int byte = a.tile ? tile_byte
                              : scale_byte(X::bits(X::WIDE ? cm[X::WIDE ? j : 0] : cm[j / 2 % X::NM] >> (16 * (j & 1)) & 0xffffu));
      const float scale = scale_of(byte);
      const int c = c0 + j;
      // 16-byte piece g / 2 of column c, pieces turned by the thread so that writes spread over the banks
      *reinterpret_cast<uint2*>(cols + c * 128 + ((g >> 1 ^ cl) & 7) * 16 + (g & 1) * 8) =
          make_uint2(X::col_codes(x, j, scale), X::col_codes(x + 4, j, scale));
      if (g == 0 && c < width) {
        uint8_t* s = a.col_scales + (k0 + c) * msp;
        s[by] = (uint8_t)byte;
        if (by == mbs - 1)
          for (int64_t q = mbs; q < msp; ++q) s[q] = 127;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = i * 256 + t, c = p >> 3, w = p & 7;
      if (c < width)
        *reinterpret_cast<uint4*>(a.col_codes + (k0 + c) * mp + m0 + w * 16) =
            *reinterpret_cast<const uint4*>(cols + c * 128 + ((w ^ c >> 3) & 7) * 16);
    }
  }
}

template <typename E>
__global__ __launch_bounds__(256, sizeof(E) == 4 ? 3 : 4) void k_fp8_quant_tile(Fp8QuantArgs a) {
  quant_tile<E>(a, blockIdx.x);
}
// two matrices in one launch (the activations and the weight of a forward): the second one's tiles come behind
template <typename E, typename W>
__global__ __launch_bounds__(256, 3) void k_fp8_quant_two(Fp8QuantArgs a, Fp8QuantArgs w, int tiles) {
  if ((int)blockIdx.x < tiles) quant_tile<E>(a, blockIdx.x);
  else quant_tile<W>(w, blockIdx.x - tiles);
}

// ---------------------------------------------------------------- product
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// whether the sums of a result of this type go through the bf16 instructions
template <typename C>
constexpr bool kFullSums = !std::is_same<C, __bf16>::value;

// 32 codes of a row, as the instructions take them from a lane.  FULL: as
// bf16 values with the scale in them; else codes and the exponent byte.
template <bool FULL>
struct Frag;
template <>
struct Frag<false> {
  i32x8 v;
  int e;  // the byte is the low one
  __device__ __forceinline__ Frag() {}
  __device__ __forceinline__ Frag(i32x8 codes, uint32_t byte) : v(codes), e((int)byte) {}
};
template <>
struct Frag<true> {
  bf16x8 v[4];
  __device__ __forceinline__ Frag() {}
  __device__ __forceinline__ Frag(i32x8 codes, uint32_t byte) {
    const float scale = __builtin_bit_cast(float, byte << 23);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int w = codes[q * 2 + h];
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false),
                     b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true);
        v[q][4 * h] = a[0];
        v[q][4 * h + 1] = a[1];
        v[q][4 * h + 2] = b[0];
        v[q][4 * h + 3] = b[1];
      }
  }
};
// 16 x 16 outputs, 128 deep
__device__ __forceinline__ f32x4 mfma_blocks(const Frag<false>& a, const Frag<false>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, c, 0, 0, 0, a.e, 0, b.e);
}
__device__ __forceinline__ f32x4 mfma_blocks(const Frag<true>& a, const Frag<true>& b, f32x4 c) {
#pragma unroll
  for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], c, 0, 0, 0);
  return c;
}
// 32 x 32 outputs, 64 deep
__device__ __forceinline__ f32x16 mfma_blocks(const Frag<false>& a, const Frag<false>& b, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a.v, b.v, c, 0, 0, 0, a.e, 0, b.e);
}
__device__ __forceinline__ f32x16 mfma_blocks(const Frag<true>& a, const Frag<true>& b, f32x16 c) {
#pragma unroll
  for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v[q], b.v[q], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ i32x8 codes32(const uint8_t* lo, const uint8_t* hi) {
  return __builtin_shufflevector(*reinterpret_cast<const i32x4*>(lo), *reinterpret_cast<const i32x4*>(hi), 0, 1, 2, 3, 4,
                                 5, 6, 7);
}

template <typename C>
__device__ __forceinline__ void store4(C* p, int valid, f32x4 v) {
  typedef C vec __attribute__((ext_vector_type(4), aligned(sizeof(C))));
  if (valid >= 4) {
    vec x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (C)v[j];
    *reinterpret_cast<vec*>(p) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < valid) p[j] = (C)v[j];
  }
}
__device__ __forceinline__ f32x4 bias4(const float* b, int n, int N) {
  typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
  f32x4 v{0.f, 0.f, 0.f, 0.f};
  if (b && n + 4 <= N) {
    v = *reinterpret_cast<const vec*>(b + n);
  } else if (b) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n + j < N) v[j] = b[n + j];
  }
  return v;
}

// LDS-DMA of 16 bytes a lane from base + off; lane l lands at lds_byte + 16 l.
// The wait is the caller's: the compiler does not know of the load.
__device__ __forceinline__ void glds16(const uint8_t* base, uint32_t off, unsigned lds_byte) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(off), "s"(base), "s"(lds_byte)
               : "memory", "m0");
}
__device__ __forceinline__ unsigned lds_addr(const void* p) {
  return (unsigned)(uintptr_t)((const __attribute__((address_space(3))) char*)p);
}
__device__ __forceinline__ void glds4(const uint8_t* base, uint32_t off, unsigned lds_byte) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               :
               : "v"(off), "s"(base), "s"(lds_byte)
               : "memory", "m0");
}
// all loads, DMAs and LDS reads of this wave are done
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void block_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Output tile of WR x WC waves, each MT x NT instruction tiles of 32 x 32.  The
// instruction's rows are b's (columns of the output), its columns a's: a lane
// then holds runs of 4 consecutive outputs of one row.
//
// LDS holds two blocks of K (BM + BN rows of 128 bytes each), filled by
// LDS-DMA in whole lines (rows of 64 bytes at a time took twice the requests
// of the L2 and bounded the kernel).  A block is used in two halves of 64:
// while one half's instructions run, the next one's fragments come from LDS
// into registers.  Before the last row of the first half's instructions all
// waves have the second half's fragments and the next block has landed: one
// barrier a block, there, frees this block's place for the block after the
// next, whose DMA then has nearly a block's time to arrive.
//
// 16-byte piece p of row r sits at place p ^ ((r / 2) & 7): the 16 rows that a
// fragment read takes in one cycle then spread over all 64 banks; the DMA
// writes lanes in order, so the turn is made in the global address.  The
// exponent bytes come by DMA too, the dwords of four blocks at once and four
// blocks ahead.
//
// 8192^3 of random values to bf16 takes 430 to 500 us (2.2 to 2.6 PFLOP/s; the
// clock falls under this load, constant data take 359), to fp32 784 to 826 us and
// to float16 767 (1.33 to 1.43 PFLOP/s: bf16 instructions and the conversion
// beside them).  The matrix instructions and the power they draw bound it.  The
// 256 x 256 form spills 16 registers for 16-bit results, outside its inner loop,
// and none for fp32.
template <int WR, int WC, int MT, int NT>
struct Fp8Tile {
  static constexpr int kThreads = 64 * WR * WC, kRows = (WR * MT + WC * NT) * 32;
  __attribute__((aligned(16))) uint8_t lds[2 * kRows * 128];
  uint32_t words[2][kRows];
};
// workgroup `wg` of the g.ksplit slices of all tiles
template <int WR, int WC, int MT, int NT, typename C>
__device__ __forceinline__ void gemm_tile(const Fp8GemmArgs& g, Fp8Tile<WR, WC, MT, NT>& shared, int wg) {
  constexpr bool FULL = kFullSums<C>;
  using F = Frag<FULL>;
  constexpr int BM = WR * MT * 32, BN = WC * NT * 32, W = WR * WC, ROWS = BM + BN, BLOCK = ROWS * 128;
  auto& lds = shared.lds;
  auto& words = shared.words;
  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wr = w / WC, wc = w % WC;
  // the 8 XCDs take workgroups in turn: give each a run of tiles, 8 rows of tiles deep, that share operands in its L2
  const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN, tiles = tm * tn;
  const int slice = wg / tiles, at = wg % tiles, q = tiles / 8, rr = tiles % 8, xcd = at % 8;
  const int id = (xcd < rr ? xcd * (q + 1) : rr * (q + 1) + (xcd - rr) * q) + at / 8;
  const int band = id / (8 * tn), deep = min(8, tm - band * 8), in = id - band * 8 * tn;
  const int m0 = (band * 8 + in % deep) * BM, n0 = in / deep * BN;
  const int64_t kp = fp8_kp(g.K), sp = fp8_sp(g.K);
  const int nb = (int)(kp / 128), per = fp8_slice(nb, g.ksplit);
  const int kb0 = slice * per, kb1 = min(nb, kb0 + per);  // kb0 is a multiple of 4; no slice is empty
  constexpr int LA = BM / 8 / W, LB = BN / 8 / W;              // DMAs of 8 rows a wave and block
  static_assert(BM % (8 * W) == 0 && BN % (8 * W) == 0, "whole loads");
  constexpr int LS = ROWS / 64 / W;  // DMAs of 64 dwords a wave and four blocks
  static_assert(BM == BN && W % 2 == 0 && ROWS % (64 * W) == 0, "a wave's dwords are all of one operand");
  const uint8_t *ga = g.a + m0 * kp, *gb = g.b + n0 * kp;
  uint32_t offa[LA], offb[LB], offs[LS];
  const int lr = lane >> 3, piece = ((lane & 7) ^ ((w & 1) * 4 + (lr >> 1))) * 16;  // a wave's rows begin at 8 w, mod 16
  // rows past the end read the last one: their outputs are not stored
#pragma unroll
  for (int i = 0; i < LA; ++i) offa[i] = (uint32_t)(min((i * W + w) * 8 + lr, g.M - 1 - m0) * kp) + piece;
#pragma unroll
  for (int i = 0; i < LB; ++i) offb[i] = (uint32_t)(min((i * W + w) * 8 + lr, g.N - 1 - n0) * kp) + piece;
  const bool of_b = w >= W / 2;
  const uint8_t* gs = of_b ? g.sb + n0 * sp : g.sa + m0 * sp;
#pragma unroll
  for (int i = 0; i < LS; ++i)
    offs[i] = (uint32_t)(min((w % (W / 2) * LS + i) * 64 + lane, (of_b ? g.N - n0 : g.M - m0) - 1) * sp);
  const unsigned base = lds_addr(lds) + w * 1024, base_s = lds_addr(words) + w * LS * 256;
  auto fill_part = [&](int buf, int kb, int i) {  // DMA i of a block's; past the last block: that one again, unused
    const int at = min(kb, kb1 - 1) * 128;
    if (i < LA) glds16(ga + at, offa[i], base + buf * BLOCK + i * W * 1024);
    else glds16(gb + at, offb[i - LA], base + buf * BLOCK + BM * 128 + (i - LA) * W * 1024);
  };
  auto fill = [&](int buf, int kb) {
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) fill_part(buf, kb, i);
  };
  auto fill_words = [&](int kb) {  // of the four blocks that kb begins
#pragma unroll
    for (int i = 0; i < LS; ++i) glds4(gs + min(kb, kb1 - 1) / 4 * 4, offs[i], base_s + (kb >> 2 & 1) * (ROWS * 4) + i * 256);
  };
  const int fr = lane & 31, fh = lane >> 5;
  uint32_t sa[MT], sb[NT];
  auto read_words = [&](int kb) {
#pragma unroll
    for (int i = 0; i < MT; ++i) sa[i] = words[kb >> 2 & 1][(wr * MT + i) * 32 + fr];
#pragma unroll
    for (int j = 0; j < NT; ++j) sb[j] = words[kb >> 2 & 1][BM + (wc * NT + j) * 32 + fr];
  };
  f32x16 acc[MT][NT];  // the sums begin with the bias: it costs nothing behind the first DMAs, and 3 us a tile at the end
  const float* bias = g.ksplit == 1 ? g.bias : nullptr;
  auto begin = [&]() {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 v = bias4(bias, n0 + (wc * NT + j) * 32 + r * 8 + fh * 4, g.N);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][4 * r + e] = v[e];
      }
  };
  i32x8 fa[2][MT], fb[2][NT];  // of the two halves
  const uint8_t *fbase = lds + (wr * MT * 32 + fr) * 128, *gbase = lds + (BM + wc * NT * 32 + fr) * 128;
  int pos[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) pos[h][e] = ((h * 4 + fh * 2 + e) ^ (fr >> 1 & 7)) * 16;
  auto read_part = [&](int buf, int h, int l) {  // fragment l of a half's: b's first, all of them are needed at once
    const uint8_t* p = l < NT ? gbase + l * 32 * 128 : fbase + (l - NT) * 32 * 128;
    (l < NT ? fb[h][l < NT ? l : 0] : fa[h][l < NT ? 0 : l - NT]) =
        codes32(p + buf * BLOCK + pos[h][0], p + buf * BLOCK + pos[h][1]);
  };
  auto have = [&](int h) {  // the compiler's wait for these fragments falls here
#pragma unroll
    for (int j = 0; j < NT; ++j) asm volatile("" : "+v"(fb[h][j]));
#pragma unroll
    for (int i = 0; i < MT; ++i) asm volatile("" : "+v"(fa[h][i]));
  };
  constexpr int LOADS = LA + LB, FRAGS = MT + NT;
  // rows [from, to) of half h's instructions; after row i reads share(i) of the fragments of (buf, half) and starts
  // share(i) of the DMAs, both counted in `gaps` equal shares from row `from`
  auto rows = [&](const F(&b)[NT], int h, int sh, int from, int to, auto between) {
    F a(fa[h][from], sa[from] >> sh & 0xffu);
#pragma unroll
    for (int i = from; i < to; ++i) {
      F next = a;
      if (i + 1 < to) next = F(fa[h][i + 1], sa[i + 1] >> sh & 0xffu);
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mfma_blocks(b[j], a, acc[i][j]);
      if (FULL && i + 1 < to) {  // the next row's codes become bf16 between this row's instructions
#pragma unroll
        for (int k = 0; k < 4 * NT; ++k) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      between(i);
      __builtin_amdgcn_sched_barrier(0);
      a = next;
    }
  };
  auto spread = [&](int i, int gaps, int n, auto f) {  // share i of n things in `gaps` equal shares
    if (i < gaps) {
#pragma unroll
      for (int l = i * n / gaps; l < (i + 1) * n / gaps; ++l) f(l);
    }
  };
  constexpr int GAPS = MT > 1 ? MT - 1 : 1, D0 = LOADS / MT;  // DMAs behind the barrier's row
  auto block = [&](int kb, int buf) {
    const int sh = (kb & 3) * 8;
    F b[NT];
    have(0);
#pragma unroll
    for (int j = 0; j < NT; ++j) b[j] = F(fb[0][j], sb[j] >> sh & 0xffu);
    rows(b, 0, sh, 0, MT - 1, [&](int i) { spread(i, MT > 2 ? MT - 2 : 1, FRAGS, [&](int l) { read_part(buf, 1, l); }); });
    wait_all();
    have(1);
    block_barrier();
    rows(b, 0, sh, MT - 1, MT, [&](int) { spread(0, 1, D0, [&](int l) { fill_part(buf, kb + 2, l); }); });
#pragma unroll
    for (int j = 0; j < NT; ++j) b[j] = F(fb[1][j], sb[j] >> sh & 0xffu);
    rows(b, 1, sh, 0, MT, [&](int i) {
      spread(i, GAPS, LOADS - D0, [&](int l) { fill_part(buf, kb + 2, D0 + l); });
      spread(i, GAPS, FRAGS, [&](int l) { read_part(buf ^ 1, 0, l); });
    });
  };
  fill_words(kb0);
  fill(0, kb0);
  fill(1, kb0 + 1);
  begin();
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
  block_barrier();
  read_words(kb0);
#pragma unroll
  for (int l = 0; l < FRAGS; ++l) read_part(0, 0, l);
  // the inner loop is one basic block: the compiler moves matrix instructions over a barrier to where a branch ends
  for (int kb = kb0; kb < kb1;) {
    const int end = min(kb + 4, kb1);
    fill_words(kb + 4);
    for (; kb < end; ++kb) block(kb, kb - kb0 & 1);
    read_words(kb);
  }
  wait_all();  // no DMA may outlive its use of LDS
  block_barrier();
  // A wave turns its tile through its own part of LDS, so that rows leave in whole lines: 16-byte piece p of row r at
  // place p ^ r (as far as there are pieces), which spreads both ways over the banks.
  auto leave = [&](auto out) {
    typedef decltype(out) O;
    typedef O vec __attribute__((ext_vector_type(16 / sizeof(O)), aligned(sizeof(O))));
    typedef O vec4 __attribute__((ext_vector_type(4)));
    constexpr int PER = 16 / sizeof(O), PIECES = NT * 32 / PER, PART = 2 * BLOCK / W;
    constexpr int TILES = PART / (PIECES * 16) / 32 < MT ? PART / (PIECES * 16) / 32 : MT;  // instruction tiles at a time
    static_assert(TILES >= 1 && MT % TILES == 0 && 64 % PIECES == 0, "whole passes");
    uint8_t* mine = lds + w * PART;
    O* c = g.ksplit > 1 ? (O*)(g.slab + (int64_t)slice * g.M * g.N) : (O*)g.c;
    const int nw = n0 + wc * NT * 32;
#pragma unroll
    for (int i0 = 0; i0 < MT; i0 += TILES) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = i * 32 + fr, col = j * 32 + r * 8 + fh * 4;
            const f32x4 v{acc[i0 + i][j][4 * r], acc[i0 + i][j][4 * r + 1], acc[i0 + i][j][4 * r + 2], acc[i0 + i][j][4 * r + 3]};
            vec4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (O)v[e];
            *reinterpret_cast<vec4*>(mine + row * PIECES * 16 + ((col / PER) ^ (row & (PIECES - 1))) * 16 +
                                     col % PER * sizeof(O)) = x;
          }
      }
      const int mw = m0 + (wr * MT + i0) * 32;
#pragma unroll 4
      for (int q = 0; q < TILES * 32 * PIECES / 64; ++q) {
        const int row = q * (64 / PIECES) + lane / PIECES, piece = lane % PIECES, m = mw + row, n = nw + piece * PER;
        const vec x = *reinterpret_cast<const vec*>(mine + row * PIECES * 16 + (piece ^ (row & (PIECES - 1))) * 16);
        if (m >= g.M || n >= g.N) continue;
        O* p = c + (int64_t)m * g.N + n;
        if (n + PER <= g.N) {
          *reinterpret_cast<vec*>(p) = x;
        } else {
#pragma unroll
          for (int e = 0; e < PER; ++e)
            if (n + e < g.N) p[e] = x[e];
        }
      }
    }
  };
  if (g.ksplit > 1) leave(float(0));
  else leave(C(0));
}

template <int WR, int WC, int MT, int NT, typename C>
__global__ __launch_bounds__(64 * WR * WC) void k_fp8_gemm(Fp8GemmArgs g) {
  __shared__ Fp8Tile<WR, WC, MT, NT> shared;
  gemm_tile<WR, WC, MT, NT, C>(g, shared, blockIdx.x);
}
// two products in one launch (a backward's dx and dW): neither fills the card alone
template <typename C, typename D>
__global__ __launch_bounds__(256) void k_fp8_gemm_two(Fp8GemmArgs g, Fp8GemmArgs h, int wgs) {
  __shared__ Fp8Tile<2, 2, 2, 2> shared;
  if ((int)blockIdx.x < wgs) gemm_tile<2, 2, 2, 2, C>(g, shared, blockIdx.x);
  else gemm_tile<2, 2, 2, 2, D>(h, shared, blockIdx.x - wgs);
}

// c = sum of the slices in order (+ bias), 4 columns a thread (about 4 us, the
// slices come from the L2)
template <typename C>
__device__ __forceinline__ void join_slices(const Fp8GemmArgs& g, int64_t i) {
  const int64_t n4 = ((int64_t)g.N + 3) / 4;
  if (i >= n4 * g.M) return;
  const int64_t m = i / n4;
  const int n = (int)(i % n4) * 4;
  typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
  f32x4 s{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < g.ksplit; ++k) {
    const float* p = g.slab + ((int64_t)k * g.M + m) * g.N + n;
    if (n + 4 <= g.N) {
      s += *reinterpret_cast<const vec*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < g.N) s[j] += p[j];
    }
  }
  store4((C*)g.c + m * g.N + n, g.N - n, s + bias4(g.bias, n, g.N));
}
inline __host__ __device__ int64_t join_wgs(const Fp8GemmArgs& g) {
  return g.ksplit > 1 ? (((int64_t)g.N + 3) / 4 * g.M + 255) / 256 : 0;
}
template <typename C>
__global__ __launch_bounds__(256) void k_fp8_join(Fp8GemmArgs g) {
  join_slices<C>(g, (int64_t)blockIdx.x * 256 + threadIdx.x);
}
// what is left of a backward behind its products, in one launch: the slices of dx and of dW, and db = column sums of
// the quantiser's slab [rows][K], in an order of the rows' number alone (64 columns a workgroup, 4 waves)
template <typename C, typename D>
__global__ __launch_bounds__(256) void k_fp8_finish(Fp8GemmArgs g, Fp8GemmArgs h, const float* slab, int rows, int K,
                                                    float* db) {
  int64_t wg = blockIdx.x;
  if (wg < join_wgs(g)) return join_slices<C>(g, wg * 256 + threadIdx.x);
  wg -= join_wgs(g);
  if (wg < join_wgs(h)) return join_slices<D>(h, wg * 256 + threadIdx.x);
  wg -= join_wgs(h);
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = (int)wg * 64 + lane;
  float s[8] = {};
  if (c < K) {
    int r = w;
    for (; r + 28 < rows; r += 32)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += slab[(int64_t)(r + 4 * i) * K + c];
    for (; r < rows; r += 4) s[0] += slab[(int64_t)r * K + c];
  }
  red[w][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (w == 0 && c < K) db[c] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

// Up to 16 MT rows of a: the bytes of b are the cost, so they go straight to
// registers, three blocks ahead (1 x 8192 x 8192: 16.8 us, 4.0 TB/s).  A
// workgroup takes 16 rows of b; its 8 waves share the blocks of K and join
// their sums through LDS in order.
template <int MT, typename C>
__global__ __launch_bounds__(512) void k_fp8_skinny(Fp8GemmArgs g) {
  using F = Frag<kFullSums<C>>;
  constexpr int AHEAD = 3;
  __shared__ f32x4 part[8][MT][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, fr = lane & 15, fg = lane >> 4;
  const int64_t kp = fp8_kp(g.K), sp = fp8_sp(g.K);
  const int nb = (int)(kp / 128), b0 = (int)((int64_t)nb * w / 8), b1 = (int)((int64_t)nb * (w + 1) / 8);
  const int n0 = blockIdx.x * 16;
  // a lane's 32 codes of a block are two 16-byte pieces, so that each load takes 64 bytes of a row
  const int64_t row_b = min(n0 + fr, g.N - 1);
  const uint8_t *pb = g.b + row_b * kp + fg * 16, *psb = g.sb + row_b * sp;
  const uint8_t *pa[MT], *psa[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t r = min(i * 16 + fr, g.M - 1);
    pa[i] = g.a + r * kp + fg * 16;
    psa[i] = g.sa + r * sp;
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  i32x8 va[AHEAD][MT], vb[AHEAD];
  uint8_t ea[AHEAD][MT], eb[AHEAD];
  auto load = [&](int at, int kb) {
    const int64_t off = (int64_t)kb * 128;
    vb[at] = codes32(pb + off, pb + off + 64);
    eb[at] = psb[kb];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      va[at][i] = codes32(pa[i] + off, pa[i] + off + 64);
      ea[at][i] = psa[i][kb];
    }
  };
#pragma unroll
  for (int u = 0; u < AHEAD; ++u)
    if (b0 + u < b1) load(u, b0 + u);
  for (int kb = b0; kb < b1; kb += AHEAD) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (kb + u >= b1) break;
      const F b(vb[u], eb[u]);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = mfma_blocks(b, F(va[u][i], ea[u][i]), acc[i]);
      if (kb + u + AHEAD < b1) load(u, kb + u + AHEAD);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) part[w][i][lane] = acc[i];
  __syncthreads();
  if (w < MT) {
    f32x4 s = part[0][w][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += part[k][w][lane];
    const int m = w * 16 + fr, n = n0 + fg * 4;
    if (m < g.M && n < g.N) store4((C*)g.c + (int64_t)m * g.N + n, g.N - n, s + bias4(g.bias, n, g.N));
  }
}

// the number of 16-row tiles as a constant
template <typename F>
void by_rows(int M, F f) {
  if (M <= 16) f(std::integral_constant<int, 1>{});
  else if (M <= 32) f(std::integral_constant<int, 2>{});
  else if (M <= 48) f(std::integral_constant<int, 3>{});
  else f(std::integral_constant<int, 4>{});
}

// Few rows of a go through k_fp8_skinny, one launch that streams b, unless b is large (every workgroup reads a) or so
// narrow that its workgroups are too few for a long K.  Both routes, us, bf16 results, b from memory (rows / tiles with
// their join; float16 results take up to 3 us more in tiles, the same in rows):
//    N x K          16 rows       24 rows       32 rows       48 rows       64 rows
//   1024 x 1024    3.3 /  8.7    3.7 /  8.6    3.9 /  8.5    4.7 /  7.7    5.3 /  8.7
//   4096 x 4096    9.0 / 14.8   10.7 / 15.2   11.7 / 15.6   14.7 / 16.9   17.5 / 18.0   (N K = 16 M: the last in rows)
//   4096 x 6144   11.3 / 17.3   12.8 / 17.7   14.0 / 18.0   17.6 / 18.9   21.3 / 19.3
//   8192 x 4096   14.4 / 16.7   18.9 / 16.8   20.8 / 17.0   27.2 / 17.9   32.5 / 18.4
//   8192 x 8192   25.5 / 24.5   33.2 / 24.5   36.9 / 24.9   48.5 / 25.7   59.2 / 26.4
//    512 x 4096    7.8 / 11.7    9.5 / 11.8   10.5 / 12.0   13.5 / 12.1   16.3 / 12.5   (the last K in rows)
//    512 x 8192   13.2 / 14.5   16.6 / 14.4   18.5 / 14.6   24.0 / 15.1   29.3 / 15.6
//   1024 x 8192   13.3 / 14.9   16.6 / 15.0   18.6 / 15.3   24.1 / 15.4   29.4 / 15.6   (the last N in rows)
// The rule is right on both sides of its borders for most of these; it loses up to 56% at 48 rows and 88% at 64 of
// 1024 x 8192, which a border at a few more columns or by rows times K would mend, and 38% at 24 rows of 4096 x 6144.
bool is_skinny(int M, int N, int64_t K) {
  if (M > 64 || (N < 1024 && K > 4096)) return false;
  return M <= 16 || (int64_t)N * K <= (int64_t)16 << 20;
}
// 256 x 256 tiles from the sizes where they fill three quarters of the card: 8192^3 to bf16 of constant data takes
// 359 us in them, 480 in 128 x 128
bool is_large(const Fp8GemmArgs& g) { return (int64_t)g.M * g.N >= (int64_t)256 * 256 * 192; }
int64_t small_tiles(const Fp8GemmArgs& g) { return (int64_t)((g.M + 127) / 128) * ((g.N + 127) / 128); }

// slices of K so that the tiles come to about `want` workgroups, at least 4 blocks each
int slices(int64_t tiles, int64_t K, int64_t want) {
  const int64_t nb = fp8_kp(K) / 128;
  int64_t split = want / tiles;
  if (split > nb / 4) split = nb / 4;
  if (split < 1) split = 1;
  const int per = fp8_slice((int)nb, (int)split);
  return (int)((nb + per - 1) / per);  // no empty slice
}

template <typename C>
void gemm(const Fp8GemmArgs& g, hipStream_t s) {
  if (is_skinny(g.M, g.N, g.K)) {
    by_rows(g.M, [&](auto mt) {
      hipLaunchKernelGGL((k_fp8_skinny<decltype(mt)::value, C>), dim3((unsigned)((g.N + 15) / 16)), dim3(512), 0, s, g);
    });
    return;
  }
  if (is_large(g)) {
    const dim3 grid((unsigned)((int64_t)((g.M + 255) / 256) * ((g.N + 255) / 256) * g.ksplit));
    hipLaunchKernelGGL((k_fp8_gemm<2, 2, 4, 4, C>), grid, dim3(256), 0, s, g);
  } else {
    hipLaunchKernelGGL((k_fp8_gemm<2, 2, 2, 2, C>), dim3((unsigned)(small_tiles(g) * g.ksplit)), dim3(256), 0, s, g);
  }
  if (g.ksplit > 1) hipLaunchKernelGGL(k_fp8_join<C>, dim3((unsigned)join_wgs(g)), dim3(256), 0, s, g);
}

template <typename F>
void by_type(BlockType t, F f) {
  if (t == kF32) f(float{});
  else if (t == kBF16) f(__bf16{});
  else f(_Float16{});
}
// a type and the same or fp32: what a weight may be beside its activations
template <typename F>
bool by_types(BlockType t, BlockType w, F f) {
  if (w != t && w != kF32) return false;
  by_type(t, [&](auto e) {
    if (w == kF32) f(e, float{});
    else f(e, e);
  });
  return true;
}

template <typename E>
void quant(const Fp8QuantArgs& a, hipStream_t s) {
  const int64_t kb = fp8_kp(a.K) / 128, mb = fp8_kp(a.M) / 128;
  if (!a.col_codes && !a.slab && !a.tile) {
    hipLaunchKernelGGL(k_fp8_quant_rows<E>, grid_of((a.M * kb + 15) / 16), dim3(256), 0, s, a);
    return;
  }
  hipLaunchKernelGGL(k_fp8_quant_tile<E>, dim3((unsigned)(kb * mb)), dim3(256), 0, s, a);
  if (a.colsum) launch_block_cols(a.slab, mb, a.K, &a.colsum, 1, a.K, s);
}

}  // namespace

int fp8_gemm_ksplit(int M, int N, int64_t K) {
  Fp8GemmArgs g;
  g.M = M;
  g.N = N;
  if (!M || !N || is_skinny(M, N, K) || is_large(g)) return 1;
  // joining slices is a launch of 4 us, about 8 blocks of K: 400 x 400 x 8192 to bf16 takes 34 us whole and 19 in slices,
  // 512 x 1024 x 1024 8.6 and 11.7
  const int split = slices(small_tiles(g), K, 256), nb = (int)(fp8_kp(K) / 128);
  return nb - fp8_slice(nb, split) >= 8 ? split : 1;
}

bool fp8_gemm_two_split(Fp8GemmArgs& g, Fp8GemmArgs& h) {
  if (is_large(g) || is_large(h) || g.M <= 64 || (h.ct != g.ct && h.ct != kF32)) return false;
  // two workgroups of 66 KB of LDS fit a CU; h (the long sum of dW) takes what g leaves of them
  g.ksplit = slices(small_tiles(g), g.K, 256);
  const int64_t left = 512 - small_tiles(g) * g.ksplit;
  h.ksplit = slices(small_tiles(h), h.K, left > 256 ? left : 256);
  return true;
}

void launch_fp8_gemm_two(const Fp8GemmArgs& g, const Fp8GemmArgs& h, const float* slab, int64_t rows, int64_t K, float* db,
                         hipStream_t s) {
  by_types(g.ct, h.ct, [&](auto c, auto d) {
    using C = decltype(c);
    using D = decltype(d);
    const int64_t n = small_tiles(g) * g.ksplit;
    hipLaunchKernelGGL((k_fp8_gemm_two<C, D>), dim3((unsigned)(n + small_tiles(h) * h.ksplit)), dim3(256), 0, s, g, h, (int)n);
    const int64_t left = join_wgs(g) + join_wgs(h) + (db ? (K + 63) / 64 : 0);
    if (left)
      hipLaunchKernelGGL((k_fp8_finish<C, D>), dim3((unsigned)left), dim3(256), 0, s, g, h, slab, (int)rows, (int)K, db);
  });
}

void launch_fp8_gemm(const Fp8GemmArgs& g, hipStream_t s) {
  if (g.M == 0 || g.N == 0) return;
  by_type(g.ct, [&](auto c) { gemm<decltype(c)>(g, s); });
}

void launch_fp8_quant(const Fp8QuantArgs& a, hipStream_t s) {
  if (a.M == 0 || a.K == 0) return;
  by_type(a.t, [&](auto e) { quant<decltype(e)>(a, s); });
}

void launch_fp8_quant_two(const Fp8QuantArgs& a, const Fp8QuantArgs& w, hipStream_t s) {
  const bool tiles = a.M && w.M && (a.col_codes || a.tile) && !a.slab && !w.slab;
  const int64_t n = fp8_kp(a.K) / 128 * (fp8_kp(a.M) / 128), m = fp8_kp(w.K) / 128 * (fp8_kp(w.M) / 128);
  // one launch for both where the backward wants x^T's codes too (forward with its quantisers: 8192 x 400 x 400 bf16 15.7
  // us, two launches 20.2; 16384 x 2048 x 2048 95 and 98), though a bf16 x beside an fp32 W then takes the fp32 body's
  // registers (151 a lane, alone 86); without gradients x goes by rows, in a launch of its own
  if (tiles && by_types(a.t, w.t, [&](auto e, auto f) {
        hipLaunchKernelGGL((k_fp8_quant_two<decltype(e), decltype(f)>), dim3((unsigned)(n + m)), dim3(256), 0, s, a, w, (int)n);
      }))
    return;
  launch_fp8_quant(w, s);
  launch_fp8_quant(a, s);
}

}  // namespace pbx
