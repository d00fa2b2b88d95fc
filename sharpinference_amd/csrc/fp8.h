// Rows and weights in 8-bit floating point: e4m3 codes, and one power of two for every 128 values of a row.
//
// Format.  A row is cut into blocks of 128 values (the last one filled up with zeros).  A block's byte s, from 1 to 247, stands for the
// scale 2^(s - 127): the smallest with which the block's largest finite magnitude is at most 448, e4m3's largest value.  A value v is
// stored as e4m3(v 2^(127 - s)), to nearest, ties to even.  Both the byte and the scaled value come from exact arithmetic (an exponent
// read from the bits, a product by a power of two), so every kernel that quantises a row gives the same codes.  Infinities and NaN
// become e4m3's NaN and do not count for the scale.
//
// Why powers of two: v_mfma_scale_f32_*_f8f6f4 multiplies each operand row by such a byte (E8M0) itself, for every 32 of k.  The scales of a
// block of 128 then cost no instruction of their own and the sums stay in the accumulators; a scale of full precision would take a
// multiply-add per accumulator and block, and gains nothing where the values are floating point themselves.
//
// Accuracy of that instruction, measured: of eight products on end those some 2^-13 below the largest are cut, the groups of eight
// are added in float: 1.5e-5 of the result's rms for normal values.  Results are therefore offered as bfloat16 only.
//
// Layouts.  Rows [M]: codes row by row, 128 U bytes each (U blocks), bytes of scales row by row, 4 U4 each (U4 = U / 4 rounded up).
// Weights [N, K]: rows in tiles of 32 (filled up with zeros), tile by tile and block by block, 4 KB each in the order
// [half s of 64 k][piece p][group g][row r of 32][16 bytes], k = 64 s + 32 g + 16 p + byte: a wave's 16-byte loads of v_mfma 32x32x64's
// operand are one kilobyte on end, and those of 16x16x128 four runs of 256.  Their scales [tile][U4][row of 32][4 blocks].
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr int kF8Block = 128;                 // values that share a scale
constexpr int kF8Tile = 32;                   // weight rows of a tile
constexpr int kF8TileBytes = kF8Tile * kF8Block;
constexpr uint32_t kF8Nan = 0x7f;
constexpr int kF8MostK = 1 << 24;             // columns of a row at most.  (A tile's loads reach 2^32 - 1 bytes of codes: 256 rows of up to 2^24 - 128, 192 of all)

static inline __host__ __device__ int f8_blocks(int k) { return (k + kF8Block - 1) / kF8Block; }
static inline __host__ __device__ int f8_scale_stride(int k) { return (f8_blocks(k) + 3) & ~3; }     // bytes of a row's scales
static inline __host__ __device__ int f8_padded_rows(int n) { return (n + kF8Tile - 1) / kF8Tile * kF8Tile; }

// The block's byte from the bits of its largest finite magnitude (448 = 1.75 x 2^8).
__device__ __forceinline__ int f8_scale_of(uint32_t top_bits) {
  const int s = (int)(top_bits >> 23) - 8 + ((top_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return s < 1 ? 1 : s;
}
__device__ __forceinline__ float f8_scale_value(int s) { return __uint_as_float((uint32_t)s << 23); }
// A block's sum of products of codes, times the scales of both operands, whose bytes are given added up: one step of the exponent, whatever either scale is
// by itself.
__device__ __forceinline__ float f8_scaled(float sum, int bytes) { return __builtin_amdgcn_ldexpf(sum, bytes - 254); }

typedef __attribute__((ext_vector_type(2))) short s16x2_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2v_t;
// Four values' codes, of floats or of two pairs of bfloat16, divided by `scale` (a power of two).
__device__ __forceinline__ uint32_t f8_codes4(float a, float b, float c, float d, float scale) {
  s16x2_t v = {0, 0};
  v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(v, a, b, scale, false);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(v, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t f8_codes4(uint32_t lo, uint32_t hi, float scale) {
  s16x2_t v = {0, 0};
  v = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(v, __builtin_bit_cast(bf16x2v_t, lo), scale, false);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(v, __builtin_bit_cast(bf16x2v_t, hi), scale, true);
  return __builtin_bit_cast(uint32_t, v);
}
// act(g) u of a gated feed-forward whose result is rounded to bfloat16 and quantised: each of the activations is g times a logistic function
// (tanh-GELU's 0.5 (1 + tanh z) is that of 2 z), by the hardware's power of two and reciprocal: 2^-22 of the result, and 2^-23 |z| of it
// from the exponent, where the general exponential and division take some 30 instructions an element.
template <int ACT> __device__ __forceinline__ float f8_unit(float limit, float g, float u) {
  if constexpr (ACT == ACT_SWISH_CLAMP) {
    // (by comparisons: a NaN stays one, and with it the row of the result)
    g = g > limit ? limit : g;
    u = (u > limit ? limit : u < -limit ? -limit : u) + 1.0f;
  }
  const float z = ACT == ACT_SWISH_CLAMP ? kSwishSlope * g : ACT == ACT_GELU_TANH ? 1.5957691216057308f * (g + 0.044715f * g * g * g) : g;
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z)) * u;
}
__device__ __forceinline__ float f8_unit(GatedAct act, float g, float u) {
  if (act.code == ACT_SWISH_CLAMP) return f8_unit<ACT_SWISH_CLAMP>(act.limit, g, u);
  if (act.code == ACT_GELU_TANH) return f8_unit<ACT_GELU_TANH>(act.limit, g, u);
  return f8_unit<ACT_SILU>(act.limit, g, u);
}
