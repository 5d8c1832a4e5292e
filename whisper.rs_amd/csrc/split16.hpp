// Operands of the kernels that run f32 rows over f16 planes on the f16 matrix pipe: values
// split into f16 parts, and V rows that pass through a wave's own LDS.
#pragma once

#include "wrs_internal.hpp"

namespace wrs {
namespace split16 {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kWeightUp = 0x1p15f;  // softmax weights, at most 1, are split in units of its inverse

__device__ inline float pow2(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }
__device__ inline int clamp_exp(int e) { return e < -126 ? -126 : (e > 127 ? 127 : e); }

// 16-byte chunk c of V row r (128 bytes) sits at c ^ swz(r): rows 4i..4i+3
// reading an aligned chunk pair (the transposed reads) hit distinct banks.
__device__ inline int swz(int r) {
  return ((2 * (r & 3)) | ((r >> 2) & 1)) ^ (((r >> 3) & 1) << 1);
}
__device__ inline u32x2 read_tr(const char* p) {
  const uint32_t addr = static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
  return __builtin_bit_cast(u32x2,
                            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)addr));
}
// Two floats, times `scale` at most 2^15, as packed f16 pairs: two parts in one unit,
// whose last ends at f16's 2^-24, or three, part p in units of kPartUnit^p: what a
// part leaves is at most 2^-11 of the value, so the next one holds 11 bits more at
// the same magnitude.
constexpr float kPartUnit = 0x1p-11f;
// The pair is formed once (v_fma_mixlo, v_fma_mixhi): with nothing to hide its origin the
// compiler rounds each element again where the next part subtracts it (23 of the 285
// instructions of a two-part step, 41 of 472 with three).
__device__ inline f16x2 pack2(float x0, float x1, float scale) {
  const f16x2 h = {static_cast<_Float16>(__builtin_fmaf(x0, scale, 0.f)),
                   static_cast<_Float16>(__builtin_fmaf(x1, scale, 0.f))};
  uint32_t w = __builtin_bit_cast(uint32_t, h);
  asm("" : "+v"(w));
  return __builtin_bit_cast(f16x2, w);
}
__device__ inline void split2(float x0, float x1, float scale, uint32_t (&out)[2]) {
  const f16x2 h = pack2(x0, x1, scale);
  const f16x2 l = {
      static_cast<_Float16>(__builtin_fmaf(x0, scale, -static_cast<float>(h[0]))),
      static_cast<_Float16>(__builtin_fmaf(x1, scale, -static_cast<float>(h[1])))};
  out[0] = __builtin_bit_cast(uint32_t, h);
  out[1] = __builtin_bit_cast(uint32_t, l);
}
__device__ inline void split2(float x0, float x1, float scale, uint32_t (&out)[3]) {
  constexpr float kUp = 1.f / kPartUnit;
  const f16x2 h = pack2(x0, x1, scale);
  x0 = __builtin_fmaf(x0, scale, -static_cast<float>(h[0]));  // exact
  x1 = __builtin_fmaf(x1, scale, -static_cast<float>(h[1]));
  const f16x2 m = pack2(x0, x1, kUp);
  x0 = __builtin_fmaf(static_cast<float>(m[0]), -kPartUnit, x0);  // exact
  x1 = __builtin_fmaf(static_cast<float>(m[1]), -kPartUnit, x1);
  const f16x2 l = {static_cast<_Float16>(__builtin_fmaf(x0, kUp * kUp, 0.f)),
                   static_cast<_Float16>(__builtin_fmaf(x1, kUp * kUp, 0.f))};
  out[0] = __builtin_bit_cast(uint32_t, h);
  out[1] = __builtin_bit_cast(uint32_t, m);
  out[2] = __builtin_bit_cast(uint32_t, l);
}

__device__ inline f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// Two floats, times `scale` at most 2^15, as packed f16 pairs in two parts, the second in a unit
// 2^-11 of the first.
constexpr int kParts = 2;
__device__ inline void split_units(float x0, float x1, float scale, uint32_t (&out)[kParts]) {
  constexpr float kUp = 1.f / kPartUnit;
  const f16x2 h = pack2(x0, x1, scale);
  x0 = __builtin_fmaf(x0, scale, -static_cast<float>(h[0]));  // exact
  x1 = __builtin_fmaf(x1, scale, -static_cast<float>(h[1]));
  out[0] = __builtin_bit_cast(uint32_t, h);
  out[1] = __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(__builtin_fmaf(x0, kUp, 0.f)),
                                              static_cast<_Float16>(__builtin_fmaf(x1, kUp, 0.f))});
}
// The parts' sums as one.
__device__ inline f32x4 join(const f32x4 (&x)[kParts]) {
  f32x4 s;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(x[1][i], kPartUnit, x[0][i]);
  return s;
}

}  // namespace split16
}  // namespace wrs
