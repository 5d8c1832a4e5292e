// MXFP4 rows: quantisation and its inverse.
//
// K13 (mx4_quantize): blocks of 32 values along a row become a scale byte and 16 bytes
//   of codes, as the OCP Microscaling Formats specification (v1.0) has them: the scale
//   is 2^(floor(log2(largest magnitude)) - 2), at least 2^-127, and the codes are the
//   nearest e2m1 values of value / scale, ties to the even code, 6 the largest. A block
//   with an infinity or NaN gets the NaN scale (255) and codes of zero; a block of zeros
//   2^-127. Four lanes take a block, 8 values each; the largest magnitude is the largest
//   bit pattern, so the block's maximum needs no floating point and keeps NaN on top.
// K14 (mx4_dequantize): the values that codes and scales stand for, rounded once to the
//   output type. Both are bound by memory: one pass, 16-byte accesses.
#include "wrs_internal.hpp"

#include <algorithm>

namespace wrs {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));

constexpr int kLane = 8;  // values per lane

template <typename T>
__device__ inline f32x8 load8(const T* p);
template <>
__device__ inline f32x8 load8<float>(const float* p) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
  return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
template <>
__device__ inline f32x8 load8<_Float16>(const _Float16* p) {
  return __builtin_convertvector(*reinterpret_cast<const f16x8*>(p), f32x8);
}
template <>
__device__ inline f32x8 load8<__bf16>(const __bf16* p) {
  return __builtin_convertvector(*reinterpret_cast<const bf16x8*>(p), f32x8);
}

template <typename T>
__device__ inline void store8(T* p, const f32x8& x);
template <>
__device__ inline void store8<float>(float* p, const f32x8& x) {
  reinterpret_cast<f32x4*>(p)[0] = f32x4{x[0], x[1], x[2], x[3]};
  reinterpret_cast<f32x4*>(p)[1] = f32x4{x[4], x[5], x[6], x[7]};
}
template <>
__device__ inline void store8<_Float16>(_Float16* p, const f32x8& x) {
  *reinterpret_cast<f16x8*>(p) = __builtin_convertvector(x, f16x8);
}
template <>
__device__ inline void store8<__bf16>(__bf16* p, const f32x8& x) {
  *reinterpret_cast<bf16x8*>(p) = __builtin_convertvector(x, bf16x8);
}

template <int CTRL>
__device__ inline uint32_t dpp(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xF, 0xF, false));
}

// x * 2^e, e in [-127, 127], exactly rounded also where 2^e or the result is subnormal.
__device__ inline float scaled(float x, int e) { return __builtin_ldexpf(x, e); }

// e2m1 code of |y| < 8: how many of the midpoints lie below it (at one, the even code).
__device__ inline uint32_t code_of(float y) {
  return (y > 0.25f) + (y >= 0.75f) + (y > 1.25f) + (y >= 1.75f) + (y > 2.5f) + (y >= 3.5f) +
         (y > 5.f);
}

// Group `t` of 8 values of packed rows is values 8 t.. of x; of strided ones (kPacked
// false), group t % per_row of row t / per_row.
template <typename T, bool kPacked>
__global__ __launch_bounds__(256) void mx4_quantize(const T* x, int64_t x_rs, int64_t groups,
                                                    uint32_t per_row, uint32_t* codes,
                                                    uint8_t* scales) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= groups) return;  // groups are a multiple of 4: whole blocks
  const T* p = x + t * kLane;
  if constexpr (!kPacked) {
    const int64_t row = t / per_row;
    p = x + row * x_rs + (t - row * per_row) * kLane;
  }
  const f32x8 v = load8<T>(p);
  const u32x8 bits = __builtin_bit_cast(u32x8, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, bits[i] & 0x7FFFFFFFu);
  top = max(top, dpp<0xB1>(top));  // xor 1
  top = max(top, dpp<0x4E>(top));  // xor 2
  const bool bad = top >= 0x7F800000u;
  // floor(log2) of a normal number is its exponent field - 127; below the normal ones
  // the scale is 2^-127 anyway.
  const int e = max(static_cast<int>(top >> 23) - 127 - 2, -127);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = code_of(__builtin_fabsf(scaled(v[i], -e))) |
                       ((bits[i] >> 28) & 8u);
    w |= c << (4 * i);
  }
  codes[t] = bad ? 0u : w;
  if ((t & 3) == 0) scales[t >> 2] = static_cast<uint8_t>(bad ? 255 : e + 127);
}

template <typename T, bool kPacked>
__global__ __launch_bounds__(256) void mx4_dequantize(const uint32_t* codes, const uint8_t* scales,
                                                      int64_t groups, uint32_t per_row, T* out,
                                                      int64_t out_rs) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (t >= groups) return;
  T* p = out + t * kLane;
  if constexpr (!kPacked) {
    const int64_t row = t / per_row;
    p = out + row * out_rs + (t - row * per_row) * kLane;
  }
  const uint32_t w = codes[t];
  const int s = scales[t >> 2];
  f32x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = w >> (4 * i);
    // Codes 2..7 are (2 + bit 0) * 2^(code / 2 - 2), 0 and 1 are halves of themselves.
    const uint32_t m = c & 7u;
    const float y = m < 2 ? 0.5f * m : __builtin_ldexpf(2.f + (m & 1u), static_cast<int>(m >> 1) - 2);
    v[i] = s == 255 ? __builtin_nanf("")
                    : scaled(__builtin_bit_cast(float, __builtin_bit_cast(uint32_t, y) |
                                                           ((c & 8u) << 28)), s - 127);
  }
  store8<T>(p, v);
}

}  // namespace

hipError_t launch_mx4_quantize(DType x_dt, const void* x, int64_t x_rs, int64_t n_rows, int n_cols,
                               uint8_t* codes, uint8_t* scales, hipStream_t s) {
  const int64_t groups = n_rows * (n_cols / kLane);
  if (groups <= 0) return hipSuccess;
  const int64_t blocks = (groups + 255) / 256;
  if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks));
  const bool packed = x_rs == n_cols || n_rows == 1;
  const uint32_t per_row = n_cols / kLane;
  auto* cw = reinterpret_cast<uint32_t*>(codes);
#define WRS_MX4(T)                                                                            \
  if (packed)                                                                                 \
    hipLaunchKernelGGL((mx4_quantize<T, true>), grid, dim3(256), 0, s,                        \
                       static_cast<const T*>(x), x_rs, groups, per_row, cw, scales);          \
  else                                                                                        \
    hipLaunchKernelGGL((mx4_quantize<T, false>), grid, dim3(256), 0, s,                       \
                       static_cast<const T*>(x), x_rs, groups, per_row, cw, scales);
  switch (x_dt) {
    case kF32: WRS_MX4(float) break;
    case kF16: WRS_MX4(_Float16) break;
    case kBF16: WRS_MX4(__bf16) break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_MX4
  return hipGetLastError();
}

hipError_t launch_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t n_rows,
                                 int n_cols, DType out_dt, void* out, int64_t out_rs,
                                 hipStream_t s) {
  const int64_t groups = n_rows * (n_cols / kLane);
  if (groups <= 0) return hipSuccess;
  const int64_t blocks = (groups + 255) / 256;
  if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(blocks));
  const bool packed = out_rs == n_cols || n_rows == 1;
  const uint32_t per_row = n_cols / kLane;
  const auto* cw = reinterpret_cast<const uint32_t*>(codes);
#define WRS_MX4(T)                                                                            \
  if (packed)                                                                                 \
    hipLaunchKernelGGL((mx4_dequantize<T, true>), grid, dim3(256), 0, s, cw, scales, groups,  \
                       per_row, static_cast<T*>(out), out_rs);                                \
  else                                                                                        \
    hipLaunchKernelGGL((mx4_dequantize<T, false>), grid, dim3(256), 0, s, cw, scales, groups, \
                       per_row, static_cast<T*>(out), out_rs);
  switch (out_dt) {
    case kF32: WRS_MX4(float) break;
    case kF16: WRS_MX4(_Float16) break;
    case kBF16: WRS_MX4(__bf16) break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_MX4
  return hipGetLastError();
}

}  // namespace wrs
