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
//   output type. Both are bound by memory: one pass, 16-byte accesses, four of them in flight a
//   lane (with one, and codes made by comparisons, 49.7 and 44.0 us). 51866 x 1280 f16 29.4 us
//   and 25.3 us, 5.7 and 6.6 TB/s; 24000 x 1280 13.0; 1500 x 1280 f32 2.9 and 3.9.
#include "wrs_internal.hpp"

#include <algorithm>

namespace wrs {
namespace {

constexpr int kLane = 8;   // values per lane and group
constexpr int kTurns = 4;  // groups a lane has in flight, 256 lanes apart

template <int CTRL>
__device__ inline uint32_t dpp(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xF, 0xF, false));
}

template <typename T>
struct Lane {  // 8 values, loaded and stored 16 bytes at a time
  typedef T t8 __attribute__((ext_vector_type(8), aligned(16)));
};

// e2m1 code of |y| < 8: how many of the midpoints lie below it (at one, the even code).
__device__ inline uint32_t code_of(float y) {
  return (y > 0.25f) + (y >= 0.75f) + (y > 1.25f) + (y >= 1.75f) + (y > 2.5f) + (y >= 3.5f) +
         (y > 5.f);
}
__device__ inline float scale_of(int byte) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(byte) << 23);
}
// Two values over a scale as codes, in byte k of w: v_cvt_scalef32_pk_fp4 rounds to nearest, ties
// to the even code, and saturates.
template <int k>
__device__ inline uint32_t encode2(uint32_t w, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a, b, scale, k);
}

// Group `t` of 8 values of packed rows is values 8 t.. of x; of strided ones (kPacked
// false), group t % per_row of row t / per_row.
template <typename T, bool kPacked>
__global__ __launch_bounds__(256) void mx4_quantize(const T* x, int64_t x_rs, int64_t groups,
                                                    uint32_t per_row, uint32_t* codes,
                                                    uint8_t* scales) {
  typedef typename Lane<T>::t8 t8;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (256 * kTurns) + threadIdx.x;
  t8 v[kTurns];
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int64_t t = min(t0 + 256 * u, groups - 1);
    const T* p = x + t * kLane;
    if constexpr (!kPacked) {
      const int64_t row = t / per_row;
      p = x + row * x_rs + (t - row * per_row) * kLane;
    }
    v[u] = *reinterpret_cast<const t8*>(p);
  }
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int64_t t = t0 + 256 * u;
    if (t >= groups) return;  // groups are a multiple of 4: whole blocks
    float f[kLane];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      f[i] = static_cast<float>(v[u][i]);
      top = max(top, __builtin_bit_cast(uint32_t, f[i]) & 0x7FFFFFFFu);
    }
    top = max(top, dpp<0xB1>(top));  // xor 1
    top = max(top, dpp<0x4E>(top));  // xor 2
    const bool bad = top >= 0x7F800000u;
    // floor(log2) of a normal number is its exponent field - 127; below the normal ones
    // the scale is 2^-127 anyway.
    const int e = max(static_cast<int>(top >> 23) - 127 - 2, -127);
    uint32_t w = 0;
    if (e > -126) {
      const float scale = scale_of(e + 127);
      w = encode2<0>(w, f[0], f[1], scale);
      w = encode2<1>(w, f[2], f[3], scale);
      w = encode2<2>(w, f[4], f[5], scale);
      w = encode2<3>(w, f[6], f[7], scale);
    } else {  // values next to or below the normal numbers: exact without them
#pragma unroll
      for (int i = 0; i < kLane; ++i)
        w |= (code_of(__builtin_fabsf(__builtin_ldexpf(f[i], -e))) |
              ((__builtin_bit_cast(uint32_t, f[i]) >> 28) & 8u)) << (4 * i);
    }
    codes[t] = bad ? 0u : w;
    if ((t & 3) == 0) scales[t >> 2] = static_cast<uint8_t>(bad ? 255 : e + 127);
  }
}

// 2 values of byte k of w, times a scale, as T.
template <typename T, int k>
__device__ inline void decode2(uint32_t w, float scale, T& a, T& b) {
  if constexpr (sizeof(T) == 4) {
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, k);
    a = v[0];
    b = v[1];
  } else if constexpr (__is_same(T, _Float16)) {
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, k);
    a = v[0];
    b = v[1];
  } else {
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, k);
    a = v[0];
    b = v[1];
  }
}

template <typename T, bool kPacked>
__global__ __launch_bounds__(256) void mx4_dequantize(const uint32_t* codes, const uint8_t* scales,
                                                      int64_t groups, uint32_t per_row, T* out,
                                                      int64_t out_rs) {
  typedef typename Lane<T>::t8 t8;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * (256 * kTurns) + threadIdx.x;
  uint32_t w[kTurns];
  int s[kTurns];
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int64_t t = min(t0 + 256 * u, groups - 1);
    w[u] = codes[t];
    s[u] = scales[t >> 2];
  }
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int64_t t = t0 + 256 * u;
    if (t >= groups) return;
    T* p = out + t * kLane;
    if constexpr (!kPacked) {
      const int64_t row = t / per_row;
      p = out + row * out_rs + (t - row * per_row) * kLane;
    }
    const float scale = scale_of(s[u]);
    T y[kLane];
    decode2<T, 0>(w[u], scale, y[0], y[1]);
    decode2<T, 1>(w[u], scale, y[2], y[3]);
    decode2<T, 2>(w[u], scale, y[4], y[5]);
    decode2<T, 3>(w[u], scale, y[6], y[7]);
    t8 v;
#pragma unroll
    for (int i = 0; i < kLane; ++i) v[i] = y[i];
    *reinterpret_cast<t8*>(p) = v;
  }
}

}  // namespace

hipError_t launch_mx4_quantize(DType x_dt, const void* x, int64_t x_rs, int64_t n_rows, int n_cols,
                               uint8_t* codes, uint8_t* scales, hipStream_t s) {
  const int64_t groups = n_rows * (n_cols / kLane);
  if (groups <= 0) return hipSuccess;
  const int64_t blocks = (groups + 256 * kTurns - 1) / (256 * kTurns);
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
  const int64_t blocks = (groups + 256 * kTurns - 1) / (256 * kTurns);
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
