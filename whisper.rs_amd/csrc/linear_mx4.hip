// Projections with MXFP4 weights.
//
// K15 (linear_mx4_tile): out[g](t, r) = act(w[g][r] . x[t] + bias[g][r]), sums in f32. A
//   workgroup takes 64 rows by 64 features; x and the weights, as the f32 values they
//   stand for, pass through LDS 32 columns (one scale block) at a time.
#include "wrs_internal.hpp"

#include <algorithm>

namespace wrs {
namespace {

constexpr int kTile = 64;

__device__ inline float value_of(uint32_t code, int scale) {
  if (scale == 255) return __builtin_nanf("");
  const uint32_t m = code & 7u;
  const float y = m < 2 ? 0.5f * m : __builtin_ldexpf(2.f + (m & 1u), static_cast<int>(m >> 1) - 2);
  return __builtin_ldexpf((code & 8u) ? -y : y, scale - 127);
}

template <typename XT, typename OT>
__global__ __launch_bounds__(256) void linear_mx4_tile(Mx4LinearArgs a) {
  __shared__ float xs[kMx4Block][kTile + 1], ws[kMx4Block][kTile + 1];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int t0 = blockIdx.x * kTile, r0 = blockIdx.y * kTile, g = blockIdx.z;
  const int blocks = a.n_in / kMx4Block;
  float acc[4][4] = {};
  for (int b = 0; b < blocks; ++b) {
    for (int e = tid; e < kTile * kMx4Block; e += 256) {
      const int i = e >> 5, k = e & 31, col = b * kMx4Block + k;
      float xv = 0.f, wv = 0.f;
      if (t0 + i < a.n_tokens) {
        if constexpr (sizeof(XT) == 1) {
          const int64_t row = t0 + i;
          const uint32_t c = static_cast<const uint8_t*>(a.x)[row * (a.n_in / 2) + col / 2];
          xv = value_of(c >> (4 * (col & 1)), a.x_scales[row * blocks + b]);
        } else {
          xv = static_cast<float>(static_cast<const XT*>(a.x)[(t0 + i) * a.x_rs + col]);
        }
      }
      if (r0 + i < a.n_out) {
        const int64_t row = r0 + i;
        const uint32_t c = a.w[g][row * (a.n_in / 2) + col / 2];
        wv = value_of(c >> (4 * (col & 1)), a.w_scales[g][row * blocks + b]);
      }
      xs[k][i] = xv;
      ws[k][i] = wv;
    }
    __syncthreads();
    for (int k = 0; k < kMx4Block; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_fmaf(xs[k][ty + 16 * i], ws[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + ty + 16 * i, r = r0 + tx + 16 * j;
      if (t >= a.n_tokens || r >= a.n_out) continue;
      float y = acc[i][j] + (a.bias[g] ? a.bias[g][r] : 0.f);
      if (a.act == kActGelu) y = gelu_tanh(y);
      static_cast<OT*>(a.out[g])[t * a.out_rs + (r >> 6) * a.out_hs + (r & 63)] = static_cast<OT>(y);
    }
}

}  // namespace

hipError_t launch_linear_mx4(const Mx4LinearArgs& a, DType x_dt, DType out_dt, hipStream_t s) {
  if (a.n_tokens <= 0 || a.n_out <= 0 || a.n_groups <= 0) return hipSuccess;
  const dim3 grid((a.n_tokens + kTile - 1) / kTile, (a.n_out + kTile - 1) / kTile, a.n_groups);
#define WRS_MX4_OUT(XT)                                                                      \
  switch (out_dt) {                                                                          \
    case kF32:                                                                               \
      hipLaunchKernelGGL((linear_mx4_tile<XT, float>), grid, dim3(256), 0, s, a);            \
      break;                                                                                 \
    case kF16:                                                                               \
      hipLaunchKernelGGL((linear_mx4_tile<XT, _Float16>), grid, dim3(256), 0, s, a);         \
      break;                                                                                 \
    case kBF16:                                                                              \
      hipLaunchKernelGGL((linear_mx4_tile<XT, __bf16>), grid, dim3(256), 0, s, a);           \
      break;                                                                                 \
    default: return hipErrorInvalidValue;                                                    \
  }
  if (a.x_scales) {
    WRS_MX4_OUT(uint8_t)
  } else {
    switch (x_dt) {
      case kF32: WRS_MX4_OUT(float) break;
      case kF16: WRS_MX4_OUT(_Float16) break;
      case kBF16: WRS_MX4_OUT(__bf16) break;
      default: return hipErrorInvalidValue;
    }
  }
#undef WRS_MX4_OUT
  return hipGetLastError();
}

}  // namespace wrs
