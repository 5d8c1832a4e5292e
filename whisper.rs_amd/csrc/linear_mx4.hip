// Projections with MXFP4 weights.
//
// K15 (linear_mx4_tile): out[g](t, r) = act(w[g][r] . x[t] + bias[g][r]), sums in f32. A
//   workgroup takes 64 rows by 64 features; x and the weights, as the f32 values they
//   stand for, pass through LDS 32 columns (one scale block) at a time.
#include "wrs_internal.hpp"

#include <algorithm>
#include <atomic>

namespace wrs {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kTop = 0xFFFF0000u;

// bf16 parts that carry a value of type T whole: 8 of its bits each.
template <typename T>
constexpr int kParts = 1;
template <>
constexpr int kParts<float> = 3;
template <>
constexpr int kParts<_Float16> = 2;

// x = the sum of its parts (the top half of their f32 patterns), exactly: each takes the
// next 8 significant bits. An infinity or NaN is its first part alone.
template <int P>
__device__ inline void split_top(float x, uint32_t (&p)[P]) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  p[0] = b & kTop;
  if constexpr (P > 1) {
    const bool odd = (b & 0x7F800000u) == 0x7F800000u;
    if (odd && (b & 0x007FFFFFu)) p[0] |= 0x00400000u;
    float rest = x - __builtin_bit_cast(float, p[0]);
#pragma unroll
    for (int i = 1; i < P; ++i) {
      p[i] = odd ? 0u : __builtin_bit_cast(uint32_t, rest) & kTop;
      rest -= __builtin_bit_cast(float, p[i]);
    }
  }
}

// 8 values of type T as f32.
template <typename T>
__device__ inline void load8(const T* p, float (&x)[8]) {
  typedef T t8 __attribute__((ext_vector_type(8), aligned(16)));
  const t8 v = *reinterpret_cast<const t8*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(v[i]);
}

__device__ inline float scale_of(int byte) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(byte) << 23);
}
// 8 codes times a scale, exactly, as bf16 (bf16 has every exponent that a scale has).
__device__ inline bf16x8 widen8(uint32_t w, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

constexpr int kRowsWaves = 8;
constexpr int kRowsBatch = 8;  // steps whose codes a wave has in flight

template <typename XT, int kCT, typename OT>
__global__ __launch_bounds__(64 * kRowsWaves) void mx4_rows(Mx4LinearArgs a, int ks, int chunk) {
  constexpr bool kBoth = sizeof(XT) == 1;  // x is MXFP4 too
  constexpr int kP = kBoth ? 1 : kParts<XT>;
  constexpr int kPitch = 16 * kCT + 1;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int tiles = kRowsWaves / ks, kw = wave % ks;
  const int grp = blockIdx.y;
  const int first = blockIdx.x * tiles * 16;  // the workgroup's first feature
  const int nb = a.n_in / kMx4Block, bytes = a.n_in / 2;
  const int64_t row = min(first + 16 * (wave / ks) + c, a.n_out - 1);
  const uint8_t* const wp = a.w[grp] + row * bytes;
  const uint8_t* const sp = a.w_scales[grp] + row * nb;
  const int64_t xrow = min(c, a.n_tokens - 1);  // kBoth
  const uint8_t* const xp = static_cast<const uint8_t*>(a.x) + xrow * bytes;
  const uint8_t* const xsp = a.x_scales + xrow * nb;

  f32x4 acc[2][kCT];
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int i = 0; i < kCT; ++i) acc[e][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int pitch = 2 * (kMx4Block * chunk + 8);  // bytes of a staged column
  for (int b0 = 0; b0 < nb; b0 += chunk) {
    const int nbc = min(chunk, nb - b0);
    const int steps = (nbc + 4 * ks - 1) / (4 * ks);
    u32x4 cw[kRowsBatch], xw[kBoth ? kRowsBatch : 1];
    int sw[kRowsBatch], xs[kBoth ? kRowsBatch : 1];
    // Blocks past the last one read as zero: the last one's codes, times 2^-127 and x's 0.
    auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < kRowsBatch; ++u) {
        const int at = b0 + 4 * ((s0 + u) * ks + kw) + g, b = min(at, nb - 1);
        cw[u] = *reinterpret_cast<const u32x4*>(wp + 16 * b);
        sw[u] = sp[b];
        if constexpr (kBoth) {
          xw[u] = *reinterpret_cast<const u32x4*>(xp + 16 * b);
          xs[u] = at < nb ? xsp[b] : 0;
        }
        if (at >= nb) sw[u] = 0;
      }
    };
    load(0);
    if constexpr (!kBoth) {
      // x's columns of the chunk: part p of row t is column p * n_tokens + t.
      const int wide = 4 * chunk;  // groups of 8 values a row
      if (b0) __syncthreads();
      for (int e = tid; e < (16 * kCT - kP * a.n_tokens) * wide; e += 64 * kRowsWaves)
        *reinterpret_cast<u32x4*>(lds + (kP * a.n_tokens + e / wide) * pitch + 16 * (e % wide)) =
            u32x4{0, 0, 0, 0};
      for (int e = tid; e < a.n_tokens * wide; e += 64 * kRowsWaves) {
        const int t = e / wide, k = e % wide;
        u32x4 w[kP];
#pragma unroll
        for (int p = 0; p < kP; ++p) w[p] = u32x4{0, 0, 0, 0};
        if (k < 4 * nbc) {
          float x[8];
          load8<XT>(static_cast<const XT*>(a.x) + t * a.x_rs + kMx4Block * b0 + 8 * k, x);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            uint32_t lo[kP], hi[kP];
            split_top<kP>(x[i], lo);
            split_top<kP>(x[i + 1], hi);
#pragma unroll
            for (int p = 0; p < kP; ++p) w[p][i >> 1] = (lo[p] >> 16) | hi[p];
          }
        }
#pragma unroll
        for (int p = 0; p < kP; ++p)
          *reinterpret_cast<u32x4*>(lds + (p * a.n_tokens + t) * pitch + 16 * k) = w[p];
      }
      __syncthreads();
    }
    for (int s0 = 0; s0 < steps; s0 += kRowsBatch) {
      if (s0) load(s0);
#pragma unroll
      for (int u = 0; u < kRowsBatch; ++u) {
        if (s0 + u >= steps) break;
        if constexpr (kBoth) {
          i32x8 wa = {}, xa = {};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            wa[j] = static_cast<int>(cw[u][j]);
            xa[j] = static_cast<int>(xw[u][j]);
          }
          acc[u & 1][0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              wa, xa, acc[u & 1][0], 4, 4, 0, sw[u], 0, xs[u]);
        } else {
          const char* const xl = lds + c * pitch + 64 * (4 * ((s0 + u) * ks + kw) + g);
          const float scale = scale_of(sw[u]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bf16x8 wv = widen8(cw[u][j], scale);
#pragma unroll
            for (int i = 0; i < kCT; ++i)
              acc[j & 1][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  wv, *reinterpret_cast<const bf16x8*>(xl + 16 * i * pitch + 16 * j),
                  acc[j & 1][i], 0, 0, 0);
          }
        }
      }
    }
  }
  // The waves' sums meet in LDS; a thread adds one output's over its waves and parts.
  __syncthreads();
  float* const red = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < kCT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      red[(16 * wave + 4 * g + e) * kPitch + 16 * i + c] = acc[0][i][e] + acc[1][i][e];
  __syncthreads();
  for (int e = tid; e < 16 * tiles * a.n_tokens; e += 64 * kRowsWaves) {
    const int t = e / (16 * tiles), rr = e % (16 * tiles), r = first + rr;
    if (r >= a.n_out) continue;
    float y = 0.f;
#pragma unroll
    for (int p = kP - 1; p >= 0; --p)
      for (int k = 0; k < ks; ++k)
        y += red[(16 * ((rr >> 4) * ks + k) + (rr & 15)) * kPitch + p * a.n_tokens + t];
    if (a.bias[grp]) y += a.bias[grp][r];
    if (a.act == kActGelu) y = gelu_tanh(y);
    static_cast<OT*>(a.out[grp])[t * a.out_rs + (r >> 6) * a.out_hs + (r & 63)] =
        static_cast<OT>(y);
  }
}

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

// Few rows: how many waves share a tile's columns, and the blocks staged at a time.
struct RowsShape {
  int ks, chunk;
  size_t lds;
};
template <int kCT>
RowsShape rows_shape(const Mx4LinearArgs& a, bool both) {
  const int nb = a.n_in / kMx4Block;
  const int64_t tiles = (a.n_out + 15ll) / 16 * a.n_groups;
  int ks = kRowsWaves;
  while (ks > 1 && (tiles * ks > 2048 || 4 * (ks / 2) >= nb)) ks /= 2;
  const int unit = 4 * ks, all = (nb + unit - 1) / unit * unit;
  const int fit = ((80 * 1024) / (32 * kCT) - 8) / kMx4Block / unit * unit;
  RowsShape r{ks, std::min(all, std::max(unit, fit)), 0};
  r.lds = sizeof(float) * 16 * kRowsWaves * (16 * kCT + 1);
  if (!both) r.lds = std::max<size_t>(r.lds, 32ull * kCT * (kMx4Block * r.chunk + 8));
  return r;
}

template <typename XT, int kCT, typename OT>
hipError_t launch_rows(const Mx4LinearArgs& a, hipStream_t s) {
  constexpr size_t kMost = 128 * 1024;
  const RowsShape r = rows_shape<kCT>(a, sizeof(XT) == 1);
  if (r.lds > kMost) return hipErrorInvalidConfiguration;
  const void* fn = reinterpret_cast<const void*>(&mx4_rows<XT, kCT, OT>);
  static std::atomic<uint64_t> attr_set{0};  // one bit per device
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev >= 64 || !(attr_set.load(std::memory_order_acquire) & (uint64_t{1} << dev))) {
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize,
                            static_cast<int>(kMost));
    if (e != hipSuccess) return e;
    if (dev < 64) attr_set.fetch_or(uint64_t{1} << dev, std::memory_order_acq_rel);
  }
  const int wide = 16 * (kRowsWaves / r.ks);
  const dim3 grid((a.n_out + wide - 1) / wide, a.n_groups);
  hipLaunchKernelGGL((mx4_rows<XT, kCT, OT>), grid, dim3(64 * kRowsWaves), r.lds, s, a, r.ks,
                     r.chunk);
  return hipGetLastError();
}

template <typename XT, typename OT>
hipError_t launch_rows_of(const Mx4LinearArgs& a, hipStream_t s) {
  if constexpr (sizeof(XT) == 1) {
    return launch_rows<XT, 1, OT>(a, s);
  } else {
    const int cols = kParts<XT> * a.n_tokens;
    if (cols <= 16) return launch_rows<XT, 1, OT>(a, s);
    if constexpr (kParts<XT> >= 2)
      if (cols <= 32) return launch_rows<XT, 2, OT>(a, s);
    if constexpr (kParts<XT> >= 3) return launch_rows<XT, 3, OT>(a, s);
    return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_linear_mx4(const Mx4LinearArgs& a, DType x_dt, DType out_dt, hipStream_t s) {
  if (a.n_tokens <= 0 || a.n_out <= 0 || a.n_groups <= 0) return hipSuccess;
  const dim3 grid((a.n_tokens + kTile - 1) / kTile, (a.n_out + kTile - 1) / kTile, a.n_groups);
#define WRS_MX4_ROWS(XT)                                                                     \
  switch (out_dt) {                                                                          \
    case kF32: return launch_rows_of<XT, float>(a, s);                                       \
    case kF16: return launch_rows_of<XT, _Float16>(a, s);                                    \
    case kBF16: return launch_rows_of<XT, __bf16>(a, s);                                     \
    default: return hipErrorInvalidValue;                                                    \
  }
  if (a.n_tokens <= kMx4Rows) {
    if (a.x_scales) {
      WRS_MX4_ROWS(uint8_t)
    }
    switch (x_dt) {
      case kF32: WRS_MX4_ROWS(float)
      case kF16: WRS_MX4_ROWS(_Float16)
      case kBF16: WRS_MX4_ROWS(__bf16)
      default: return hipErrorInvalidValue;
    }
  }
#undef WRS_MX4_ROWS
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
