// Attention over the KV arena whose rows see a sliding window and the first tokens, and every
// attention over 8-bit arenas.
//
// K19 (window_attend): row r of a sequence stands at position p = past + r (`causal`; else every
//   row at the last key) and sees the keys j <= p with j > p - window or j < sinks:
//   s_j = q.k_j / 8, out = softmax(s) V over those j only.
//   A workgroup of four waves runs one block of 16 kRT rows of one head. The block's keys are the
//   first tokens' 32-key steps, then those from its first row's window to its last row's own key:
//   steps in between are never read. Wave w takes steps w, w + 4, ... with an online softmax of its
//   own, the waves merge their (max, sum, O) in LDS, and where a block's steps are dealt over several
//   workgroups those merge through memory (the last to count in adds the partials up in order, so
//   results do not depend on which it is). Only steps that hold a key hidden from some row test keys.
//   f16 planes run on the f16 matrix pipe with operands in two parts, f32 ones on the f32 pipe.
//   8-bit planes: codes are whole numbers that f16 and bf16 hold as they are. Scores take them as
//   f16 against q in two f16 parts, then the keys' powers of two, whatever they are, in f32. Weights
//   take the values' powers before they are split, into two bf16 parts: bf16 has f32's range, so rows
//   of any scale meet in one sum, and two parts hold 2^-18 of a weight.
#include "split16.hpp"

#include <algorithm>

namespace wrs {
namespace {

using namespace split16;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kN = 32;              // keys per step
constexpr int kPitch = 68;          // LDS pitch (floats) of a merge row
constexpr int kCounterStride = 32;  // 128 bytes between merge counters
constexpr int kMergeLoads = 8;      // partials in flight per thread in the merge
constexpr int kRawBuffer = 0x00020000;  // buffer resource word 3: raw, 32-bit data format

// The steps of rows at positions p0..p1: `sink_steps` of them from key 0 on, the others from key
// `lo` on (a multiple of kN), up to key p1. Where the two meet, all lie from key 0 on.
struct Span {
  int lo, sink_steps, n_steps;
};
__host__ __device__ inline Span span_of(int p0, int p1, int window, int sinks) {
  Span s;
  const int first = p0 - window + 1;  // window <= 2^24
  s.lo = first > 0 ? first / kN * kN : 0;
  s.sink_steps = (sinks < p1 + 1 ? sinks + kN - 1 : p1 + kN) / kN;
  if (s.sink_steps * kN >= s.lo) s.lo = s.sink_steps = 0;
  s.n_steps = s.sink_steps + (p1 - s.lo + kN) / kN;
  return s;
}

// What a wave knows of its block.
struct Block {
  int p0, p1;            // positions of the block's first and last row
  int window, sinks;
  Span span;
  int step0, step1;      // the workgroup's steps
  __amdgpu_buffer_rsrc_t k, v, ks, vs;  // the head's planes, zero past key p1

  __device__ inline int key_of(int step) const {
    return kN * step + (step < span.sink_steps ? 0 : span.lo - kN * span.sink_steps);
  }
  // Whether some row of the block does not see some of `n` keys from j0 on.
  __device__ inline bool masked(int j0, int n) const {
    return j0 + n - 1 > p0 || (j0 <= p1 - window && j0 + n > sinks);
  }
  __device__ inline bool sees(int p, int j) const {
    return j <= p && (j > p - window || j < sinks);
  }
};

// A wave's running sums: of lane (c, g), rows 16 rt + c.
template <int kRT>
struct Sums {
  f32x4 o[kRT][4];
  float m[kRT], l[kRT];
  __device__ inline void clear() {
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[rt] = -INFINITY;
      l[rt] = 0.f;
    }
  }
};

// 4 values of a plane row at byte offset `o` (multiple of 4 values), zero past the range.
template <DType kD>
__device__ inline f32x4 load4(const __amdgpu_buffer_rsrc_t& rs, uint32_t o) {
  if constexpr (kD == kF32)
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0));
  else
    return __builtin_convertvector(
        __builtin_bit_cast(f16x4, __builtin_amdgcn_raw_buffer_load_b64(rs, o, 0, 0)), f32x4);
}

// A wave's steps on the f32 matrix pipe, 16 keys at a time, f16 planes widened exactly: lane
// (c, g) holds key c's values d = 16 g + 0..15, so that lane (r, g) gets scores of keys 4 g + 0..3 of
// row r, which are the B operand of O^T += V^T P^T as they stand. o[rt][dt][e] is column 16 g + 4 e +
// dt. q: d = 16 g + 0..15 of row c, times scale * log2(e). pos: row c's position.
template <DType kD, int kRT>
__device__ inline void attend_f32(const Block& b, const f32x4 (&qx)[kRT][4],
                                  const int (&pos)[kRT], int wave, int lane, Sums<kRT>& st) {
  constexpr uint32_t kSize = kD == kF32 ? 4 : 2, kRowBytes = 64 * kSize;
  const int c = lane & 15, g = lane >> 4;
  f32x4 kn[4], vn[4];
  auto load = [&](int j0) __attribute__((always_inline)) {
    const uint32_t ko = static_cast<uint32_t>(j0 + c) * kRowBytes + 16 * g * kSize;
    const uint32_t vo = static_cast<uint32_t>(j0 + 4 * g) * kRowBytes + 4 * c * kSize;
#pragma unroll
    for (int i = 0; i < 4; ++i) kn[i] = load4<kD>(b.k, ko + 4 * i * kSize);
#pragma unroll
    for (int i = 0; i < 4; ++i) vn[i] = load4<kD>(b.v, vo + i * kRowBytes);
  };
  // Piece u: half u % 2 of step u / 2.
  auto key_of = [&](int u) { return b.key_of(u >> 1) + 16 * (u & 1); };
  int u = 2 * (b.step0 + wave);
  const int end = 2 * b.step1;
  if (u < end) load(key_of(u));
  st.clear();
  for (int next; u < end; u = next) {
    next = u & 1 ? u + 1 + 2 * (kWaves - 1) : u + 1;
    const int j0 = key_of(u);
    f32x4 kx[4], vx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kx[i] = kn[i];
      vx[i] = vn[i];
    }
    if (next < end) load(key_of(next));
    // Values that a row does not see have weight 0, and 0 times an infinity or NaN is NaN: such
    // values leave the product and are added row by row.
    const bool masked = b.masked(j0, 16);
    bool odd = false;
    if (masked) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= !__builtin_isfinite(vx[i][e]);
      odd = __any(odd);
    }
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
      f32x4 s0 = {}, s1 = {};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[i][e], qx[rt][i][e], s0, 0, 0, 0);
          s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[i][e + 1], qx[rt][i][e + 1], s1, 0, 0, 0);
        }
      f32x4 s = s0 + s1;
      int seen = 0xF;  // bit i: the row sees key j0 + 4 g + i
      if (masked) {
        seen = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (b.sees(pos[rt], j0 + 4 * g + i))
            seen |= 1 << i;
          else
            s[i] = -INFINITY;
      }
      const float mx = max_x16_x32(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
      const float m_new = fmaxf(st.m[rt], mx);
      const float alpha = st.m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m[rt] - m_new);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      st.m[rt] = m_new;
      f32x4 p;
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(s[i] - m_use);
      st.l[rt] = __builtin_fmaf(st.l[rt], alpha, (p[0] + p[1]) + (p[2] + p[3]));
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) st.o[rt][dt] *= alpha;
      if (odd) {
#pragma unroll 1
        for (int key = 0; key < 16; ++key) {
          // Weight and sight of key j0 + key, and its row's values of this lane's columns.
          const int i = key & 3;
          const float mine = i == 0 ? p[0] : i == 1 ? p[1] : i == 2 ? p[2] : p[3];
          const float pk = __shfl(mine, c + 16 * (key >> 2));
          const bool vis = (__shfl(seen, c + 16 * (key >> 2)) >> i) & 1;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x4 vk = load4<kD>(b.v, static_cast<uint32_t>(j0 + key) * kRowBytes +
                                                (16 * g + 4 * e) * kSize);
#pragma unroll
            for (int dt = 0; dt < 4; ++dt)
              if (vis && !__builtin_isfinite(vk[dt])) st.o[rt][dt][e] += pk * vk[dt];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
          st.o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(
              odd && !__builtin_isfinite(vx[i][dt]) ? 0.f : vx[i][dt], p[i], st.o[rt][dt], 0, 0, 0);
    }
  }
}

// Codes (offset by 128) of 4 values as f16: 1024 + code, less 1152.
__device__ inline void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const f16x2 off = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
  const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u));
  const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u));
  lo = __builtin_bit_cast(uint32_t, a + off);
  hi = __builtin_bit_cast(uint32_t, b + off);
}
// The same as bf16, which holds whole numbers to 256: the upper half of each f32.
__device__ inline void codes_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = __builtin_bit_cast(uint32_t, static_cast<float>((w >> (8 * i)) & 0xFFu) - 128.f);
  lo = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);
  hi = __builtin_amdgcn_perm(x[3], x[2], 0x07060302u);
}
// 2^(byte - 127) of byte i of four scales (255: infinity, and its codes are zeros: NaN).
__device__ inline float scale_at(uint32_t w, int i) {
  const uint32_t up = i == 0 ? w << 23 : i == 1 ? w << 15 : i == 2 ? w << 7 : w >> 1;
  return __builtin_bit_cast(float, up & 0x7F800000u);
}
// Two weights in two bf16 parts: both to nearest, the second of what the first leaves.
__device__ inline void split_bf16(float x0, float x1, uint32_t (&out)[kParts]) {
  const f32x2 x = {x0, x1};
  const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
  const f32x2 r = {x0 - __builtin_bit_cast(float, h << 16),
                   x1 - __builtin_bit_cast(float, h & 0xFFFF0000u)};
  out[0] = h;
  out[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
}
__device__ inline f32x4 mfma_bf16(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Query rows (d = 16 g + 0..15 of row c of each tile) times a power of two that puts a row's
// largest element into [2^14, 2^15), in two f16 parts; down: its inverse.
template <int kRT>
__device__ inline void split_rows(const f32x4 (&qx)[kRT][4], u32x4 (&qf)[kRT][kParts][2],
                                  float (&down)[kRT]) {
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) amax = fmaxf(amax, __builtin_fabsf(qx[rt][i][e]));
    amax = max_x16_x32(amax);
    const int e_max = static_cast<int>((__builtin_bit_cast(uint32_t, amax) >> 23) & 0xFF);
    const int sh = e_max == 0 ? 0 : clamp_exp(141 - e_max);
    const float up = pow2(sh);
    down[rt] = pow2(clamp_exp(-sh));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t w[kParts];
      split_units(qx[rt][i >> 1][2 * (i & 1)], qx[rt][i >> 1][2 * (i & 1) + 1], up, w);
#pragma unroll
      for (int p = 0; p < kParts; ++p) qf[rt][p][i >> 2][i & 3] = w[p];
    }
  }
}

// A wave's steps of an f16 or 8-bit plane on the 16-bit matrix pipe. K comes from memory in operand
// layout, V passes through the wave's own swizzled LDS rows and is read transposed; the packed weights
// are the B operand of O^T += V^T P^T as they stand. o[rt][dt][e] is column 16 dt + 4 g + e. Returns
// whether a sum came out infinite or NaN: parts of an infinity are not numbers, so a wave over f16
// planes starts again with f32 operands.
template <bool k8, int kRT>
__device__ inline bool attend_16(const Block& b, const f32x4 (&qx)[kRT][4], const int (&pos)[kRT],
                                 int wave, int lane, char* vw, Sums<kRT>& st) {
  const int c = lane & 15, g = lane >> 4;
  constexpr int kK = k8 ? 1 : 2;  // 16-byte pieces of a lane's share of a key
  constexpr int kV = k8 ? 2 : 4;  // and of the step's values
  u32x4 kx[2][kK], vx[kV];
  uint32_t ks[2], vs[2];
  auto load = [&](int j0) __attribute__((always_inline)) {
    const uint32_t ko = static_cast<uint32_t>(j0 + c) * (64u * kK) + 16u * kK * g;
    const uint32_t vo = static_cast<uint32_t>(j0) * (64u * kK) + 16u * lane;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int kk = 0; kk < kK; ++kk)
        kx[t][kk] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                  b.k, ko + 1024 * kK * t + 16 * kk, 0, 0));
      if constexpr (k8) {
        const uint32_t so = static_cast<uint32_t>(j0 + 16 * t + 4 * g);
        ks[t] = __builtin_amdgcn_raw_buffer_load_b32(b.ks, so, 0, 0);
        vs[t] = __builtin_amdgcn_raw_buffer_load_b32(b.vs, so, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < kV; ++i)
      vx[i] = __builtin_bit_cast(u32x4,
                                 __builtin_amdgcn_raw_buffer_load_b128(b.v, vo + 1024 * i, 0, 0));
  };
  st.clear();
  int step = b.step0 + wave;
  if (step < b.step1) load(b.key_of(step));
  u32x4 qf[kRT][kParts][2];  // d = 16 g + 8 kk + 0..7
  float down[kRT];
  split_rows<kRT>(qx, qf, down);
  for (; step < b.step1; step += kWaves) {
    const int j0 = b.key_of(step);
    u32x4 pf[kRT][kParts];
    f32x4 s[kRT][2];
    float alpha[kRT], sv[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      u32x4 kf[2];
      if constexpr (k8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t lo, hi;
          codes_f16(kx[t][0][i], lo, hi);
          kf[i >> 1][2 * (i & 1)] = lo;
          kf[i >> 1][2 * (i & 1) + 1] = hi;
        }
      } else {
        kf[0] = kx[t][0];
        kf[1] = kx[t][kK - 1];
      }
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) {
        f32x4 sp[kParts] = {};
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int p = 0; p < kParts; ++p) sp[p] = mfma16(kf[kk], qf[rt][p][kk], sp[p]);
        s[rt][t] = join(sp);
        if constexpr (k8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[rt][t][i] *= scale_at(ks[t], i);
        }
      }
      if constexpr (k8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[t][i] = scale_at(vs[t], i);
      }
    }
    wave_sync();  // the last step's transposed reads are done
    if constexpr (k8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 16 * i + (lane >> 2);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          u32x4 y;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t lo, hi;
            codes_bf16(vx[i][2 * e + n], lo, hi);
            y[2 * n] = lo;
            y[2 * n + 1] = hi;
          }
          *reinterpret_cast<u32x4*>(vw + row * 128 + (((2 * (lane & 3) + e) ^ swz(row)) * 16)) = y;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const int row = 8 * i + (lane >> 3);
        *reinterpret_cast<u32x4*>(vw + row * 128 + (((lane & 7) ^ swz(row)) * 16)) = vx[i];
      }
    }
    wave_sync();
    if (step + kWaves < b.step1) load(b.key_of(step + kWaves));
    const bool masked = b.masked(j0, kN);
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
      // Register i of tile t holds key 16 t + 4 g + i.
      uint32_t seen = 0xFFu;
      if (masked) {
        seen = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (b.sees(pos[rt], j0 + 16 * t + 4 * g + i))
              seen |= 1u << (4 * t + i);
            else
              s[rt][t][i] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][t][i]);
      // Maxima are kept in the units of the parts' sums: times down, a power of two, exact.
      const float m_new = fmaxf(st.m[rt], max_x16_x32(mx));
      alpha[rt] = st.m[rt] == -INFINITY
                      ? 0.f
                      : __builtin_amdgcn_exp2f((st.m[rt] - m_new) * down[rt]);
      st.m[rt] = m_new;
      const float md = m_new == -INFINITY ? 0.f : m_new * down[rt];
      float ls = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][t][i], down[rt], -md));
          float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][t][i + 1], down[rt], -md));
          ls += p0 + p1;
          uint32_t w[kParts];
          if constexpr (k8) {
            // A hidden key's scale may be the NaN one: it takes no part.
            p0 *= masked && !(seen >> (4 * t + i) & 1) ? 0.f : sv[t][i];
            p1 *= masked && !(seen >> (4 * t + i + 1) & 1) ? 0.f : sv[t][i + 1];
            split_bf16(p0, p1, w);
          } else {
            split_units(p0, p1, kWeightUp, w);
          }
#pragma unroll
          for (int p = 0; p < kParts; ++p) pf[rt][p][2 * t + (i >> 1)] = w[p];
        }
      st.l[rt] = __builtin_fmaf(st.l[rt], alpha[rt], ls);
    }
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      u32x2 t[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 16 * e + 4 * g + (c >> 2);
        t[e] = read_tr(vw + row * 128 + (((2 * dt + ((c & 3) >> 1)) ^ swz(row)) * 16) + 8 * (c & 1));
      }
      const u32x4 va = {t[0].x, t[0].y, t[1].x, t[1].y};
#pragma unroll
      for (int rt = 0; rt < kRT; ++rt) {
        f32x4 y;
        if constexpr (k8) {
          y = mfma_bf16(va, pf[rt][1], f32x4{0.f, 0.f, 0.f, 0.f});
          y = mfma_bf16(va, pf[rt][0], y);
        } else {
          f32x4 x[kParts];
#pragma unroll
          for (int p = 0; p < kParts; ++p) x[p] = mfma16(va, pf[rt][p], f32x4{0.f, 0.f, 0.f, 0.f});
          y = join(x);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[rt][dt][e] = __builtin_fmaf(st.o[rt][dt][e], alpha[rt], y[e]);
      }
    }
  }
  bool odd = false;
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    odd |= !__builtin_isfinite(st.l[rt]);
    st.m[rt] *= down[rt];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) {
      if constexpr (!k8) st.o[rt][dt] *= 1.f / kWeightUp;
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= !__builtin_isfinite(st.o[rt][dt][e]);
    }
  }
  return !k8 && __any(odd);
}

template <DType kD, int kRT>
__global__ __launch_bounds__(64 * kWaves, 2) void window_attend(WindowArgs a) {
  constexpr int kRows = 16 * kRT;
  __shared__ __attribute__((aligned(128))) char vs[kD == kF32 ? 1 : kWaves][kN * 128];
  __shared__ __attribute__((aligned(16))) float mo[kWaves][kRows * kPitch];  // a wave's O rows
  __shared__ float ml[kWaves][2][kRows];  // and their max and sum
  __shared__ int last_flag;

  // The workgroups of one head's keys, which read the same rows, share an XCD's L2 (a sequence's
  // row of the grid is a multiple of the XCDs).
  const int t = blockIdx.y;
  const int lid = xcd_remap(blockIdx.x, gridDim.x);
  if (lid >= a.n_wgs[t]) return;
  const int past = a.past[t], rows = a.rows[t];
  const int n_blk = a.n_blk[t], n_split = a.n_split[t];
  int blk, split;
  const int hs = divide(lid, n_blk, a.blk_inv[t], blk);
  const int h = divide(hs, n_split, a.split_inv[t], split);
  const int row0 = blk * kRows;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t q_row = a.row0[t];

  Block b;
  b.p0 = a.causal ? past + row0 : past - 1;
  b.p1 = a.causal ? past + min(row0 + kRows, rows) - 1 : past - 1;
  b.window = a.window;
  b.sinks = a.sinks;
  b.span = span_of(b.p0, b.p1, a.window, a.sinks);
  b.step0 = split * a.chunk;
  b.step1 = min(b.step0 + a.chunk, b.span.n_steps);
  // The head's planes: rows past the last key read as zero (scales by whole words: their planes
  // are padded to 64).
  constexpr uint32_t kRowBytes = kD == kF32 ? 256 : kD == kF16 ? 128 : 64;
  const int64_t plane = a.plane[t] + h;
  auto rows_of = [&](const void* p, int64_t stride, uint32_t range) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(static_cast<const char*>(p)) + plane * stride, 0, range, kRawBuffer);
  };
  const uint32_t keys = static_cast<uint32_t>(b.p1) + 1u;
  b.k = rows_of(a.k, a.plane_rows * kRowBytes, keys * kRowBytes);
  b.v = rows_of(a.v, a.plane_rows * kRowBytes, keys * kRowBytes);
  if constexpr (kD == kI8) {
    b.ks = rows_of(a.k_scale, a.scale_rows, (keys + 3u) & ~3u);
    b.vs = rows_of(a.v_scale, a.scale_rows, (keys + 3u) & ~3u);
  }

  // Query rows: d = 16 g + 0..15 of row c of each tile, times scale * log2(e).
  f32x4 qx[kRT][4];
  int pos[kRT];
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    const int r = row0 + 16 * rt + c;
    pos[rt] = a.causal ? min(past + r, b.p1) : past - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) qx[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r < rows) {
      const float* qp = a.q + (q_row + r) * a.q_rs + h * 64 + 16 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qx[rt][i] = *reinterpret_cast<const f32x4u*>(qp + 4 * i) * a.scale_log2;
    }
  }

  Sums<kRT> st;
  bool f32_order = true;  // which column o[rt][dt][e] is
  if constexpr (kD == kF32) {
    attend_f32<kD, kRT>(b, qx, pos, wave, lane, st);
  } else {
    f32_order = attend_16<kD == kI8, kRT>(b, qx, pos, wave, lane, vs[wave], st);
    if constexpr (kD == kF16) {
      if (f32_order) attend_f32<kD, kRT>(b, qx, pos, wave, lane, st);
    }
  }

  // The waves' rows meet in LDS.
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    st.l[rt] = sum_x16_x32(st.l[rt]);
    float* const row = &mo[wave][(16 * rt + c) * kPitch];
    const f32x4(&o)[4] = st.o[rt];
    if (f32_order) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f32x4*>(row + 16 * g + 4 * e) =
            f32x4{o[0][e], o[1][e], o[2][e], o[3][e]};
    } else {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) *reinterpret_cast<f32x4*>(row + 16 * dt + 4 * g) = o[dt];
    }
    if (g == 0) {
      ml[wave][0][16 * rt + c] = st.m[rt];
      ml[wave][1][16 * rt + c] = st.l[rt];
    }
  }
  __syncthreads();
  // Thread (r, kCols columns from d0 on) adds the waves up, and the last of a block's chunks
  // to count in adds the chunks, in their order (exp2 domain).
  constexpr int kCols = kRows / kWaves;
  const int r = tid / (64 / kCols), d0 = kCols * (tid % (64 / kCols));
  const bool mine = row0 + r < rows;
  auto store = [&](float L, const float (&acc)[kCols]) {
    float* const op = a.o + (q_row + row0 + r) * a.o_rs + h * 64 + d0;
    const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int e = 0; e < kCols; e += 2)
      *reinterpret_cast<f32x2u*>(op + e) = f32x2{acc[e] * inv, acc[e + 1] * inv};
  };
  float M = -INFINITY, L = 0.f, acc[kCols] = {};
  {
    float mw[kWaves], lw[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      mw[w] = ml[w][0][r];
      lw[w] = ml[w][1][r];
      M = fmaxf(M, mw[w]);
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      // A wave without a maximum saw no key, or NaN scores only (sums of NaN, which 0 keeps).
      const float x = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw[w] - M);
      L = __builtin_fmaf(lw[w], x, L);
#pragma unroll
      for (int e = 0; e < kCols; ++e)
        acc[e] = __builtin_fmaf(mo[w][r * kPitch + d0 + e], x, acc[e]);
    }
  }
  if (n_split == 1) {
    if (mine) store(L, acc);
    return;
  }
  const int at = a.wg0[t] + (h * n_split) * n_blk + blk;  // the block's first chunk
  float* const part = a.part + (static_cast<int64_t>(at) * kRows + r) * kTreePart;
  const int64_t part_step = static_cast<int64_t>(n_blk) * kRows * kTreePart;  // to the next chunk
  if (mine) {
    float* const p = part + split * part_step;
    if (d0 == 0) st_agent2(p, M, L);
#pragma unroll
    for (int e = 0; e < kCols; e += 2) st_agent2(p + 2 + d0 + e, acc[e], acc[e + 1]);
  }
  // Every wave's stores are performed before the chunk counts in.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  unsigned* const counter = a.counters + static_cast<int64_t>(at) * kCounterStride;
  if (tid == 0)
    last_flag = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                static_cast<unsigned>(n_split - 1);
  __syncthreads();
  if (!last_flag) return;
  M = -INFINITY;
  L = 0.f;
#pragma unroll
  for (int e = 0; e < kCols; ++e) acc[e] = 0.f;
  for (int s0 = 0; mine && s0 < n_split; s0 += kMergeLoads) {
    float ms[kMergeLoads], ls[kMergeLoads], as[kMergeLoads][kCols];
#pragma unroll
    for (int j = 0; j < kMergeLoads; ++j) {
      // Chunks past the last one: that one again, without weight.
      const float* p = part + min(s0 + j, n_split - 1) * part_step;
      ld_agent2(p, ms[j], ls[j]);
#pragma unroll
      for (int e = 0; e < kCols; e += 2) ld_agent2(p + 2 + d0 + e, as[j][e], as[j][e + 1]);
    }
    float Mb = M;
#pragma unroll
    for (int j = 0; j < kMergeLoads; ++j) Mb = fmaxf(Mb, ms[j]);
    const float x = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - Mb);
    L *= x;
#pragma unroll
    for (int e = 0; e < kCols; ++e) acc[e] *= x;
#pragma unroll
    for (int j = 0; j < kMergeLoads; ++j) {
      if (s0 + j >= n_split) break;
      const float w = ms[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[j] - Mb);
      L = __builtin_fmaf(ls[j], w, L);
#pragma unroll
      for (int e = 0; e < kCols; ++e) acc[e] = __builtin_fmaf(as[j][e], w, acc[e]);
    }
    M = Mb;
  }
  if (mine) store(L, acc);
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Rows of a block.
int block_rows(const WindowArgs& a, DType) {
  int most = 0;
  for (int t = 0; t < a.n_seqs; ++t) most = std::max(most, a.rows[t]);
  return most > 16 ? 32 : 16;
}

}  // namespace

int64_t window_plan(WindowArgs& a, DType dt, bool split) {
  const int rows = block_rows(a, dt);
  int64_t blocks = 0, work = 0;
  int steps[kWindowMaxSeqs], longest = 1;  // of a sequence's longest block, at most
  for (int t = 0; t < a.n_seqs; ++t) {
    a.n_blk[t] = (a.rows[t] + rows - 1) / rows;
    const int64_t b = static_cast<int64_t>(a.n_blk[t]) * a.n_heads;
    const int p1 = a.past[t] - 1 + (a.causal ? a.rows[t] : 0);
    const int wide = std::min(a.rows[t], rows);
    const Span s = span_of(a.causal ? p1 - wide + 1 : p1, p1, a.window, a.sinks);
    // A block before the last may begin its window at another place within a step.
    steps[t] = s.n_steps + (a.n_blk[t] > 1 ? 1 : 0);
    steps[t] = std::min(steps[t], (p1 + kN) / kN);
    blocks += b;
    work += b * steps[t];
    longest = std::max(longest, steps[t]);
  }
  int64_t widest = 0;
  auto lay = [&](int64_t chunk) {
    int64_t sum = 0;
    widest = 0;
    a.chunk = static_cast<int>(chunk);
    for (int t = 0; t < a.n_seqs; ++t) {
      a.n_split[t] = static_cast<int>((steps[t] + chunk - 1) / chunk);
      a.blk_inv[t] = inverse(a.n_blk[t]);
      a.split_inv[t] = inverse(a.n_split[t]);
      a.wg0[t] = static_cast<int>(std::min<int64_t>(sum, 0x7fffffff));
      const int64_t n = static_cast<int64_t>(a.n_blk[t]) * a.n_heads * a.n_split[t];
      a.n_wgs[t] = static_cast<int>(std::min<int64_t>(n, 0x7fffffff));
      sum += n;
      widest = std::max(widest, n);
    }
    widest = (widest + 7) / 8 * 8;
    return sum;
  };
  const int whole = dt == kF32 ? 10 : 16, least = dt == kF32 ? 4 : 8;
  if (split && blocks < kTreeMaxWgs && longest > whole) {
    int64_t chunk = std::max<int64_t>(least, (work + kTreeMaxWgs - 1) / kTreeMaxWgs);
    for (chunk = (chunk + 3) / 4 * 4; chunk < longest; chunk += 4)
      if (lay(chunk) <= kTreeMaxWgs) return widest;
  }
  lay(longest);
  return widest;
}

hipError_t launch_window_attend(const WindowArgs& a, DType dt, int64_t wgs, hipStream_t s) {
  if (wgs <= 0) return hipSuccess;
  if (wgs > 0x7fffffff) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(wgs), a.n_seqs), block(64 * kWaves);
  const bool few = block_rows(a, dt) == 16;
#define WRS_WINDOW(D, RT) hipLaunchKernelGGL((window_attend<D, RT>), grid, block, 0, s, a)
  switch (dt) {
    case kF16:
      if (few) { WRS_WINDOW(kF16, 1); } else { WRS_WINDOW(kF16, 2); }
      break;
    case kF32:
      if (few) { WRS_WINDOW(kF32, 1); } else { WRS_WINDOW(kF32, 2); }
      break;
    case kI8:
      if (few) { WRS_WINDOW(kI8, 1); } else { WRS_WINDOW(kI8, 2); }
      break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_WINDOW
  return hipGetLastError();
}

}  // namespace wrs
