// Attention over the KV arena whose rows see a sliding window and the first tokens, and every
// attention over 8-bit arenas.
//
// K19 (window_attend): row r of a sequence stands at position p = past + r (`causal`; else every
//   row at the last key) and sees the keys j <= p with j > p - window or j < sinks:
//   s_j = q.k_j / 8, out = softmax(s) V over those j only.
//   A workgroup of four waves runs one block of 16 rows of one head. The block's keys are the
//   first tokens' 32-key steps, then those from its first row's window to its last row's own key:
//   steps in between are never read. Wave w takes steps w, w + 4, ... with an online softmax of its
//   own, the waves merge their (max, sum, O) in LDS, and where a block's steps are dealt over several
//   workgroups those merge through memory (the last to count in adds the partials up in order, so
//   results do not depend on which it is). Only steps that hold a key hidden from some row test keys.
//   f16 planes run on the f16 matrix pipe with f32 operands in two parts (Rows16), f32 planes on
//   the f32 pipe. 8-bit codes are whole numbers that f16 holds as they are: they enter the same way,
//   and the keys' powers of two go to the scores in f32, the values' to the weights before they are split.
//   One row of q a step costs what 16 do, so few rows are bound by latency: a step of a wave takes 0.7 us
//   from the load to the weights' product when it is alone on its SIMD (f32: 1.9), and window_plan
//   deals a block's steps over workgroups by that. Bytes are the other bound: 16 sequences of 20 heads
//   that see 8192 keys each (f16: 672 MB) take 121 us, 5.5 TB/s, and the 8-bit ones half the bytes in
//   80 us, 4.3 TB/s (three caches in turn; two, of which the L3 keeps a part, 68): with as many steps in
//   flight, each loads half. Deeper prefetch (2 to 4 steps), steps of 64 keys and 32 rows a wave were
//   measured and are no faster (79 to 88 us; registers then allow 2 or 3 waves a SIMD instead of 4).
#include "split16.hpp"

#include <algorithm>
#include <type_traits>

namespace wrs {
namespace {

using namespace split16;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kN = 32;              // keys per step
constexpr int kPitch = 68;          // LDS pitch (floats) of a merge row
constexpr int kCounterStride = 16;  // 64 bytes between merge counters
constexpr int kMergeLoads = 8;      // partials in flight per thread in the merge
constexpr int kRawBuffer = 0x00020000;  // buffer resource word 3: raw, 32-bit data format

// The steps of kSize keys of rows at positions p0..p1: `sink_steps` of them from key 0 on, the others
// from key `lo` on (a multiple of kSize), up to key p1. Where the two meet, all lie from key 0 on.
template <int kSize>
struct Span {
  int lo, sink_steps, n_steps;
  __host__ __device__ inline Span(int p0, int p1, int window, int sinks) {
    const int first = p0 - window + 1;  // window <= 2^24
    lo = first > 0 ? first / kSize * kSize : 0;
    sink_steps = (sinks < p1 + 1 ? sinks + kSize - 1 : p1 + kSize) / kSize;
    if (sink_steps * kSize >= lo) lo = sink_steps = 0;
    n_steps = sink_steps + (p1 - lo + kSize) / kSize;
  }
  __device__ inline int key_of(int step) const {
    return kSize * step + (step < sink_steps ? 0 : lo - kSize * sink_steps);
  }
};

// What a wave knows of its rows.
struct Block {
  int p0, p1;  // positions of the first and last row
  int window, sinks;
  Span<kN> span;
  int step0, step1;  // the workgroup's steps
  __amdgpu_buffer_rsrc_t k, v, ks, vs;  // the head's planes, zero past the last key

  __device__ inline Block(int first, int last, int w, int n)
      : p0(first), p1(last), window(w), sinks(n), span(first, last, w, n) {}
  __device__ inline int key_of(int step) const { return span.key_of(step); }
  // Whether some row sees one of `n` keys from j0 on.
  __device__ inline bool any(int j0, int n) const {
    return j0 <= p1 && (j0 + n - 1 > p0 - window || j0 < sinks);
  }
  // Whether some row of the block does not see some of `n` keys from j0 on.
  __device__ inline bool masked(int j0, int n) const {
    return j0 + n - 1 > p0 || (j0 <= p1 - window && j0 + n > sinks);
  }
  __device__ inline bool sees(int p, int j) const {
    return j <= p && (j > p - window || j < sinks);
  }
};

// A wave's running sums: of lane (c, g), row c.
struct Sums {
  f32x4 o[4];
  float m, l;
  __device__ inline void clear() {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
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
// row r, which are the B operand of O^T += V^T P^T as they stand. o[dt][e] is column 16 g + 4 e +
// dt. q: d = 16 g + 0..15 of row c, times scale * log2(e). pos: row c's position.
// Steps b.step0 + wave, + waves, .. of the block's, 16 keys at a time, the next 16 on their way.
template <DType kD>
__device__ inline void attend_f32(const Block& b, const f32x4 (&qx)[4], int pos,
                                  int wave, int waves, int lane, Sums& st) {
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
  // The wave's piece n: 16 keys of its step n / kPer.
  constexpr int kPer = kN / 16;
  const int steps = b.step1 - b.step0 - wave;
  const int end = steps > 0 ? kPer * ((steps + waves - 1) / waves) : 0;
  auto key_of = [&](int n) {
    return b.key_of(b.step0 + wave + waves * (n / kPer)) + 16 * (n % kPer);
  };
  if (end > 0) load(key_of(0));
  st.clear();
  for (int n = 0; n < end; ++n) {
    const int j0 = key_of(n);
    f32x4 kx[4], vx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kx[i] = kn[i];
      vx[i] = vn[i];
    }
    if (n + 1 < end) load(key_of(n + 1));
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
    f32x4 s0 = {}, s1 = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[i][e], qx[i][e], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[i][e + 1], qx[i][e + 1], s1, 0, 0, 0);
      }
    f32x4 s = s0 + s1;
    int seen = 0xF;  // bit i: the row sees key j0 + 4 g + i
    if (masked) {
      seen = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b.sees(pos, j0 + 4 * g + i))
          seen |= 1 << i;
        else
          s[i] = -INFINITY;
    }
    const float mx = max_x16_x32(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
    const float m_new = fmaxf(st.m, mx);
    const float alpha = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m - m_new);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    st.m = m_new;
    f32x4 p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(s[i] - m_use);
    st.l = __builtin_fmaf(st.l, alpha, (p[0] + p[1]) + (p[2] + p[3]));
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) st.o[dt] *= alpha;
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
            if (vis && !__builtin_isfinite(vk[dt])) st.o[dt][e] += pk * vk[dt];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
        st.o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(
            odd && !__builtin_isfinite(vx[i][dt]) ? 0.f : vx[i][dt], p[i], st.o[dt], 0, 0, 0);
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
__device__ inline void codes_f16(const u32x4& w, u32x4 (&out)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo, hi;
    codes_f16(w[i], lo, hi);
    out[i >> 1][2 * (i & 1)] = lo;
    out[i >> 1][2 * (i & 1) + 1] = hi;
  }
}
// 2^(byte - 127) of byte i of four scales (255: infinity, and its codes are zeros: NaN).
__device__ inline float scale_at(uint32_t w, int i) {
  return __builtin_bit_cast(float, ((w >> (8 * i)) & 0xFFu) << 23);
}

// The values' operand of columns 16 dt.. from 32 rows of V in LDS: lane (c, g) gets column 16 dt + c of
// keys 4 g + 0..3 and 16 + 4 g + 0..3, the order that the packed weights have. Chunk c of 16 bytes of row r
// sits at c ^ vswz(r): four rows' pairs of chunks, and two rows' chunks of one parity (which a wave
// stores together from 8-bit codes: with rows of one parity 32 of 100 LDS cycles a step were conflicts),
// hit distinct banks. Rows r and r + 16 swizzle alike.
__device__ inline int vswz(int r) { return (2 * (r & 3)) | (r & 1); }
__device__ inline int value_offset(int dt, int c, int g) {
  const int row = 4 * g + (c >> 2);
  return row * 128 + (((2 * dt + ((c & 3) >> 1)) ^ vswz(row)) * 16) + 8 * (c & 1);
}
__device__ inline u32x4 value_operand(const char* v) {
  const u32x2 a = read_tr(v), b = read_tr(v + 2048);
  return u32x4{a.x, a.y, b.x, b.y};
}

// Two weights (below 2^16) as packed f16 pairs in two parts of one unit: to nearest, and what that
// leaves.
__device__ inline void split_weights(float x0, float x1, uint32_t (&out)[2]) {
  const f32x2 x = {x0, x1};
  uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, f16x2));
  asm("" : "+v"(w));  // formed once, not again by each element that the rest takes
  const f16x2 h = __builtin_bit_cast(f16x2, w);
  float one = 1.f;
  asm("" : "+s"(one));  // so that a remainder is one mixed fma, not a subtraction and a conversion
  const f16x2 l = {static_cast<_Float16>(__builtin_fmaf(x0, one, -static_cast<float>(h[0]))),
                   static_cast<_Float16>(__builtin_fmaf(x1, one, -static_cast<float>(h[1])))};
  out[0] = w;
  out[1] = __builtin_bit_cast(uint32_t, l);
}

// Rows of a wave on the f16 matrix pipe: lane (c, g) has row c of each tile of 16.
//   Query rows, times a power of two that puts the largest element into [2^14, 2^15), and weights
//   are split into two f16 parts in one unit, whose products add up in one chain: within 2^-22 of
//   themselves, small ones within 2^-40 of the row's largest element and 2^-31 of its largest weight.
//   Weights are taken against a reference, the row's maximum so far or less than kRoom below it (a whole
//   number, so that what is taken off the exponents is the reference that sums are joined by, exactly),
//   so that the sums are scaled only where a score passes that (for a row's first step and hardly
//   ever after), and times a unit 2^u, which the quotient at the end drops. 8-bit values have powers of
//   two, which go to the weights; the largest product of the two sets the unit, so that rows of
//   any scale meet in one sum (values of 2^-80 and more to 2^-22 of the largest product).
constexpr float kRoom = 8.f;
constexpr float kUnit = 7.f;      // f16 planes: weights below 2^15
constexpr float kMostUnit = 87.f;  // 8-bit planes: 2^24 weights of 2^kRoom stay below f32's largest
template <bool k8>
struct Rows16 {
  u32x4 qf[2][2];  // d = 16 g + 8 kk + 0..7
  float down;      // the inverse of the rows' power of two
  f32x4 o[4];      // column 16 dt + 4 g + e
  float m, l;
  float unit;
  float zero;   // what exponents are taken against: the reference (0 before there is one), less the unit
  float limit;  // a score past this (before `down`) moves the reference

  __device__ inline void start(const f32x4 (&qx)[4]) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) amax = fmaxf(amax, __builtin_fabsf(qx[i][e]));
    amax = max_x16_x32(amax);
    const int e_max = static_cast<int>((__builtin_bit_cast(uint32_t, amax) >> 23) & 0xFF);
    const int sh = e_max == 0 ? 0 : clamp_exp(141 - e_max);
    const float x = pow2(sh);
    down = pow2(clamp_exp(-sh));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t w[2];
      split2(qx[i >> 1][2 * (i & 1)], qx[i >> 1][2 * (i & 1) + 1], x, w);
#pragma unroll
      for (int p = 0; p < 2; ++p) qf[p][i >> 2][i & 3] = w[p];
    }
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = limit = -INFINITY;
    l = 0.f;
    unit = k8 ? kMostUnit : kUnit;
    zero = -unit;
  }

  // 32 keys from j0 on: their operands (key 16 t + c, d = 16 g + 8 kk + 0..7), the powers of two of keys
  // 16 t + 4 g + i and of their values, and values(dt), the values' operand of columns 16 dt.. .
  template <typename V>
  __device__ inline void step(const Block& b, int pos, int j0, int g,
                              const u32x4 (&kf)[2][2], const float (&ks)[2][4],
                              const float (&vs)[2][4], V values) {
    const bool masked = b.masked(j0, kN);
    u32x4 pf[2], va[4];
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 1; p >= 0; --p)  // the smaller part first
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          s[t] = mfma16(kf[t][kk], qf[p][kk], s[t]);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) va[dt] = values(dt);  // on their way under the softmax
    // Register i of tile t holds key 16 t + 4 g + i.
    if constexpr (k8) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[t][i] *= ks[t][i];
    }
    if (masked) {
      asm volatile("");  // a branch: whole steps pay for no selection
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!b.sees(pos, j0 + 16 * t + 4 * g + i)) s[t][i] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(s[0][0], s[0][1]), s[0][2]);
    mx = fmaxf(fmaxf(mx, s[0][3]), s[1][0]);
    mx = fmaxf(fmaxf(mx, s[1][1]), s[1][2]);
    mx = fmaxf(mx, s[1][3]);
    if (__any(mx > limit)) {
      const float m_new = fmaxf(m, ceilf(max_x16_x32(mx) * down)), d = m_new - m;
      // The products so far fall with the weights, so 8-bit planes' unit may rise as much.
      const float u = k8 ? fminf(unit + d, kMostUnit) : kUnit;
      move(m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((u - unit) - d));
      unit = u;
      m = m_new;
      zero = (m_new == -INFINITY ? 0.f : m_new) - u;
      limit = (m_new + kRoom) / down;  // a power of two
    }
    float p[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        p[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], down, -zero));
    if constexpr (k8) {
      float w[2][4];
      auto weigh = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) w[t][i] = p[t][i] * vs[t][i];
        if (masked) {
          // A hidden row's scale may be the NaN one: it takes no part.
          asm volatile("");
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (s[t][i] == -INFINITY) w[t][i] = 0.f;
        }
        float top = fmaxf(fmaxf(w[0][0], w[0][1]), w[0][2]);
        top = fmaxf(fmaxf(top, w[0][3]), w[1][0]);
        top = fmaxf(fmaxf(top, w[1][1]), w[1][2]);
        return fmaxf(top, w[1][3]);
      };
      float top = weigh();
      // Twice at most: a product past f32's range has e of 128, and is in range once that is taken off
      // (a NaN row's never is).
      for (int turn = 0; turn < 2 && __any(top > 0x1p15f); ++turn) {
        // The largest comes to [2^7, 2^8): 2^e <= it < 2^(e + 1).
        top = max_x16_x32(top);
        const int e = static_cast<int>(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
        const float u = fminf(unit, unit + 7.f - static_cast<float>(e));
        const float x = __builtin_amdgcn_exp2f(u - unit);
        move(x);
        zero += unit - u;
        unit = u;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            p[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], down, -zero));
        top = weigh();
      }
      l += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) +
               ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[t][i] = w[t][i];
    } else {
      l += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) +
               ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        uint32_t w[2];
        split_weights(p[t][i], p[t][i + 1], w);
#pragma unroll
        for (int q = 0; q < 2; ++q) pf[q][2 * t + (i >> 1)] = w[q];
      }
#pragma unroll
    for (int p = 1; p >= 0; --p)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
        o[dt] = mfma16(va[dt], pf[p], o[dt]);
  }
  // The row's sums so far, times x.
  __device__ inline void move(float x) {
    l *= x;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[dt] *= x;
  }

  // The sums without their unit. Returns whether one came out infinite or NaN: parts of an infinity
  // are not numbers, so a wave over f16 planes starts again with f32 operands.
  __device__ inline bool finish() {
    bool odd = false;
    const float x = __builtin_amdgcn_exp2f(-unit);
    move(x);
    odd |= !__builtin_isfinite(l);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= !__builtin_isfinite(o[dt][e]);
    return !k8 && __any(odd);
  }
};

// A wave's steps of an f16 or 8-bit plane. K comes from memory in operand layout, V passes through
// the wave's own swizzled LDS rows and is read transposed; the packed weights are the B operand of
// O^T += V^T P^T as they stand. Returns whether the wave has to start again with f32 operands.
template <bool k8>
__device__ inline bool attend_16(const Block& b, const f32x4 (&qx)[4], int pos,
                                 int wave, int lane, char* vw, Rows16<k8>& r) {
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
  int step = b.step0 + wave;
  if (step < b.step1) load(b.key_of(step));
  r.start(qx);
  for (; step < b.step1; step += kWaves) {
    u32x4 kf[2][2];
    float kscale[2][4], vscale[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (k8) {
        codes_f16(kx[t][0], kf[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kscale[t][i] = scale_at(ks[t], i);
          vscale[t][i] = scale_at(vs[t], i);
        }
      } else {
        kf[t][0] = kx[t][0];
        kf[t][1] = kx[t][kK - 1];
      }
    }
    wave_sync();  // the last step's transposed reads are done
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      if constexpr (k8) {
        const int row = 16 * i + (lane >> 2);
        u32x4 y[2];
        codes_f16(vx[i], y);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<u32x4*>(vw + row * 128 + (((2 * (lane & 3) + e) ^ vswz(row)) * 16)) = y[e];
      } else {
        const int row = 8 * i + (lane >> 3);
        *reinterpret_cast<u32x4*>(vw + row * 128 + (((lane & 7) ^ vswz(row)) * 16)) = vx[i];
      }
    }
    wave_sync();
    if (step + kWaves < b.step1) load(b.key_of(step + kWaves));
    r.step(b, pos, b.key_of(step), g, kf, kscale, vscale, [&](int dt) __attribute__((always_inline)) {
      return value_operand(vw + value_offset(dt, c, g));
    });
  }
  return r.finish();
}

// The head's planes: rows past the `keys` first read as zero (scales by whole words: their planes
// are padded to 64).
template <DType kD, int kSeqs>
__device__ inline void set_planes(const WindowArgs<kSeqs>& a, int64_t plane, uint32_t keys, Block& b) {
  constexpr uint32_t kRowBytes = kD == kF32 ? 256 : kD == kF16 ? 128 : 64;
  auto rows_of = [&](const void* p, int64_t stride, uint32_t range) __attribute__((always_inline)) {
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(static_cast<const char*>(p)) + plane * stride, 0, range, kRawBuffer);
  };
  b.k = rows_of(a.k, a.plane_rows * kRowBytes, keys * kRowBytes);
  b.v = rows_of(a.v, a.plane_rows * kRowBytes, keys * kRowBytes);
  if constexpr (kD == kI8) {
    b.ks = rows_of(a.k_scale, a.scale_rows, (keys + 3u) & ~3u);
    b.vs = rows_of(a.v_scale, a.scale_rows, (keys + 3u) & ~3u);
  }
}
// Query row r0 + c of a sequence (of `rows`): d = 16 g + 0..15, times scale * log2(e), and
// where they stand (rows past the last one are zero and stand at the last key, p1).
template <int kSeqs>
__device__ inline void load_rows(const WindowArgs<kSeqs>& a, int t, int h, int r0, int p1, int c, int g,
                                 f32x4 (&qx)[4], int& pos) {
  const int past = a.past[t], rows = a.rows[t];
  const int r = r0 + c;
  pos = a.causal ? min(past + r, p1) : past - 1;
#pragma unroll
  for (int i = 0; i < 4; ++i) qx[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (r < rows) {
    const float* qp = a.q + (a.row0[t] + r) * a.q_rs + h * 64 + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qx[i] = *reinterpret_cast<const f32x4u*>(qp + 4 * i) * a.scale_log2;
  }
}

// The workgroup's sequence, and which of the sequence's workgroups it is. There is none without one:
// with a grid as wide as the widest sequence the dispatcher put the others' workgroups on few CUs
// (16 single tokens over 8192 keys and a text of 256 rows, 20 heads, f16: 533 us, now 141).
template <int kSeqs>
__device__ inline int sequence_of(const WindowArgs<kSeqs>& a, int& lid) {
  lid = a.remap ? xcd_remap(blockIdx.x, gridDim.x) : blockIdx.x;
  if (a.n_seqs == 1) return 0;
  if (a.like) {
    return divide(lid, a.n_wgs[0], a.wgs_inv, lid);
  }
  // Those past the last sequence start past every workgroup.
  int t = -1;
  for (int i = 0; i < a.n_seqs; i += 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) t += a.wg0[i + j] <= lid;
  }
  lid -= a.wg0[t];
  return t;
}

// The square root of what sums against `m` weigh against `all` (at or above it): a sum whose weight is
// past f32's range may still count, where its values are as much larger.
__device__ inline float half_weight(float m, float all) {
  return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(0.5f * (m - all));
}

template <DType kD, int kSeqs>
__global__ __launch_bounds__(64 * kWaves, 4) void window_attend(WindowArgs<kSeqs> a) {
  constexpr int kRows = 16;
  __shared__ __attribute__((aligned(128))) char vs[kD == kF32 ? 1 : kWaves][kN * 128];
  __shared__ __attribute__((aligned(16))) float mo[kWaves][kRows * kPitch];  // a wave's O rows
  __shared__ float ml[kWaves][2][kRows];  // and their max and sum
  __shared__ int last_flag;

  // Chunks of one sequence or of like ones: the workgroups of one head's keys, which read the same rows,
  // share an XCD's L2. Whole blocks: the last ones of all heads first, which have the most keys
  // (1000 rows on each other, 20 heads, 8-bit: 17.7 us, 22.1 with the heads on an XCD each).
  int lid;
  const int t = sequence_of(a, lid);
  const int past = a.past[t], rows = a.rows[t];
  const int n_blk = a.n_blk[t], n_split = a.n_split[t];
  int blk, split = 0, h;
  if (n_split > 1) {
    const int hs = divide(lid, n_blk, a.blk_inv[t], blk);
    h = divide(hs, n_split, a.split_inv[t], split);
  } else {
    blk = n_blk - 1 - divide(lid, a.n_heads, a.head_inv, h);
  }
  const int row0 = blk * kRows;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t q_row = a.row0[t];

  Block b(a.causal ? past + row0 : past - 1,
          a.causal ? past + min(row0 + kRows, rows) - 1 : past - 1, a.window, a.sinks);
  b.step0 = split * a.chunk;
  b.step1 = min(b.step0 + a.chunk, b.span.n_steps);
  set_planes<kD>(a, a.plane[t] + h, static_cast<uint32_t>(b.p1) + 1u, b);
  f32x4 qx[4];
  int pos;
  load_rows(a, t, h, row0, b.p1, c, g, qx, pos);

  Sums st;
  bool f32_order = true;  // which column o[dt][e] is
  if constexpr (kD != kF32) {
    Rows16<kD == kI8> r;
    f32_order = attend_16<kD == kI8>(b, qx, pos, wave, lane, vs[wave], r);
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) st.o[dt] = r.o[dt];
    st.m = r.m;
    st.l = r.l;
  }
  if constexpr (kD != kI8) {
    if (f32_order) {
      // The rows again, rather than kept through the steps.
      if (kD == kF16) load_rows(a, t, h, row0, b.p1, c, g, qx, pos);
      attend_f32<kD>(b, qx, pos, wave, kWaves, lane, st);
    }
  }

  // The waves' rows meet in LDS.
  st.l = sum_x16_x32(st.l);
  float* const row = &mo[wave][(c) * kPitch];
  const f32x4(&o)[4] = st.o;
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
    ml[wave][0][c] = st.m;
    ml[wave][1][c] = st.l;
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
      const float x = half_weight(mw[w], M);
      L = __builtin_fmaf(lw[w] * x, x, L);
#pragma unroll
      for (int e = 0; e < kCols; ++e)
        acc[e] = __builtin_fmaf(mo[w][r * kPitch + d0 + e] * x, x, acc[e]);
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
    const float x = half_weight(M, Mb);
    L = L * x * x;
#pragma unroll
    for (int e = 0; e < kCols; ++e) acc[e] = acc[e] * x * x;
#pragma unroll
    for (int j = 0; j < kMergeLoads; ++j) {
      if (s0 + j >= n_split) break;
      const float w = half_weight(ms[j], Mb);
      L = __builtin_fmaf(ls[j] * w, w, L);
#pragma unroll
      for (int e = 0; e < kCols; ++e) acc[e] = __builtin_fmaf(as[j][e] * w, w, acc[e]);
    }
    M = Mb;
  }
  if (mine) store(L, acc);
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// K20 (window_tiles): the same for many rows. A workgroup of four waves takes 64 rows of one head, 16 a
//   wave, and goes through their keys in tiles of 64 that pass through LDS once for all four, so that K
//   and V are read and widened for 64 rows; a wave leaves out the halves of a tile that none of its rows
//   see. No merge: a wave has its rows to itself. Blocks start with the last ones of every head, which
//   see the most keys (4000 rows on each other, 20 heads, f16: 99 us; heads in turn: 175).
//   Bound by what a wave issues (the softmax and the split of its weights, vector pipe 55%, next to
//   29% of the matrix pipe): 4000 rows take 41 GFLOP each for scores and outputs (two parts), 0.83
//   PFLOP/s, of 1.26 that a large product reaches here. 32 rows a wave halve the LDS reads, but leave 2 or
//   3 waves a SIMD and half the blocks (110 us; 1500 rows: 39 us, 26 with 16 rows a wave).
constexpr int kTile = 64;
constexpr int kTileRows = 64;
__device__ inline int kswz(int r) { return (r >> 1) & 7; }  // 16 rows' equal chunks hit distinct banks

template <bool k8, int kSeqs>
__global__ __launch_bounds__(64 * kWaves, 4) void window_tiles(WindowArgs<kSeqs> a) {
  constexpr int kPieces = k8 ? 1 : 2;  // 16-byte pieces of a tile's K (or V) a thread
  constexpr DType kD = k8 ? kI8 : kF16;
  __shared__ __attribute__((aligned(128))) char kt[2][kTile * 128], vt[2][kTile * 128];
  __shared__ __attribute__((aligned(16))) float st[2][2][k8 ? kTile : 4];  // K's and V's powers of two
  int lid;
  const int t = sequence_of(a, lid);
  const int past = a.past[t], rows = a.rows[t];
  int h;
  const int blk = a.n_blk[t] - 1 - divide(lid, a.n_heads, a.head_inv, h);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int first = blk * kTileRows, row0 = first + 16 * wave;
  // The block's tiles, and the wave's rows (a wave past the last row only loads).
  const int p1 = a.causal ? past + min(first + kTileRows, rows) - 1 : past - 1;
  const Span<kTile> span(a.causal ? past + first : past - 1, p1, a.window, a.sinks);
  const bool idle = row0 >= rows;
  Block b(a.causal ? past + min(row0, rows - 1) : past - 1,
          a.causal ? past + min(row0 + 16, rows) - 1 : past - 1, a.window, a.sinks);
  b.step0 = 0;
  b.step1 = b.span.n_steps;
  set_planes<kD>(a, a.plane[t] + h, static_cast<uint32_t>(p1) + 1u, b);

  u32x4 kx[kPieces], vx[kPieces];
  uint32_t sx = 0;
  auto load = [&](int j0) __attribute__((always_inline)) {
    const uint32_t o = static_cast<uint32_t>(j0) * (64u * kPieces) + 16u * tid;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      kx[i] = __builtin_bit_cast(u32x4,
                                 __builtin_amdgcn_raw_buffer_load_b128(b.k, o + 4096 * i, 0, 0));
      vx[i] = __builtin_bit_cast(u32x4,
                                 __builtin_amdgcn_raw_buffer_load_b128(b.v, o + 4096 * i, 0, 0));
    }
    if constexpr (k8) {
      if (tid < 2 * kTile) {
        const uint32_t so = static_cast<uint32_t>(j0 + (tid & (kTile - 1)));
        sx = tid < kTile ? __builtin_amdgcn_raw_buffer_load_b8(b.ks, so, 0, 0)
                         : __builtin_amdgcn_raw_buffer_load_b8(b.vs, so, 0, 0);
      }
    }
  };
  auto put = [&](char* p, int row, int chunk, int swizzle, const u32x4& x)
                 __attribute__((always_inline)) {
    *reinterpret_cast<u32x4*>(p + row * 128 + ((chunk ^ swizzle) * 16)) = x;
  };
  auto store = [&](int buf) __attribute__((always_inline)) {
    if constexpr (k8) {
      const int row = tid >> 2, chunk = 2 * (tid & 3);
      u32x4 y[2];
      codes_f16(kx[0], y);
      put(kt[buf], row, chunk, kswz(row), y[0]);
      put(kt[buf], row, chunk + 1, kswz(row), y[1]);
      codes_f16(vx[0], y);
      put(vt[buf], row, chunk, vswz(row), y[0]);
      put(vt[buf], row, chunk + 1, vswz(row), y[1]);
      if (tid < 2 * kTile) st[buf][tid >= kTile][tid & (kTile - 1)] = scale_at(sx, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int row = 32 * i + (tid >> 3), chunk = tid & 7;
        put(kt[buf], row, chunk, kswz(row), kx[i]);
        put(vt[buf], row, chunk, vswz(row), vx[i]);
      }
    }
  };
  load(span.key_of(0));
  f32x4 qx[4];
  int pos;
  load_rows(a, t, h, row0, b.p1, c, g, qx, pos);
  Rows16<k8> r;
  r.start(qx);
  store(0);
  if (span.n_steps > 1) load(span.key_of(1));
  __syncthreads();
  // A lane's places in a tile: its share of a key, and the values of its columns.
  int k_at[2], v_at[4];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) k_at[kk] = c * 128 + (((2 * g + kk) ^ kswz(c)) * 16);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) v_at[dt] = value_offset(dt, c, g);
  for (int i = 0; i < span.n_steps; ++i) {
    const int buf = i & 1;
    if (i + 1 < span.n_steps) {
      store(buf ^ 1);  // last read before the last barrier
      if (i + 2 < span.n_steps) load(span.key_of(i + 2));
    }
    const char *const kp = kt[buf], *const vp = vt[buf];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int j0 = span.key_of(i) + kN * half;
      if (idle || !b.any(j0, kN)) continue;
      u32x4 kf[2][2];
      float ks[2][4], vs[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int at = kN * half + 16 * u;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
          kf[u][kk] = *reinterpret_cast<const u32x4*>(kp + k_at[kk] + 128 * at);
        if constexpr (k8) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(&st[buf][0][at + 4 * g]);
          const f32x4 y = *reinterpret_cast<const f32x4*>(&st[buf][1][at + 4 * g]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            ks[u][e] = x[e];
            vs[u][e] = y[e];
          }
        }
      }
      r.step(b, pos, j0, g, kf, ks, vs, [&](int dt) __attribute__((always_inline)) {
        return value_operand(vp + v_at[dt] + 4096 * half);
      });
    }
    __syncthreads();
  }
  bool f32_order = r.finish();  // which column o[dt][e] is
  if constexpr (!k8) {
    if (f32_order) {
      Sums sums;
      load_rows(a, t, h, row0, b.p1, c, g, qx, pos);  // again, rather than kept so long
      attend_f32<kD>(b, qx, pos, 0, 1, lane, sums);
      r.l = sums.l;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) r.o[dt] = sums.o[dt];
    }
  }
  const float l = sum_x16_x32(r.l), inv = l == 0.f ? 0.f : 1.f / l;
  const int row = row0 + c;
  if (row >= rows) return;
  float* const op = a.o + (a.row0[t] + row) * a.o_rs + h * 64;
  const f32x4(&o)[4] = r.o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x4 x = f32_order ? f32x4{o[0][i], o[1][i], o[2][i], o[3][i]} : o[i];
    *reinterpret_cast<f32x4u*>(op + (f32_order ? 16 * g + 4 * i : 16 * i + 4 * g)) = x * inv;
  }
}

// Rows of a block: 64 where their tiles of 64 keys, in whole blocks, come to 150 times the longest block's
// own (8-bit planes, of which blocks of 16 rows read half the bytes: 400), so that no block runs on
// alone. Measured, tiles against blocks of 16 at so many times: 20 heads of rows on each other, f16 1000
// rows (170) 19.3 us against 19.7, 1500 (250) 26 against 34, 4000 (630) 99 against 183; 8 heads of 1500
// rows (100) 23.4 against 17.8, 3500 (220) 54 against 61; 8-bit 1500 rows (250) 35 against 29, 2500 (410)
// 60 against 66, 4000 (630) 107 against 146. A single token is 1/64 of a block: 39 of them over 8192 keys
// with a text of 64 or 256 rows, 8-bit, 192 and 192 us against 179 and 168 (with 2000 rows 287 and 237; 16 of
// them with 2000 rows, f16 (163) 172 us against 242, 8-bit (163) 208 and 153).
template <int kSeqs>
int block_rows(const WindowArgs<kSeqs>& a, DType dt) {
  if (dt == kF32) return 16;
  int64_t work = 0;
  int longest = 1;
  for (int t = 0; t < a.n_seqs; ++t) {
    auto steps = [&](int row0, int row1) {
      const int p1 = a.past[t] - 1 + (a.causal ? row1 : 0);
      return Span<kTile>(a.causal ? a.past[t] + row0 : p1, p1, a.window, a.sinks).n_steps;
    };
    const int rows = a.rows[t], part = std::min(rows, kTileRows);
    const int last = steps(rows - part, rows);
    work += static_cast<int64_t>(rows) * (steps(0, part) + last);
    longest = std::max(longest, last);
  }
  return work * a.n_heads / (2 * kTileRows) >= (dt == kI8 ? 400 : 150) * static_cast<int64_t>(longest)
             ? kTileRows
             : 16;
}

// Steps of the longest block of a sequence, at most.
template <int kSeqs>
int most_steps(const WindowArgs<kSeqs>& a, int t, int rows) {
  const int p1 = a.past[t] - 1 + (a.causal ? a.rows[t] : 0), wide = std::min(a.rows[t], rows);
  const Span<kN> s(a.causal ? p1 - wide + 1 : p1, p1, a.window, a.sinks);
  // A block before the last may begin its window at another place within a step.
  return std::min(s.n_steps + (a.rows[t] > rows ? 1 : 0), (p1 + kN) / kN);
}

}  // namespace

template <int kSeqs>
int64_t window_plan(WindowArgs<kSeqs>& a, DType dt, bool split) {
  const int rows = a.block_rows = block_rows(a, dt);
  int steps[kSeqs], longest = 1;
  int64_t work = 0;
  for (int t = 0; t < a.n_seqs; ++t) {
    a.n_blk[t] = (a.rows[t] + rows - 1) / rows;
    steps[t] = most_steps(a, t, rows);
    longest = std::max(longest, steps[t]);
    work += static_cast<int64_t>(a.n_blk[t]) * a.n_heads * steps[t];
  }
  a.head_inv = inverse(a.n_heads);
  auto lay = [&](int64_t chunk) {
    int64_t sum = 0;
    a.like = a.remap = 1;
    a.chunk = static_cast<int>(chunk);
    for (int t = 0; t < a.n_seqs; ++t) {
      a.n_split[t] = static_cast<int>((steps[t] + chunk - 1) / chunk);
      a.blk_inv[t] = inverse(a.n_blk[t]);
      a.split_inv[t] = inverse(a.n_split[t]);
      a.wg0[t] = static_cast<int>(std::min<int64_t>(sum, 0x7fffffff));
      const int64_t n = static_cast<int64_t>(a.n_blk[t]) * a.n_heads * a.n_split[t];
      a.n_wgs[t] = static_cast<int>(std::min<int64_t>(n, 0x7fffffff));
      sum += n;
      a.like &= a.n_wgs[t] == a.n_wgs[0];
      a.remap &= a.n_split[t] > 1;
    }
    for (int t = a.n_seqs; t < kSeqs; ++t) a.wg0[t] = 0x7fffffff;
    a.wgs_inv = inverse(a.n_wgs[0]);
    return sum;
  };
  int64_t chunk = longest;
  if (split && rows == 16) {
    // What a launch takes, in us, next to its fixed 3.5: the fullest CU's workgroups share it (a step
    // alone 0.7, f32 1.9), and chunks cost their merge, in turns of kMergeLoads.
    const float alone = dt == kF32 ? 0.95f : 0.25f, each = dt == kF32 ? 0.95f : 0.45f;
    float best = 0.f;
    for (int n = 1; n <= 256; n += n < 4 ? 1 : n & (n - 1) ? n / 3 : n / 2) {
      const int c = ((longest + n - 1) / n + kWaves - 1) / kWaves * kWaves;
      int64_t wgs = 0;
      for (int t = 0; t < a.n_seqs; ++t)
        wgs += static_cast<int64_t>(a.n_blk[t]) * a.n_heads * ((steps[t] + c - 1) / c);
      if (n > 1 && wgs > 2 * kTreeMaxWgs) break;  // what the scratch takes, of 16 rows
      const int64_t turn = static_cast<int64_t>(c) * 256;
      float us = static_cast<float>(c / kWaves) *
                 (alone + each * static_cast<float>(std::max<int64_t>((work + turn - 1) / turn, 1)));
      if (n > 1)
        us += 1.1f + 0.7f * static_cast<float>((n + kMergeLoads - 1) / kMergeLoads) +
              static_cast<float>(wgs) / 240.f;
      if (n == 1 || us < best) {
        best = us;
        chunk = n == 1 ? longest : c;
      }
    }
  }
  return lay(chunk);
}

template <int kSeqs>
hipError_t launch_window_attend(const WindowArgs<kSeqs>& a, DType dt, int64_t wgs, hipStream_t s) {
  if (wgs <= 0) return hipSuccess;
  if (wgs > 0x7fffffff) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(wgs)), block(64 * kWaves);
  const bool tiles = a.block_rows == kTileRows;
#define WRS_WINDOW(K, ...) hipLaunchKernelGGL((K<__VA_ARGS__, kSeqs>), grid, block, 0, s, a)
  switch (dt) {
    case kF16:
      if (tiles) { WRS_WINDOW(window_tiles, false); } else { WRS_WINDOW(window_attend, kF16); }
      break;
    case kF32: WRS_WINDOW(window_attend, kF32); break;
    case kI8:
      if (tiles) { WRS_WINDOW(window_tiles, true); } else { WRS_WINDOW(window_attend, kI8); }
      break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_WINDOW
  return hipGetLastError();
}

template int64_t window_plan(WindowArgs<kWindowMaxSeqs>&, DType, bool);
template int64_t window_plan(WindowArgs<kWindowFewSeqs>&, DType, bool);
template hipError_t launch_window_attend(const WindowArgs<kWindowMaxSeqs>&, DType, int64_t,
                                         hipStream_t);
template hipError_t launch_window_attend(const WindowArgs<kWindowFewSeqs>&, DType, int64_t,
                                         hipStream_t);

}  // namespace wrs
