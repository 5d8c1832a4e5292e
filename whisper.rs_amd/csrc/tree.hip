// Attention of drafted trees over the KV arena.
//
// K11 (tree_attend): the rows of a tree of drafted tokens against one slot's cache.
//   Row i of a tree sees the slot's `past` keys and, of the drafted rows stored
//   behind them, itself and its ancestors: s_j = q_i.k_j / 8, out_i = softmax(s) V
//   over those j only. parents[i] in [0, i) is the row's parent; anything else
//   makes it a child of the last cached token, so any parents end every walk.
//   A workgroup of four waves runs one block of 16 kRT rows of one head over one
//   chunk of the keys; wave w takes the chunk's steps w, w + 4, ... (of 16 f32 keys or
//   32 f16 ones) with an online softmax of its own, the waves merge their (max, sum, O)
//   in LDS, and the chunks of a block merge through memory (the last workgroup to count
//   in adds the partials up in chunk order, so results do not depend on which it is).
//   Only the steps that reach past the cache test the ancestor bits.
//   f16 planes run on the f16 matrix pipe with operands in two parts, f32 ones on the
//   f32 matrix pipe.
//   Short caches are bound by latency: 8 nodes over 60 keys, 6 heads 5.0 us, five trees of up to
//   26 over 223, 20 heads 6.2, four of 13 over 430, 12 heads f32 8.2 (smallest launch 2.3).
//   Long ones by the chain from scores to weights to products, whose vector instructions hold the
//   SIMDs 39% of the time and whose MFMAs 19%: 64 nodes x 20 heads over 65471 f16 keys 94 us, 3.5
//   TB/s of K and V (floor 66), 16 nodes 73 us, 4.6 TB/s.
#include "split16.hpp"

#include <algorithm>

namespace wrs {
namespace {

using namespace split16;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2u __attribute__((ext_vector_type(2), aligned(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kStep = 16;       // keys per wave step of the f32 path
constexpr int kPitch = 68;      // LDS pitch (floats) of a merge row
constexpr int kCounterStride = 32;  // 128 bytes between merge counters
constexpr int kMergeLoads = 8;  // partials in flight per thread in the merge
constexpr int kRawBuffer = 0x00020000;  // buffer resource word 3: raw, 32-bit data format

// Two floats at once, as st_agent and ld_agent (8-byte aligned).
__device__ inline void st_agent2(float* p, float x, float y) {
  const uint64_t v = __builtin_bit_cast(uint32_t, x) |
                     static_cast<uint64_t>(__builtin_bit_cast(uint32_t, y)) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline void ld_agent2(const float* p, float& x, float& y) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  x = __builtin_bit_cast(float, static_cast<uint32_t>(v));
  y = __builtin_bit_cast(float, static_cast<uint32_t>(v >> 32));
}

// 4 values of a plane row at byte offset `o` (multiple of 4 values), zero past the range.
template <typename KT>
__device__ inline f32x4 load4(const __amdgpu_buffer_rsrc_t& rs, uint32_t o) {
  if constexpr (sizeof(KT) == 4)
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0));
  else
    return __builtin_convertvector(
        __builtin_bit_cast(f16x4, __builtin_amdgcn_raw_buffer_load_b64(rs, o, 0, 0)), f32x4);
}

// What a wave knows of its block and chunk.
struct Block {
  int past, nodes;      // keys that every row sees, drafted rows behind them
  int key0, key1;       // the workgroup's keys
  int row0;             // its first row within the tree
  const uint32_t* anc;  // LDS: words of ancestors-or-self per row, and one of zeros
  __amdgpu_buffer_rsrc_t k, v;  // the chunk's rows of the head's planes, zero at key1
};
// Which drafted rows the rows of a block see: ancestors-or-self of row c of each tile. Trees of
// up to 64 nodes are worked out by every wave for itself, in registers; larger ones in LDS.
template <int kRT>
struct Sight {
  uint64_t seen[kRT];
  bool small;
};
constexpr int kWords = kTreeMaxNodes / 32;
constexpr int kAncPitch = kWords + 1;  // a row's words, and one of zeros

// Which of the 32 keys from j0 on (j0 + 32 > past) row r = 16 rt + c of the block sees: keys of
// the cache, and its ancestors' bits from j0 - past on. Bits past the drafted rows are zero.
template <int kRT>
__device__ inline uint32_t sight_of(const Block& b, const Sight<kRT>& s, int rt, int c, int j0) {
  const int n = j0 - b.past;
  if (s.small) {
    if (n < 0) return (static_cast<uint32_t>(s.seen[rt]) << -n) | ((1u << -n) - 1u);
    return n < 64 ? static_cast<uint32_t>(s.seen[rt] >> n) : 0u;
  }
  const uint32_t* const w = b.anc + (16 * rt + c) * kAncPitch;
  if (n < 0) return (w[0] << -n) | ((1u << -n) - 1u);
  const int i = min(n >> 5, kWords);
  return __builtin_amdgcn_alignbit(w[min(i + 1, kWords)], w[i], n & 31);
}

// A row's parent, or -1: the last cached token. Whatever the array holds, parents lie below.
__device__ inline int valid_parent(int p, int i) {
  return static_cast<unsigned>(p) < static_cast<unsigned>(i) ? p : -1;
}
// Up to 64 nodes, one a lane: their ancestors' reach doubles every round. p: the node's parent.
template <int kRT>
__device__ inline void find_sight(int p, int nodes, int row0, int lane, Sight<kRT>& s) {
  int up = lane < nodes ? valid_parent(p, lane) : -1;  // the first ancestor that seen lacks
  uint64_t seen = uint64_t{1} << lane;
  while (__any(up >= 0)) {
    const int from = max(up, 0);
    const uint32_t lo = __shfl(static_cast<uint32_t>(seen), from);
    const uint32_t hi = __shfl(static_cast<uint32_t>(seen >> 32), from);
    const int next = __shfl(up, from);
    if (up >= 0) {
      seen |= lo | static_cast<uint64_t>(hi) << 32;
      up = next;
    }
  }
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    const int r = row0 + 16 * rt + (lane & 15);
    const uint32_t lo = __shfl(static_cast<uint32_t>(seen), r & 63);
    const uint32_t hi = __shfl(static_cast<uint32_t>(seen >> 32), r & 63);
    s.seen[rt] = r < nodes ? lo | static_cast<uint64_t>(hi) << 32 : 0;
  }
}
// More nodes: words of `rows` rows from row0 on in LDS (zero past the tree's), to be read after a
// barrier; every thread of the workgroup calls it. Every node's next four ancestors lie
// together, so that a chain of 256 is walked in 64 reads (one by one: 13 us of 31).
__device__ inline void find_ancestors(const int* parents, int nodes, int row0, int rows,
                                      uint64_t* up, uint32_t* anc) {
  constexpr uint32_t kNone = 0xFFFFu;
  static_assert(kTreeMaxNodes <= 64 * kWaves, "a node a thread");
  const int tid = threadIdx.x;
  uint32_t* const pair = reinterpret_cast<uint32_t*>(up) + 2 * kTreeMaxNodes;
  const uint32_t p1 = tid < nodes ? valid_parent(parents[tid], tid) & kNone : kNone;
  if (tid < nodes) pair[tid] = p1;
  for (int i = tid; i < rows * kAncPitch; i += 64 * kWaves) anc[i] = 0u;
  __syncthreads();
  const uint32_t two = p1 | (p1 == kNone ? kNone : pair[p1]) << 16;
  __syncthreads();
  if (tid < nodes) pair[tid] = two;
  __syncthreads();
  const uint32_t p2 = two >> 16;
  if (tid < nodes)
    up[tid] = two | static_cast<uint64_t>(p2 == kNone ? ~0u : pair[p2]) << 32;
  __syncthreads();
  if (tid < rows && row0 + tid < nodes) {
    // Ancestors come in falling order: a word is whole when the walk leaves it.
    uint32_t n = row0 + tid, w = n >> 5, bits = 1u << (n & 31);
    while (n != kNone) {
      const uint64_t next = up[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        n = static_cast<uint32_t>(next >> (16 * i)) & kNone;
        if (n == kNone) break;
        if ((n >> 5) != w) {
          anc[tid * kAncPitch + w] = bits;
          bits = 0;
          w = n >> 5;
        }
        bits |= 1u << (n & 31);
      }
    }
    anc[tid * kAncPitch + w] = bits;
  }
}

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

// A wave's pieces of kSpan keys (kSpan * wave, + kSpan * kWaves, ..) on the f32 matrix pipe, 16
// at a time, f16 planes widened exactly: lane (c, g) holds key c's values d = 16 g + 0..15, so
// that lane (r, g) gets scores of keys 4 g + 0..3 of row r, which are the B operand of
// O^T += V^T P^T as they stand. o[rt][dt][e] is column 16 g + 4 e + dt. q: d = 16 g + 0..15 of row
// c, times scale * log2(e). `sight` runs once the first loads are on their way (it may hold barriers).
template <typename KT, int kRT, int kSpan, typename F>
__device__ inline void attend_f32(const Block& b, const f32x4 (&qx)[kRT][4], int wave, int lane,
                                  F sight, const Sight<kRT>& seen_by, Sums<kRT>& st) {
  constexpr uint32_t kRowBytes = 64 * sizeof(KT);
  const int c = lane & 15, g = lane >> 4;
  f32x4 kn[4], vn[4];
  auto load = [&](int j0) __attribute__((always_inline)) {
    const uint32_t ko = static_cast<uint32_t>(j0 - b.key0 + c) * kRowBytes + 16 * g * sizeof(KT);
    const uint32_t vo = static_cast<uint32_t>(j0 - b.key0 + 4 * g) * kRowBytes + 4 * c * sizeof(KT);
#pragma unroll
    for (int i = 0; i < 4; ++i) kn[i] = load4<KT>(b.k, ko + 4 * i * sizeof(KT));
#pragma unroll
    for (int i = 0; i < 4; ++i) vn[i] = load4<KT>(b.v, vo + i * kRowBytes);
  };
  auto after = [&](int j) {
    j += kStep;
    return (j - b.key0) % kSpan ? j : j + kSpan * (kWaves - 1);
  };
  int j0 = b.key0 + kSpan * wave;
  if (j0 < b.key1) load(j0);
  st.clear();
  sight();
  for (int next; j0 < b.key1; j0 = next) {
    next = after(j0);
    f32x4 kx[4], vx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kx[i] = kn[i];
      vx[i] = vn[i];
    }
    if (next < b.key1) load(next);
    // Drafted values that a row does not see have weight 0, and 0 times an infinity or
    // NaN is NaN: such values leave the product and are added row by row.
    const bool masked = j0 + kStep > b.past;
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
        seen = static_cast<int>(sight_of(b, seen_by, rt, c, j0) >> (4 * g));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(seen >> i & 1)) s[i] = -INFINITY;
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
        for (int key = 0; key < kStep; ++key) {
          // Weight and sight of key j0 + key, and its row's values of this lane's columns.
          const int i = key & 3;
          const float mine = i == 0 ? p[0] : i == 1 ? p[1] : i == 2 ? p[2] : p[3];
          const float pk = __shfl(mine, c + 16 * (key >> 2));
          const bool vis = (__shfl(seen, c + 16 * (key >> 2)) >> i) & 1;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x4 vk =
                load4<KT>(b.v, static_cast<uint32_t>(j0 - b.key0 + key) * kRowBytes +
                                   (16 * g + 4 * e) * static_cast<uint32_t>(sizeof(KT)));
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

// Keys key0 + 32 wave, + 128, .. of an f16 plane on the f16 matrix pipe. Query rows (times a
// power of two that puts the largest element into [2^14, 2^15)) and weights (in units of 2^-15)
// are split into two f16 parts, the second in a unit 2^-11 of the first and with sums of its
// own: within 2^-22 of themselves down to 2^-28 of the row's largest, smaller ones to 2^-51 of it,
// next to v_exp_f32's 2^-23 and what f32 sums over a head's 64 columns round off. A third part
// (all 24 bits) took 110 us instead of 96 at 64 rows x 65471 keys, 20 heads, and the outputs' error
// was 2.6e-7 with either. K comes from
// memory in operand layout, V passes through the wave's own swizzled LDS rows and is read
// transposed; the packed weights are the B operand of O^T += V^T P^T as they stand.
// o[rt][dt][e] is column 16 dt + 4 g + e. Returns whether a sum came out infinite or NaN: parts
// of an infinity are not numbers, so such a wave starts again with f32 operands.
template <int kRT, typename F>
__device__ inline bool attend_f16(const Block& b, const f32x4 (&qx)[kRT][4], int wave, int lane,
                                  char* vw, F sight, const Sight<kRT>& seen_by,
                                  Sums<kRT>& st) {
  constexpr int kN = 32;  // keys per step
  const int c = lane & 15, g = lane >> 4;
  u32x4 kx[2][2], vx[4];
  auto load = [&](int j0) __attribute__((always_inline)) {
    const uint32_t ko = static_cast<uint32_t>(j0 - b.key0 + c) * 128u + 32u * g;
    const uint32_t vo = static_cast<uint32_t>(j0 - b.key0) * 128u + 16u * lane;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
        kx[t][kk] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(b.k, ko + 2048 * t + 16 * kk, 0, 0));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      vx[i] = __builtin_bit_cast(u32x4,
                                 __builtin_amdgcn_raw_buffer_load_b128(b.v, vo + 1024 * i, 0, 0));
  };
  st.clear();
  int j0 = b.key0 + kN * wave;
  if (j0 < b.key1) load(j0);
  u32x4 qf[kRT][kParts][2];  // d = 16 g + 8 kk + 0..7
  float down[kRT];
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
  sight();
  for (; j0 < b.key1; j0 += kN * kWaves) {
    u32x4 pf[kRT][kParts];
    f32x4 s[kRT][2];
    float alpha[kRT];
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 sp[kParts] = {};
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int p = 0; p < kParts; ++p) sp[p] = mfma16(kx[t][kk], qf[rt][p][kk], sp[p]);
        s[rt][t] = join(sp);
      }
    wave_sync();  // the last step's transposed reads are done
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 8 * i + (lane >> 3);
      *reinterpret_cast<u32x4*>(vw + row * 128 + (((lane & 7) ^ swz(row)) * 16)) = vx[i];
    }
    wave_sync();
    if (j0 + kN * kWaves < b.key1) load(j0 + kN * kWaves);
    const bool masked = j0 + kN > b.past;
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt) {
      // Register i of tile t holds key 16 t + 4 g + i.
      if (masked) {
        const uint32_t seen = sight_of(b, seen_by, rt, c, j0) >> (4 * g);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(seen >> (16 * t + i) & 1)) s[rt][t][i] = -INFINITY;
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
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][t][i], down[rt], -md));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][t][i + 1], down[rt], -md));
          ls += p0 + p1;
          uint32_t w[kParts];
          split_units(p0, p1, kWeightUp, w);
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
        // The step's sums join at once: kept apart over the steps they took 32 registers more a
        // tile, and as many multiplications by alpha.
        f32x4 x[kParts];
#pragma unroll
        for (int p = 0; p < kParts; ++p) x[p] = mfma16(va, pf[rt][p], f32x4{0.f, 0.f, 0.f, 0.f});
        const f32x4 y = join(x);
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
      st.o[rt][dt] *= 1.f / kWeightUp;
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= !__builtin_isfinite(st.o[rt][dt][e]);
    }
  }
  return __any(odd);
}

// x / n, with the remainder; inv: 2^32 / n rounded up (for n 1: 2^32 - 1).
__device__ inline int divide(int x, int n, uint32_t inv, int& rest) {
  int q = static_cast<int>(__umulhi(static_cast<uint32_t>(x), inv));
  rest = x - q * n;
  if (rest < 0) {
    --q;
    rest += n;
  }
  if (rest >= n) {
    ++q;
    rest -= n;
  }
  return q;
}

template <typename KT, int kRT>
__global__ __launch_bounds__(64 * kWaves, 2) void tree_attend(TreeArgs a) {
  constexpr int kRows = 16 * kRT;
  constexpr bool kHalf = sizeof(KT) == 2;
  __shared__ __attribute__((aligned(128))) char vs[kHalf ? kWaves : 1][32 * 128];
  __shared__ __attribute__((aligned(16))) float mo[kWaves][kRows * kPitch];  // a wave's O rows
  __shared__ float ml[kWaves][2][kRows];        // and their max and sum
  __shared__ uint64_t up[kTreeMaxNodes + kTreeMaxNodes / 2];  // of a large tree: ancestors, pairs
  __shared__ uint32_t anc[kRows][kAncPitch];  // ancestors-or-self of the block's rows
  __shared__ int last_flag;

  // The workgroups of one head's chunk, which read the same rows, share an XCD's L2 (a tree's row
  // of the grid is a multiple of the XCDs).
  const int t = blockIdx.y;
  const int lid = xcd_remap(blockIdx.x, gridDim.x);
  if (lid >= a.n_wgs[t]) return;
  const int past = a.past[t], nodes = a.nodes[t], total = past + nodes;
  const int n_blk = a.n_blk[t], n_split = a.n_split[t];
  int blk, split;
  const int hs = divide(lid, n_blk, a.blk_inv[t], blk);
  const int h = divide(hs, n_split, a.split_inv[t], split);
  const int row0 = blk * kRows;
  const int key0 = split * a.chunk, key1 = min(key0 + a.chunk, total);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int64_t q_row = a.row0[t];

  // This chunk of the head's planes: rows at or past key1 read as zero.
  constexpr uint32_t kRowBytes = 64 * sizeof(KT);
  const int64_t plane = a.off[t] + h * a.kv_hs + static_cast<int64_t>(key0) * 64;
  const uint32_t range = static_cast<uint32_t>(key1 - key0) * kRowBytes;
  const Block b = {past, nodes, key0, key1, row0, &anc[0][0],
                   __builtin_amdgcn_make_buffer_rsrc(
                       const_cast<KT*>(static_cast<const KT*>(a.k) + plane), 0, range, kRawBuffer),
                   __builtin_amdgcn_make_buffer_rsrc(
                       const_cast<KT*>(static_cast<const KT*>(a.v) + plane), 0, range, kRawBuffer)};

  const int parent = key1 > past && nodes <= 64 && lane < nodes ? a.parents[q_row + lane] : -1;
  // Query rows: d = 16 g + 0..15 of row c of each tile, times scale * log2(e).
  f32x4 qx[kRT][4];
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    const int r = row0 + 16 * rt + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) qx[rt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r < nodes) {
      const float* qp = a.q + (q_row + r) * a.q_rs + h * 64 + 16 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qx[rt][i] = *reinterpret_cast<const f32x4u*>(qp + 4 * i) * a.scale_log2;
    }
  }

  Sight<kRT> seen_by;
  seen_by.small = nodes <= 64;
  const bool drafted = key1 > past;  // the chunk holds drafted rows
  auto sight = [&]() __attribute__((always_inline)) {
    if (!drafted) return;
    if (seen_by.small) {
      find_sight<kRT>(parent, nodes, row0, lane, seen_by);
    } else {
      find_ancestors(a.parents + q_row, nodes, row0, kRows, up, &anc[0][0]);
      __syncthreads();
    }
  };
  Sums<kRT> st;
  bool f32_order = true;  // which column o[rt][dt][e] is
  if constexpr (kHalf) {
    f32_order = attend_f16<kRT>(b, qx, wave, lane, vs[wave], sight, seen_by, st);
    if (f32_order) attend_f32<KT, kRT, 32>(b, qx, wave, lane, [] {}, seen_by, st);
  } else {
    attend_f32<KT, kRT, kStep>(b, qx, wave, lane, sight, seen_by, st);
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
  const bool mine = row0 + r < nodes;
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
  float* const part =
      a.part + (static_cast<int64_t>(at) * kRows + r) * kTreePart;
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

// Rows of a block: 16, so that a tree's blocks run on CUs of their own, or 32, which read a cache
// half as often, where an even number of three blocks or more would read one past what the caches
// hold (the f32 matrix pipe, slower, later). us, 16 / 32 rows, 20 heads: f16 26 nodes over 223 keys
// 6.3/8.1, 64 over 1500 11.6/16.6, 32 over 8000 (41 MB) 19.5/29.9, 64 over 20000 (102 MB)
// 47.9/45.9, 32 over 40000 (205 MB) 58.6/64.8, 48 over 40000 70.1/68.8, 64 over 40000 85.0/70.3, 64
// over 65471 (335 MB) 132/99; f32 64 over 20000 (205 MB) 101/102, 8 trees of 64 over 4000 (333 MB)
// 162/185, 48 over 40000 146/171, 64 over 40000 (410 MB) 183/172.
int block_rows(const TreeArgs& a, DType dt) {
  int most = 0;
  int64_t bytes = 0;
  for (int t = 0; t < a.n_trees; ++t) {
    most = std::max(most, a.nodes[t]);
    bytes += static_cast<int64_t>(a.past[t] + a.nodes[t]) * a.n_heads * 64 * 2 * (dt == kF16 ? 2 : 4);
  }
  const int64_t wide = (dt == kF16 ? 128ll : 384ll) << 20;
  return most > 32 && (most + 15) / 16 % 2 == 0 && bytes >= wide ? kTreeMaxRows : 16;
}

}  // namespace

int64_t tree_plan(TreeArgs& a, DType dt, bool split) {
  const int rows = block_rows(a, dt);
  int64_t blocks = 0, work = 0;
  int longest = 1;
  for (int t = 0; t < a.n_trees; ++t) {
    a.n_blk[t] = (a.nodes[t] + rows - 1) / rows;
    const int64_t b = static_cast<int64_t>(a.n_blk[t]) * a.n_heads;
    const int total = a.past[t] + a.nodes[t];
    blocks += b;
    work += b * total;
    longest = std::max(longest, total);
  }
  auto inverse = [](int n) {
    return static_cast<uint32_t>(std::min<uint64_t>(((uint64_t{1} << 32) + n - 1) / n, 0xffffffffu));
  };
  // Chunks of so many keys; returns the sum of all trees' workgroups and the grid's width.
  int64_t widest = 0;
  auto lay = [&](int64_t chunk) {
    int64_t sum = 0;
    widest = 0;
    a.chunk = static_cast<int>(chunk);
    for (int t = 0; t < a.n_trees; ++t) {
      a.n_split[t] = static_cast<int>((a.past[t] + a.nodes[t] + chunk - 1) / chunk);
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
  // A split costs ~1.5 us: caches of fewer keys than `whole` are not worth it, nor chunks of fewer
  // than `least`. us, whole / split, 12 heads, 4 trees of 13: f16 430 keys 7.7/8.6 (20 heads, 1500
  // keys 9.9/8.9), f32 430 keys 10.4/8.9 (249 keys 8.3/8.4). Two workgroups a CU in all, which run
  // at once (f16, 16 nodes over 65471 keys: 90 us with one, 73 with two, 76 with three; 64 nodes
  // 122, and 130 with eight workgroups more).
  const int whole = dt == kF16 ? 512 : 320, least = dt == kF16 ? 256 : 128;
  if (split && blocks < kTreeMaxWgs && longest > whole) {
    int64_t chunk = std::max<int64_t>(least, (work + kTreeMaxWgs - 1) / kTreeMaxWgs);
    for (chunk = (chunk + 127) / 128 * 128; chunk < longest; chunk += 128)
      if (lay(chunk) <= kTreeMaxWgs) return widest;
  }
  lay(longest);
  return widest;
}

hipError_t launch_tree_attend(const TreeArgs& a, DType dt, int64_t wgs, hipStream_t s) {
  if (wgs <= 0) return hipSuccess;
  if (wgs > 0x7fffffff) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(wgs), a.n_trees), block(64 * kWaves);
  const bool few = block_rows(a, dt) == 16;
#define WRS_TREE(KT, RT) hipLaunchKernelGGL((tree_attend<KT, RT>), grid, block, 0, s, a)
  switch (dt) {
    case kF16:
      if (few) { WRS_TREE(_Float16, 1); } else { WRS_TREE(_Float16, 2); }
      break;
    case kF32:
      if (few) { WRS_TREE(float, 1); } else { WRS_TREE(float, 2); }
      break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_TREE
  return hipGetLastError();
}

}  // namespace wrs
