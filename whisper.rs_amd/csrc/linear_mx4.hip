// Projections with MXFP4 weights: out[g](t, r) = act(w[g][r] . x[t] + bias[g][r]), sums in f32.
// Weights keep their 4 bits up to the MFMA: widened to 16-bit operands in registers, exactly, or
// with MXFP4 x taken as they are by the scaled MFMAs. Up to 16 rows of x stream the weights
// (K15), more go by tiles (K16).
#include "wrs_internal.hpp"

#include <algorithm>
#include <atomic>
#include <type_traits>

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

// x = the sum of its parts, the top halves of the words of p, exactly down to bf16's last bit,
// 2^-133: each takes the next 8 significant bits. An infinity is its first part alone; a NaN stays
// one.
template <int P>
__device__ inline void split_top(float x, uint32_t (&p)[P]) {
  p[0] = __builtin_bit_cast(uint32_t, x);
#pragma unroll
  for (int i = 1; i < P; ++i) {
    float rest = x - __builtin_bit_cast(float, p[i - 1] & kTop);
    if (i == 1 && __builtin_fabsf(x) == __builtin_inff()) rest = 0.f;
    x = rest;
    p[i] = __builtin_bit_cast(uint32_t, rest);
  }
}
// The top halves of two words.
__device__ inline uint32_t pack_top(uint32_t lo, uint32_t hi) {
  return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
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

// GELU of the projections, x / (1 + exp(-2 u)): 0.5 x (1 + tanh u) without the tanh, u = 0.7978846
// (x + 0.044715 x^3). Seven instructions (two more, with u formed first, took 3 us of 165), and
// small results keep their bits, which 1 + tanh u loses as tanh u nears -1.
__device__ inline float gelu_exp(float x) {
  constexpr float kOne = -2.f * 0.7978846f * 1.44269504f, kThree = kOne * 0.044715f;
  const float e = __builtin_amdgcn_exp2f(x * __builtin_fmaf(x * x, kThree, kOne));
  return x * __builtin_amdgcn_rcpf(1.f + e);
}

constexpr int kRawBuffer = 0x00020000;  // buffer resource word 3: raw, 32-bit data format
constexpr uint32_t kPast = 0xFFFF0000u;  // an offset past every buffer
constexpr uint32_t kPastRows = 0x80000000u;  // so with offsets of rows (below 2^28) added

constexpr int kRowsWaves = 8;
constexpr int kMx4MaxSplits = 8;
constexpr int kMx4CounterStride = 32;  // words between counters: a 128-byte line
constexpr int kGroup = 8;       // blocks of a row that a wave takes at a time: 128 bytes of codes
constexpr int kCodeBytes = 16 * kGroup * 16;            // of a tile's group
constexpr int kStage = kCodeBytes + 16 * kGroup + 128;  // LDS of a wave: codes, scales, pad

// K15 (mx4_rows): up to 16 rows of x, bound by the stream of codes. A wave multiplies tiles of
//   16 features; `ks` waves share a tile and take its groups of 8 blocks in turn, `chunk` groups
//   at a time for a workgroup. Codes come in whole 128-byte pieces of rows (a lane's operand is
//   16 bytes of its own row: loaded so, with a byte of scale each, 36 MB took 15.4 us, in
//   whole pieces and without scales 9.9), wait in registers, and change places in the wave's
//   own LDS. x is staged in LDS once for the workgroup, f32 in three bf16 parts (every bit of
//   it), f16 in two, each with an MFMA column of its own.
//   5 rows f32 1280 -> 51866 11.8 us, 3.0 TB/s of weights (read alone, the same bytes take 7.9; the
//   rest is x's way in and the last tiles' sums; f16 weights, K7m, 29); 1280 -> 5120 6.1; 5120 ->
//   1280 7.3; 3 x 1280 -> 1280 5.1.
// kMany: grids of more than one workgroup per CU keep their registers to what two need;
// others have x in flight at once (5 rows 5120 -> 1280: 11.3 us with 2 groups a thread).
template <typename XT, int kCT, int kBatch, bool kMany>
__global__ __launch_bounds__(64 * kRowsWaves, kMany ? 4 : 2) void mx4_rows(Mx4LinearArgs a, int ks,
                                                                           int chunk,
                                                                           uint32_t wide_inv,
                                                                           int per_split,
                                                                           int out_dt) {
  constexpr bool kBoth = sizeof(XT) == 1;  // x is MXFP4 too
  constexpr int kP = kBoth ? 1 : kParts<XT>;
  constexpr int kXBatch = kMany ? 2 : 4;  // groups of 8 values of x in flight per thread
  constexpr int kPitch = 16 * kCT + 1;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int tiles = kRowsWaves / ks, kw = wave % ks;
  const int grp = blockIdx.y;
  const int first = blockIdx.x * tiles * 16;  // the workgroup's first feature
  const int nb = a.n_in / kMx4Block, bytes = a.n_in / 2;
  const int n_wg = min(16 * tiles, a.n_out - first);  // features of the workgroup
  // Rows past the last feature and blocks past the last one read as zero.
  const __amdgpu_buffer_rsrc_t wrs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w[grp] + static_cast<int64_t>(first) * bytes), 0, n_wg * bytes,
      kRawBuffer);
  const __amdgpu_buffer_rsrc_t srs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w_scales[grp] + static_cast<int64_t>(first) * nb), 0, n_wg * nb,
      kRawBuffer);
  char* const mine = lds + wave * kStage;           // this wave's codes, then scales
  char* const xl = lds + kRowsWaves * kStage;       // x of the chunk
  const int tile_row = 16 * (wave / ks);

  // Load h of a group: lane j takes 16 bytes of row 8 h + (j / 8 ^ h), block (j ^ j / 8) % 8,
  // and puts them at place 64 h + j, so that 16 rows read at one block meet distinct banks.
  const int lr = lane >> 3, lb = (lane ^ lr) & 7;
  const uint32_t wo0 = (tile_row + lr) * bytes + 16 * lb;
  const uint32_t wo1 = (tile_row + 8 + (lr ^ 1)) * bytes + 16 * lb;
  const uint32_t so = (tile_row + (lane >> 2)) * nb + 2 * (lane & 3);
  // Where this lane's operand of block b of a group lies (block 4 e + g in step e).
  const int cr = (c & 7) ^ (c >> 3), at = 1024 * (c >> 3) + 128 * cr;
  const int place[2] = {at + 16 * (g ^ cr), at + 16 * ((g + 4) ^ cr)};
  static_assert(kGroup == 8, "a group is two steps of four blocks");

  const int pitch = 2 * (kMx4Block * kGroup * chunk + 8);  // bytes of a staged column
  int col[kCT];  // this lane's staged columns (past the last one, that one again: not stored)
#pragma unroll
  for (int i = 0; i < kCT; ++i) col[i] = min(16 * i + c, kP * a.n_tokens - 1) * pitch + 64 * g;

  f32x4 acc[2][kCT];
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int i = 0; i < kCT; ++i) acc[e][i] = f32x4{0.f, 0.f, 0.f, 0.f};

  u32x4 cw[kBatch][2];
  uint16_t sw[kBatch];
  const int first_g = blockIdx.z * per_split, nb1 = min(nb, kGroup * (first_g + per_split));
  for (int g0 = first_g; kGroup * g0 < nb1; g0 += chunk) {
    const int nbc = min(kGroup * chunk, nb1 - kGroup * g0);  // blocks of the chunk
    const int n = ((nbc + kGroup - 1) / kGroup - kw + ks - 1) / ks;  // this wave's groups
    auto load = [&](int u, int i) __attribute__((always_inline)) {
      int b = kGroup * (g0 + kw + ks * i);  // the group's first block
      // Formed anew for each load: kept as running offsets they cost 18 registers a group.
      asm("" : "+s"(b));
      const bool in = i < n && b + lb < nb;
      cw[u][0] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(wrs, in ? wo0 + 16 * b : kPast, 0, 0));
      cw[u][1] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(wrs, in ? wo1 + 16 * b : kPast, 0, 0));
      sw[u] = __builtin_amdgcn_raw_buffer_load_b16(
          srs, i < n && b + 2 * (lane & 3) < nb ? so + b : kPast, 0, 0);
    };
    if constexpr (kBoth) {
      // Codes of block b, row t at (16 b + t) * 16, scales behind them.
#pragma unroll
      for (int u = 0; u < kBatch; ++u) load(u, u);
      if (g0 != first_g) __syncthreads();
      for (int e = tid; e < 16 * kGroup * chunk; e += 64 * kRowsWaves) {
        const int b = e >> 4, t = e & 15, at_b = kGroup * g0 + b;
        u32x4 v = {0, 0, 0, 0};
        uint8_t sc = 0;
        if (t < a.n_tokens && b < nbc) {
          v = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.x) +
                                              static_cast<int64_t>(t) * bytes + 16 * at_b);
          sc = a.x_scales[t * nb + at_b];
        }
        *reinterpret_cast<u32x4*>(xl + 16 * e) = v;
        xl[256 * kGroup * chunk + e] = sc;
      }
    } else {
      // x's columns: part p of row t is column p * n_tokens + t. The first rows' loads go
      // ahead of the codes', which then load under the conversion.
      const int wide = 4 * kGroup * chunk;  // groups of 8 values a row
      const int groups = a.n_tokens * wide;
      typedef XT x8 __attribute__((ext_vector_type(8), aligned(16)));
      x8 xv[kXBatch];
      auto load_x = [&](int e0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kXBatch; ++i) {
          const int e = e0 + 64 * kRowsWaves * i + tid;
          const int t = __umulhi(e, wide_inv), k = e - t * wide;
          const bool in = e < groups && k < 4 * nbc;
          const int64_t x_at = in ? t * a.x_rs + kMx4Block * kGroup * g0 + 8 * k : 0;
          xv[i] = *reinterpret_cast<const x8*>(static_cast<const XT*>(a.x) + x_at);
        }
      };
      load_x(0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) load(u, u);
      if (g0 != first_g) __syncthreads();
      for (int e0 = 0; e0 < groups; e0 += 64 * kRowsWaves * kXBatch) {
        if (e0) load_x(e0);
#pragma unroll
        for (int i = 0; i < kXBatch; ++i) {
          const int e = e0 + 64 * kRowsWaves * i + tid;
          if (e >= groups) break;
          const int t = __umulhi(e, wide_inv), k = e - t * wide;
          const bool in = k < 4 * nbc;
          u32x4 w[kP];
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            uint32_t lo[kP], hi[kP];
            split_top<kP>(in ? static_cast<float>(xv[i][j]) : 0.f, lo);
            split_top<kP>(in ? static_cast<float>(xv[i][j + 1]) : 0.f, hi);
#pragma unroll
            for (int p = 0; p < kP; ++p) w[p][j >> 1] = pack_top(lo[p], hi[p]);
          }
#pragma unroll
          for (int p = 0; p < kP; ++p)
            *reinterpret_cast<u32x4*>(xl + (p * a.n_tokens + t) * pitch + 16 * k) = w[p];
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kBatch) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u;
        wave_sync();  // the last group's operands are read
        *reinterpret_cast<u32x4*>(mine + 16 * lane) = cw[u][0];
        *reinterpret_cast<u32x4*>(mine + 1024 + 16 * lane) = cw[u][1];
        *reinterpret_cast<uint16_t*>(mine + kCodeBytes + 2 * lane) = sw[u];
        wave_sync();
        load(u, i + kBatch);
        int b = kGroup * (kw + ks * i);  // in the chunk
        asm("" : "+s"(b));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (i >= n) continue;
          const u32x4 w = *reinterpret_cast<const u32x4*>(mine + place[e]);
          const int sc = *reinterpret_cast<const uint8_t*>(mine + kCodeBytes + 8 * c + 4 * e + g);
          if constexpr (kBoth) {
            const int xb = 16 * (b + 4 * e + g) + c;
            const u32x4 x = *reinterpret_cast<const u32x4*>(xl + 16 * xb);
            const int xs = *reinterpret_cast<const uint8_t*>(xl + 256 * kGroup * chunk + xb);
            i32x8 wa = {}, xa = {};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              wa[j] = static_cast<int>(w[j]);
              xa[j] = static_cast<int>(x[j]);
            }
            acc[e][0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, xa, acc[e][0], 4, 4,
                                                                         0, sc, 0, xs);
          } else {
            const char* const xc = xl + 64 * (b + 4 * e);
            const float scale = scale_of(sc);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const bf16x8 wv = widen8(w[j], scale);
#pragma unroll
              for (int t = 0; t < kCT; ++t)
                acc[j & 1][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    wv, *reinterpret_cast<const bf16x8*>(xc + col[t] + 16 * j), acc[j & 1][t], 0,
                    0, 0);
            }
          }
          __builtin_amdgcn_sched_barrier(0);  // one step's operands in registers at a time
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
  auto store = [&](int t, int r, float y) __attribute__((always_inline)) {
    if (a.bias[grp]) y += a.bias[grp][r];
    if (a.act == kActGelu) y = gelu_exp(y);
    const int64_t o = t * a.out_rs + (r >> 6) * a.out_hs + (r & 63);
    if (out_dt == kF32)
      static_cast<float*>(a.out[grp])[o] = y;
    else if (out_dt == kF16)
      static_cast<_Float16*>(a.out[grp])[o] = static_cast<_Float16>(y);
    else
      static_cast<__bf16*>(a.out[grp])[o] = static_cast<__bf16>(y);
  };
  const int splits = gridDim.z, n_e = 16 * tiles * a.n_tokens;
  const int unit = grp * gridDim.x + blockIdx.x;
  float* const part = splits > 1 ? a.part + static_cast<int64_t>(unit) * splits * n_e : nullptr;
  for (int e = tid; e < n_e; e += 64 * kRowsWaves) {
    const int t = e / (16 * tiles), rr = e % (16 * tiles), r = first + rr;
    if (r >= a.n_out) continue;
    float y = 0.f;
#pragma unroll
    for (int p = kP - 1; p >= 0; --p)
      for (int k = 0; k < ks; ++k)
        y += red[(16 * ((rr >> 4) * ks + k) + (rr & 15)) * kPitch + p * a.n_tokens + t];
    if (splits == 1)
      store(t, r, y);
    else
      st_agent(part + blockIdx.z * n_e + e, y);
  }
  if (splits == 1) return;
  // The workgroup that counts in last adds the splits in their order and re-arms the counter.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  unsigned* const counter = a.counters + unit * kMx4CounterStride;
  if (tid == 0)
    *reinterpret_cast<unsigned*>(lds) =
        __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (*reinterpret_cast<const unsigned*>(lds) != static_cast<unsigned>(splits - 1)) return;
  for (int e = tid; e < n_e; e += 64 * kRowsWaves) {
    const int t = e / (16 * tiles), r = first + e % (16 * tiles);
    if (r >= a.n_out) continue;
    float x[kMx4MaxSplits], y = 0.f;
#pragma unroll
    for (int s = 0; s < kMx4MaxSplits; ++s) x[s] = s < splits ? ld_agent(part + s * n_e + e) : 0.f;
#pragma unroll
    for (int s = 0; s < kMx4MaxSplits; ++s) y += x[s];
    store(t, r, y);
  }
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// 2 codes (byte k of w) times a scale as packed 16-bit values.
template <typename E, int k>
__device__ inline uint32_t widen2(uint32_t w, float scale) {
  if constexpr (__is_same(E, __bf16))
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, k));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, k));
}
template <typename E>
__device__ inline u32x4 widen8_as(uint32_t w, float scale) {
  return u32x4{widen2<E, 0>(w, scale), widen2<E, 1>(w, scale), widen2<E, 2>(w, scale),
               widen2<E, 3>(w, scale)};
}
template <typename E>
__device__ inline f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (__is_same(E, __bf16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Tile of a workgroup: BF features x BT rows of x, waves of WF x WT; KG groups of waves take the
// tile's columns in turn.
template <int BF_, int BT_, int WF_, int WT_, int KG_>
struct Tile {
  static constexpr int BF = BF_, BT = BT_, WF = WF_, WT = WT_, KG = KG_;
  static constexpr int kWaves = (BF / WF) * (BT / WT);  // of a group
  static constexpr int kGroupThreads = 64 * kWaves, kThreads = kGroupThreads * KG;
  static constexpr bool kSplits = KG == 4;  // whose columns may split over workgroups
};
constexpr int kK = 64;           // columns per stage
constexpr int kUnit = 256;       // columns in which a tile's columns split
constexpr int kRow = 2 * kK;     // bytes of a staged row
constexpr int kOutPitch = 68;    // floats of an output row in LDS

constexpr int kCodeRow = kK;     // bytes of codes of a row in two stages

// 16-byte chunk c of staged row r sits at c ^ (r / 2): 16 rows read at one chunk hit
// distinct banks. So for rows of codes of half the length, at c ^ (r / 4).
__device__ inline int chunk_at(int r, int c) { return r * kRow + 16 * (c ^ ((r >> 1) & 7)); }
__device__ inline int code_at(int r, int c) { return r * kCodeRow + 16 * (c ^ ((r >> 2) & 3)); }

template <typename T, int P>
constexpr size_t tile_lds() {  // P 0: MXFP4 x, whose scales lie behind its codes
  const size_t stage = (2ull * (P ? P * kRow : kRow + 8) * T::BT +
                        static_cast<size_t>(T::kWaves) * T::WF * (P ? kCodeRow : kRow)) * T::KG;
  const size_t out = sizeof(float) * T::kWaves * 32 * kOutPitch;
  const size_t join = sizeof(float) * T::BF * T::BT * (T::KG - 1);
  return stage > out ? (stage > join ? stage : join) : (out > join ? out : join);
}

// f32 x as two f16 parts of x * 2^7, the second in a unit 2^-11 of the first: within 2^-22 of a
// value down to 2^-21, and 2^-43 below. Rows whose largest value lies in [2^-10, 511] take them:
// there that is 2^-33 of it at most. Both parts meet one sum, so the second one's weights are
// 2^-11 of the first one's, and f16 holds both of a scale in 2^-20 .. 2^5 (their unit is 2^-8).
// (With both parts in one unit, 2^-32 was lost of every value: next to large values that meet
// weights of 0, 10^-6 kept 12 bits.)
constexpr float kXUp = 128.f, kXLeast = 0x1p-10f, kXMost = 511.f;
constexpr float kPartUnit = 0x1p-11f;
constexpr int kWUpLog2 = 8;
constexpr float kHalvesDown = 1.f / (kXUp * (1 << kWUpLog2));

// Whether f16 holds every weight under a scale: 6 * 2^13 and 0.5 * 2^-23, of two parts' weights
// 0.5 * 2^-12 * kPartUnit.
template <int P>
__device__ inline bool f16_scale(int byte) {
  constexpr int kLeast = P == 2 ? 127 - 12 - kWUpLog2 : 127 - 23;
  constexpr int kMost = P == 2 ? 127 + 13 - kWUpLog2 : 127 + 13;
  return static_cast<unsigned>(byte - kLeast) <= static_cast<unsigned>(kMost - kLeast);
}

constexpr int kOddX = 1, kOddW = 2;
// The workgroup's threads' bits (of 0..3) in one, for every thread; lds: free after a barrier.
// (__syncthreads_or has LDS of its own, which two workgroups of 80 KB do not leave.)
template <typename T>
__device__ inline int any_of(int bits, char* lds) {
  int* const votes = reinterpret_cast<int*>(lds);
  const int mine = (__any(bits & 1) ? 1 : 0) | (__any(bits & 2) ? 2 : 0);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) votes[threadIdx.x >> 6] = mine;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int i = 0; i < T::kThreads / 64; ++i) any |= votes[i];
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(any);
}

// Four scale bytes from `at` of a row on (an even place): one load where they lie on a word.
template <bool kWords>
__device__ inline uint32_t load_scales(const __amdgpu_buffer_rsrc_t& rs, uint32_t at, bool in,
                                       bool in_high) {
  if constexpr (kWords) return __builtin_amdgcn_raw_buffer_load_b32(rs, in ? at : kPast, 0, 0);
  const uint32_t lo = static_cast<uint16_t>(
      __builtin_amdgcn_raw_buffer_load_b16(rs, in ? at : kPast, 0, 0));
  const uint32_t hi = static_cast<uint16_t>(
      __builtin_amdgcn_raw_buffer_load_b16(rs, in_high ? at + 2 : kPast, 0, 0));
  return lo | (hi << 16);
}

// Adds one tile's products with operands of type E to acc. x goes in P parts: one of its own
// type, two of f16 (f32 x, E f16: results over kHalvesDown), or with bf16 E part `part` of kParts.
// Returns (to every thread) whether E cannot hold the tile's operands: kOddX, a row of f32 x, and
// kOddW, a scale of its weights, which may be that of zeros.
//   A wave's own rows of W come 64 bytes of codes at a time, 4 lanes a row, and change places in
//   its own LDS: lanes that load the 16 bytes that they multiply touch a cache line each, and
//   the line lookups bound the kernel (24000 x 5120 -> 1280 f16: 376 us). Lane (r, h)
//   of a 32-row block takes block h of a stage of row r, widened in registers, and step j
//   multiplies values 8 j.. of both blocks, so x's operand is chunk 4 h + j of its staged row.
template <typename T, typename XT, typename E, int P, bool kWords>
__device__ inline int tile_product(const Mx4LinearArgs& a, int grp, int f0, int t0, char* lds,
                                    int u0, int u1, int part,
                                    f32x16 (&acc)[T::WF / 32][T::WT / 32]) {
  constexpr int kF = T::WF / 32, kT = T::WT / 32;
  constexpr int kXn = T::BT * (kK / 8) / T::kGroupThreads;  // groups of 8 values a thread stages
  static_assert(kXn >= 1 && T::BT * (kK / 8) % T::kGroupThreads == 0, "whole groups");
  constexpr int kWn = T::WF * 4 / 64;  // chunks of codes a lane loads
  constexpr int kXBytes = T::BT * kRow, kStageBytes = P * kXBytes;
  constexpr bool kHalves = P == 2;  // f32 x in two f16 parts
  static_assert(!kHalves || (__is_same(XT, float) && __is_same(E, _Float16)), "");
  typedef XT x8 __attribute__((ext_vector_type(8), aligned(16)));
  const int lane = threadIdx.x & 63;
  const int kg = __builtin_amdgcn_readfirstlane(threadIdx.x / T::kGroupThreads);
  const int tid = threadIdx.x - kg * T::kGroupThreads;  // in the group
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const codes = lds + T::KG * 2 * kStageBytes + (kg * T::kWaves + wave) * T::WF * kCodeRow;
  lds += kg * 2 * kStageBytes;
  const int r32 = lane & 31, hl = lane >> 5;
  const int wf = (wave % (T::BF / T::WF)) * T::WF, wt = (wave / (T::BF / T::WF)) * T::WT;
  const int nb = a.n_in / kMx4Block, bytes = a.n_in / 2, stages = a.n_in / kK;

  // Rows past the last feature read as zero.
  const int n_f = min(T::BF, a.n_out - f0), n_t = min(T::BT, a.n_tokens - t0);
  const __amdgpu_buffer_rsrc_t wrs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w[grp] + static_cast<int64_t>(f0) * bytes), 0, n_f * bytes,
      kRawBuffer);
  const __amdgpu_buffer_rsrc_t srs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w_scales[grp] + static_cast<int64_t>(f0) * nb), 0, n_f * nb,
      kRawBuffer);
  // Rows of x: pointers of this thread's groups (rows past the last one: that one again,
  // not stored).
  const XT* xp[kXn];
#pragma unroll
  for (int i = 0; i < kXn; ++i) {
    const int e = tid + T::kGroupThreads * i, row = min(e >> 3, n_t - 1);
    xp[i] = static_cast<const XT*>(a.x) + (t0 + row) * a.x_rs + 8 * (e & 7);
  }

  u32x4 cw[kWn];
  uint32_t sw[kF], sw_next[kF];  // four scales of each row
  x8 xv[kXn];
  float most[kXn];  // largest magnitudes of this thread's rows of x
#pragma unroll
  for (int i = 0; i < kXn; ++i) most[i] = 0.f;
  // Pair i of the group, of two stages, is pair i * KG + kg of the tile's.
  const int pair0 = 2 * u0, pair1 = min((stages + 1) / 2, 2 * u1), stages1 = min(stages, 4 * u1);
  // Loads of stage i_s of x and pair i_p of W: number k of kXn + kWn + kF.
  constexpr int kLoads = kXn + kWn + kF;
  auto load = [&](int k, int i_s, int i_p) __attribute__((always_inline)) {
    if (k < kXn) {
      const int at = kK * min(2 * (pair0 + (i_s >> 1) * T::KG + kg) + (i_s & 1), stages - 1);
      xv[k] = *reinterpret_cast<const x8*>(xp[k] + at);
      return;
    }
    int p = pair0 + i_p * T::KG + kg;
    asm("" : "+s"(p));  // offsets are formed per pair, not kept per load
    if (k < kXn + kWn) {
      const int i = k - kXn, at = 4 * p + (lane & 3);
      const uint32_t o = at < nb ? (wf + (lane >> 2)) * bytes + 16 * at : kPastRows;
      cw[i] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(wrs, o + i * 16 * bytes, 0, 0));
    } else {
      const int i = k - kXn - kWn;
      sw_next[i] = load_scales<kWords>(srs, (wf + 32 * i + r32) * nb + 4 * p, 4 * p < nb,
                                       4 * p + 2 < nb);
    }
  };
  auto put_w = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kWn; ++i)
      *reinterpret_cast<u32x4*>(codes + code_at((lane >> 2) + 16 * i, lane & 3)) = cw[i];
#pragma unroll
    for (int i = 0; i < kF; ++i) sw[i] = sw_next[i];
    wave_sync();  // other lanes read the codes
  };
  auto store_x = [&](char* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kXn; ++i) {
      const int e = tid + T::kGroupThreads * i;
      char* const at = buf + chunk_at(e >> 3, e & 7);
      const x8& x = xv[i];
      if constexpr (kHalves) {
        u32x4 h, l;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          most[i] = fmaxf(most[i], fmaxf(__builtin_fabsf(x[j]), __builtin_fabsf(x[j + 1])));
          f16x2 hi = {static_cast<_Float16>(__builtin_fmaf(x[j], kXUp, 0.f)),
                      static_cast<_Float16>(__builtin_fmaf(x[j + 1], kXUp, 0.f))};
          uint32_t w = __builtin_bit_cast(uint32_t, hi);
          asm("" : "+v"(w));  // formed once, not again where it is taken off
          hi = __builtin_bit_cast(f16x2, w);
          // The difference is exact, and so is its product with the unit's inverse.
          constexpr float kUp = 1.f / kPartUnit;
          const f16x2 lo = {
              static_cast<_Float16>(
                  __builtin_fmaf(static_cast<float>(hi[0]), -kUp, x[j] * (kXUp * kUp))),
              static_cast<_Float16>(
                  __builtin_fmaf(static_cast<float>(hi[1]), -kUp, x[j + 1] * (kXUp * kUp)))};
          h[j >> 1] = w;
          l[j >> 1] = __builtin_bit_cast(uint32_t, lo);
        }
        *reinterpret_cast<u32x4*>(at) = h;
        *reinterpret_cast<u32x4*>(at + kXBytes) = l;
      } else if constexpr (__is_same(XT, E)) {
        *reinterpret_cast<u32x4*>(at) = __builtin_bit_cast(u32x4, x);
      } else {
        constexpr int kAll = kParts<XT>;
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          uint32_t lo[kAll], hi[kAll];
          split_top<kAll>(static_cast<float>(x[j]), lo);
          split_top<kAll>(static_cast<float>(x[j + 1]), hi);
          uint32_t v = pack_top(lo[0], hi[0]);
#pragma unroll
          for (int p = 1; p < kAll; ++p) v = part == p ? pack_top(lo[p], hi[p]) : v;
          w[j >> 1] = v;
        }
        *reinterpret_cast<u32x4*>(at) = w;
      }
    }
  };
  bool odd_x = false, odd_w = false;
  // Stage d of a pair: operands of step j + 1 are formed behind the products that use their
  // registers last, and the first `n` loads of stage i_s and pair i_p go between them.
  auto multiply = [&](int d, const char* buf, auto n, int i_s, int i_p)
      __attribute__((always_inline)) {
    float scale[kF];
    u32x4 c[kF];
#pragma unroll
    for (int i = 0; i < kF; ++i) {
      const int byte = (sw[i] >> (16 * d + 8 * hl)) & 255;
      if constexpr (__is_same(E, _Float16))
        odd_w |= wf + 32 * i + r32 < n_f && !f16_scale<P>(byte);
      scale[i] = scale_of(kHalves ? byte + kWUpLog2 : byte);
      c[i] = *reinterpret_cast<const u32x4*>(codes + code_at(32 * i + r32, 2 * d + hl));
    }
    // Operands of x are read a step ahead. With two parts, waves of several tiles read them a part
    // ahead and form the second part's weights in the first one's registers, just before its
    // products: waves of 64 x 128 spill as it is, and 64 x 64 are no faster the other way (3000
    // rows 5120 -> 1280: 110 us, 111 to 113).
    constexpr bool kTight = P > 1 && kT >= 2;
    constexpr int kAhead = kTight ? 1 : P;  // parts
    u32x4 wv[2][kF], wl[kF], xw[kAhead][kT];
    auto widen = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kF; ++i) wv[j & 1][i] = widen8_as<E>(c[i][j], scale[i]);
    };
    auto lower = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kF; ++i)
        wl[i] = __builtin_bit_cast(u32x4, __builtin_bit_cast(f16x8, wv[j & 1][i]) *
                                              static_cast<_Float16>(kPartUnit));
    };
    // Part p of step j, numbered s = j * P + p.
    auto read_x = [&](int s, int t) __attribute__((always_inline)) {
      xw[s % kAhead][t] = *reinterpret_cast<const u32x4*>(
          buf + s % P * kXBytes + chunk_at(wt + 32 * t + r32, 4 * hl + s / P));
    };
    constexpr int kSteps = kK / 16 * P, kSlots = kSteps * kT, kNow = decltype(n)::value;
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int t = 0; t < kT; ++t) read_x(s, t);
    widen(0);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int j = s / P, p = s % P;
      if (kTight && p) lower(j);
#pragma unroll
      for (int t = 0; t < kT; ++t) {
#pragma unroll
        for (int i = 0; i < kF; ++i)
          acc[i][t] = mfma32<E>(p ? wl[i] : wv[j & 1][i], xw[s % kAhead][t], acc[i][t]);
        if (!kTight && P > 1 && p == 0 && t == 0) lower(j);
        if (p == 0 && t == 0 && s + P < kSteps) widen(j + 1);
        if (s + kAhead < kSteps) read_x(s + kAhead, t);
#pragma unroll
        for (int k = 0; k < kNow; ++k)
          if (k * kSlots / (kNow ? kNow : 1) == s * kT + t) load(k, i_s, i_p);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

#pragma unroll
  for (int k = 0; k < kLoads; ++k) load(k, 0, 0);
  store_x(lds);
#pragma unroll
  for (int k = 0; k < kXn; ++k) load(k, 1, 0);
  __syncthreads();
  const int turns = (pair1 - pair0 + T::KG - 1) / T::KG;  // every group's; the last may be empty
  int i_p = 0;
  // No branch in this loop: one around the products costs copies of the sums (64 moves per two
  // stages of a 64 x 128 wave).
  for (; i_p + 1 < turns; ++i_p) {
    put_w();
    store_x(lds + kStageBytes);
    multiply(0, lds, std::integral_constant<int, kLoads>{}, 2 * i_p + 2, i_p + 1);
    __syncthreads();
    store_x(lds);
    multiply(1, lds + kStageBytes, std::integral_constant<int, kXn>{}, 2 * i_p + 3, 0);
    __syncthreads();
  }
  // The second stage, stored here already, is a repeated one where there is none.
  put_w();
  store_x(lds + kStageBytes);
  const int last = 2 * (pair0 + i_p * T::KG + kg);
  if (last < stages1) multiply(0, lds, std::integral_constant<int, 0>{}, 0, 0);
  __syncthreads();
  if (last + 1 < stages1) multiply(1, lds + kStageBytes, std::integral_constant<int, 0>{}, 0, 0);
  if constexpr (kHalves) {
    // 8 neighbouring lanes staged a row. Rows past the last one repeat it.
#pragma unroll
    for (int i = 0; i < kXn; ++i) {
      float m = most[i];
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
      if constexpr (T::KG > 1) {
        // The groups staged other columns of the same rows.
        float* const all = reinterpret_cast<float*>(lds - kg * 2 * kStageBytes);
        const int row = (tid + T::kGroupThreads * i) >> 3;
        if (i == 0) __syncthreads();  // the last stage is read
        if ((tid & 7) == 0) all[kg * T::BT + row] = m;
      }
      if constexpr (T::KG == 1) odd_x |= m != 0.f && !(m >= kXLeast && m <= kXMost);
    }
    if constexpr (T::KG > 1) {
      __syncthreads();
      const float* const all = reinterpret_cast<const float*>(lds - kg * 2 * kStageBytes);
      if (threadIdx.x < T::BT) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < T::KG; ++i) m = fmaxf(m, all[i * T::BT + threadIdx.x]);
        odd_x |= m != 0.f && !(m >= kXLeast && m <= kXMost);
      }
    }
  }
  return any_of<T>((odd_x ? kOddX : 0) | (odd_w ? kOddW : 0), lds - kg * 2 * kStageBytes);
}

// Whether a block of a tile's weights has a scale that f16 does not hold and is not of zeros, whose
// small scale (2^-127 as quantised) does not matter: padded columns and pruned weights. Asked after
// the product, for tiles that met such a scale. us, 24000 x 5120 -> 1280 without zeros / with the
// last block of every row of zeros: f16 268/300, f32 575/604, 130 rows 1280 -> 3 x 1280 8.0/9.7,
// 13.3/14.8 (formed again in bf16 parts 857, 1690, 22.2, 34.6; with the codes looked at within the
// product's loop f16 286/285, f32, which then spills 63 registers, 814/814).
template <typename T, int P>
__device__ inline bool odd_weights(const Mx4LinearArgs& a, int grp, int f0, int u0, int u1,
                                   char* lds) {
  const int nb = a.n_in / kMx4Block, b0 = u0 * (kUnit / kMx4Block);
  const int pairs = (min(nb, u1 * (kUnit / kMx4Block)) - b0) / 2;  // of blocks, of a row
  const int n = min(T::BF, a.n_out - f0) * pairs;
  constexpr int kAtOnce = 4;
  int odd = 0;
  for (int e0 = threadIdx.x; e0 < n; e0 += kAtOnce * T::kThreads) {
    int64_t at[kAtOnce];
    uint32_t two[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int e = min(e0 + i * T::kThreads, n - 1), row = e / pairs;
      at[i] = static_cast<int64_t>(f0 + row) * nb + b0 + 2 * (e - row * pairs);
      two[i] = *reinterpret_cast<const uint16_t*>(a.w_scales[grp] + at[i]);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int byte = (two[i] >> (8 * k)) & 255;
        if (f16_scale<P>(byte)) continue;
        const u32x4 c = *reinterpret_cast<const u32x4*>(a.w[grp] + 16 * (at[i] + k));
        if (byte > 127 || ((c[0] | c[1] | c[2] | c[3]) & 0x77777777u)) odd = 1;
      }
  }
  return any_of<T>(odd, lds) != 0;
}

// The same for MXFP4 x: 256 columns a stage, codes as they are into 32x32x64 MFMAs. Lane (r, h)
// holds blocks 4 h + 0..3 of row r, step q multiplies block 4 h + q, whose scale is byte q of
// the row's word h.
template <typename T, bool kWords>
__device__ inline void tile_product_mx4(const Mx4LinearArgs& a, int grp, int f0, int t0, char* lds,
                                        int u0, int u1, f32x16 (&acc)[T::WF / 32][T::WT / 32]) {
  constexpr int kF = T::WF / 32, kT = T::WT / 32;
  constexpr int kXn = T::BT * 8 / T::kGroupThreads;  // 16-byte chunks of x a thread stages
  static_assert(kXn >= 1 && T::BT * 8 % T::kGroupThreads == 0, "whole chunks");
  static_assert(2 * T::BT <= T::kGroupThreads, "a word of scales a thread");
  constexpr int kStageBytes = T::BT * kRow + T::BT * 8;
  constexpr int kBlocks = 8;  // of a stage
  constexpr int kWn = T::WF * 8 / 64;  // chunks of codes of W a lane loads
  const int lane = threadIdx.x & 63;
  const int kg = __builtin_amdgcn_readfirstlane(threadIdx.x / T::kGroupThreads);
  const int tid = threadIdx.x - kg * T::kGroupThreads;  // in the group
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  char* const codes = lds + T::KG * 2 * kStageBytes + (kg * T::kWaves + wave) * T::WF * kRow;
  lds += kg * 2 * kStageBytes;
  const int r32 = lane & 31, hl = lane >> 5;
  const int wf = (wave % (T::BF / T::WF)) * T::WF, wt = (wave / (T::BF / T::WF)) * T::WT;
  const int nb = a.n_in / kMx4Block, bytes = a.n_in / 2;
  const int nb1 = min(nb, kBlocks * u1);  // where the tile's columns end

  // Rows past the last and blocks past a row's last read as zero: codes of 0, scale 2^-127.
  const int n_f = min(T::BF, a.n_out - f0), n_t = min(T::BT, a.n_tokens - t0);
  const __amdgpu_buffer_rsrc_t wrs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w[grp] + static_cast<int64_t>(f0) * bytes), 0, n_f * bytes,
      kRawBuffer);
  const __amdgpu_buffer_rsrc_t srs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.w_scales[grp] + static_cast<int64_t>(f0) * nb), 0, n_f * nb,
      kRawBuffer);
  const __amdgpu_buffer_rsrc_t xrs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(static_cast<const uint8_t*>(a.x) + static_cast<int64_t>(t0) * bytes),
      0, n_t * bytes, kRawBuffer);
  const __amdgpu_buffer_rsrc_t xsrs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(a.x_scales + static_cast<int64_t>(t0) * nb), 0, n_t * nb, kRawBuffer);
  u32x4 cw[kWn], xv[kXn];
  uint32_t sw[kF], sw_next[kF], xs;
  // Loads of stage i_s of W and stage i_x of x: number k of kWn + kF + kXn + 1. Offsets are formed
  // per stage, not kept per load.
  constexpr int kLoads = kWn + kF + kXn + 1;
  auto load = [&](int k, int i_s, int i_x) __attribute__((always_inline)) {
    int b = kBlocks * (u0 + i_s * T::KG + kg), bx = kBlocks * (u0 + i_x * T::KG + kg);
    asm("" : "+s"(b), "+s"(bx));
    if (k < kXn) {
      const int e = tid + T::kGroupThreads * k, at = bx + (e & 7);
      xv[k] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                     xrs, at < nb1 ? (e >> 3) * bytes + 16 * at : kPast, 0, 0));
    } else if (k == kXn) {
      const int at = bx + 4 * (tid & 1);
      const bool mine = tid < 2 * T::BT;
      xs = load_scales<kWords>(xsrs, (tid >> 1) * nb + at, mine && at < nb1, mine && at + 2 < nb1);
    } else if (k <= kXn + kWn) {
      const int i = k - kXn - 1, at = b + (lane & 7);
      const uint32_t o = at < nb1 ? (wf + (lane >> 3)) * bytes + 16 * at : kPastRows;
      cw[i] = __builtin_bit_cast(
          u32x4, __builtin_amdgcn_raw_buffer_load_b128(wrs, o + i * 8 * bytes, 0, 0));
    } else {
      const int i = k - kXn - 1 - kWn, sb = b + 4 * hl;
      sw_next[i] = load_scales<kWords>(srs, (wf + 32 * i + r32) * nb + sb, sb < nb1, sb + 2 < nb1);
    }
  };
  auto put_w = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kWn; ++i)
      *reinterpret_cast<u32x4*>(codes + chunk_at((lane >> 3) + 8 * i, lane & 7)) = cw[i];
#pragma unroll
    for (int i = 0; i < kF; ++i) sw[i] = sw_next[i];
    wave_sync();  // other lanes read the codes
  };
  auto store_x = [&](char* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kXn; ++i) {
      const int e = tid + T::kGroupThreads * i;
      *reinterpret_cast<u32x4*>(buf + chunk_at(e >> 3, e & 7)) = xv[i];
    }
    if (2 * T::BT == T::kGroupThreads || tid < 2 * T::BT)
      *reinterpret_cast<uint32_t*>(buf + T::BT * kRow + 4 * tid) = xs;
  };
  // One stage: operands of step q + 1 are read behind the products that use their registers last,
  // and the loads of later stages go between them (all reads of a step before its products and all
  // loads before both: 138 us instead of 132).
  auto multiply = [&](const char* buf, int i_s) __attribute__((always_inline)) {
    int xsc[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t)
      xsc[t] = *reinterpret_cast<const int*>(buf + T::BT * kRow + 8 * (wt + 32 * t + r32) + 4 * hl);
    u32x4 w[2][kF], x[kT];
    auto read_w = [&](int q) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kF; ++i)
        w[q & 1][i] =
            *reinterpret_cast<const u32x4*>(codes + chunk_at(32 * i + r32, 4 * hl + q));
    };
    auto read_x = [&](int q, int t) __attribute__((always_inline)) {
      x[t] = *reinterpret_cast<const u32x4*>(buf + chunk_at(wt + 32 * t + r32, 4 * hl + q));
    };
    read_w(0);
#pragma unroll
    for (int t = 0; t < kT; ++t) read_x(0, t);
    auto step = [&](auto q_) __attribute__((always_inline)) {
      constexpr int q = decltype(q_)::value;
#pragma unroll
      for (int t = 0; t < kT; ++t) {
#pragma unroll
        for (int i = 0; i < kF; ++i) {
          const u32x4 &u = w[q & 1][i], &v = x[t];
          const i32x8 wa = {(int)u[0], (int)u[1], (int)u[2], (int)u[3], 0, 0, 0, 0};
          const i32x8 xa = {(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
          acc[i][t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
              wa, xa, acc[i][t], 4, 4, q, static_cast<int>(sw[i]), q, xsc[t]);
        }
        if constexpr (q < 3) {
          if (t == 0) read_w(q + 1);
          read_x(q + 1, t);
        }
        constexpr int kSlots = 4 * kT;
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
          if (k * kSlots / kLoads == q * kT + t) load(k, i_s + 1, i_s + 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  };

#pragma unroll
  for (int k = 0; k < kLoads; ++k) load(k, 0, 0);
  store_x(lds);
#pragma unroll
  for (int k = 0; k <= kXn; ++k) load(k, 0, 1);
  __syncthreads();
  // Stages past the last one are zeros.
  const int turns = (u1 - u0 + T::KG - 1) / T::KG;
  auto stage = [&](int i_s, int d) __attribute__((always_inline)) {
    put_w();
    store_x(lds + (1 - d) * kStageBytes);
    multiply(lds + d * kStageBytes, i_s);
    __syncthreads();
  };
  int i_s = 0;
  for (; i_s + 1 < turns; i_s += 2) {
    stage(i_s, 0);
    stage(i_s + 1, 1);
  }
  if (i_s < turns) stage(i_s, 0);
}

// The tile's outputs: each wave passes 32 rows x 64 features at a time through its own LDS, so
// that rows are stored in whole pieces (16 bytes a lane straight from the MFMA layout go to
// 32 rows each). Stores pass by the cache that holds W and x: 24000 x 5120 -> 1280 f16 338 -> 323
// us.
template <typename T, typename OT>
__device__ inline void tile_store(const Mx4LinearArgs& a, int grp, int f0, int t0, char* lds,
                                  bool whole, float down,
                                  f32x16 (&acc)[T::WF / 32][T::WT / 32]) {
  constexpr int kF = T::WF / 32, kT = T::WT / 32, kFe = kF > 1 ? 2 : 1;  // feature blocks a pass
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if constexpr (T::KG > 1) {
    // The groups' sums join the first group's, in order.
    f32x4* const join = reinterpret_cast<f32x4*>(lds);
    constexpr int kQuads = kF * kT * 4;
    if (wave >= T::kWaves) {
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const f32x16& x = acc[q / 4 / kT][q / 4 % kT];
        join[((wave - T::kWaves) * kQuads + q) * 64 + lane] =
            f32x4{x[4 * (q & 3)], x[4 * (q & 3) + 1], x[4 * (q & 3) + 2], x[4 * (q & 3) + 3]};
      }
    }
    __syncthreads();
    if (wave < T::kWaves) {
      for (int k = 0; k < T::KG - 1; ++k)
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
          const f32x4 x = join[((k * T::kWaves + wave) * kQuads + q) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[q / 4 / kT][q / 4 % kT][4 * (q & 3) + e] += x[e];
        }
    }
    __syncthreads();
    if (wave >= T::kWaves) return;
  }
  if constexpr (T::kSplits) {
    const int splits = gridDim.z;
    if (splits > 1) {
      // A wave's sums meet those of the same wave of the other splits, in their order: the wave that
      // counts in last adds them and re-arms the counter.
      static_assert(kF == 1 && kT == 1, "one MFMA tile a wave");
      const int unit = (grp * gridDim.x + blockIdx.x) * T::kWaves + wave, split = blockIdx.z;
      float* const part = a.part + static_cast<int64_t>(unit) * splits * 1024 + lane;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[0][0][e] *= down;
        st_agent(part + split * 1024 + 64 * e, acc[0][0][e]);
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
      unsigned* const counter = a.counters + static_cast<int64_t>(unit) * kMx4CounterStride;
      unsigned before = 0;
      if (lane == 0)
        before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      asm volatile("" ::: "memory");
      if (__builtin_amdgcn_readfirstlane(static_cast<int>(before)) != splits - 1) return;
      f32x16 sum = {};
      constexpr int kAtOnce = 4;
#pragma unroll 1
      for (int s0 = 0; s0 < splits; s0 += kAtOnce) {
        float x[kAtOnce][16];
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            x[s][e] = s0 + s < splits ? ld_agent(part + (s0 + s) * 1024 + 64 * e) : 0.f;
#pragma unroll
        for (int s = 0; s < kAtOnce; ++s)
#pragma unroll
          for (int e = 0; e < 16; ++e) sum[e] += x[s][e];
      }
      acc[0][0] = sum;
      down = 1.f;
      if (lane == 0)
        __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  const int r32 = lane & 31, hl = lane >> 5;
  const int wf = (wave % (T::BF / T::WF)) * T::WF, wt = (wave / (T::BF / T::WF)) * T::WT;
  float* const mine = reinterpret_cast<float*>(lds) + wave * 32 * kOutPitch;
  constexpr int kLanes = 4 * kFe;  // lanes of a row, 8 features each
  constexpr int kStep = 64 / kLanes;
  const int lr = lane / kLanes, lf = 8 * (lane % kLanes);
  // Locals: the compiler cannot tell that stores leave the arguments alone.
  const int n_tokens = a.n_tokens, n_out = a.n_out, act = a.act;
  const int64_t out_rs = a.out_rs, out_hs = a.out_hs;
  OT* const out = static_cast<OT*>(a.out[grp]);
  const float* const bias = a.bias[grp];
  // Tiles without an edge store without a test (the tests, and what the compiler waits for at
  // each, took 15 us of 160).
  auto pass = [&](auto full) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kF; i += kFe) {
      const int r = f0 + wf + 32 * i + lf;  // this lane's first feature
      float b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = 0.f;
      if (bias) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (full || r + e < n_out) b[e] = bias[r + e];
      }
      const int row0 = t0 + wt + lr;
      OT* const to = out + row0 * out_rs + (r >> 6) * out_hs + (r & 63);
#pragma unroll
      for (int t = 0; t < kT; ++t) {
        wave_sync();
#pragma unroll
        for (int f = 0; f < kFe; ++f)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<f32x4*>(mine + r32 * kOutPitch + 32 * f + 2 * e + 4 * hl) =
                f32x4{acc[i + f][t][e], acc[i + f][t][e + 1], acc[i + f][t][e + 2],
                      acc[i + f][t][e + 3]};
        wave_sync();
#pragma unroll
        for (int j = 0; j < 32; j += kStep) {
          const f32x4 y0 = *reinterpret_cast<const f32x4*>(mine + (j + lr) * kOutPitch + lf);
          const f32x4 y1 = *reinterpret_cast<const f32x4*>(mine + (j + lr) * kOutPitch + lf + 4);
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            y[e] = __builtin_fmaf(e < 4 ? y0[e & 3] : y1[e & 3], down, b[e]);
          if (act == kActGelu) {
            asm volatile("");  // a branch, not both ways and a choice for each value
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = gelu_exp(y[e]);
          }
          const int in_tile = 32 * t + j;
          OT* const op = to + in_tile * out_rs;
          if (full || (whole && row0 + in_tile < n_tokens && r + 8 <= n_out)) {
            typedef OT o8 __attribute__((ext_vector_type(8), aligned(16)));
            o8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = static_cast<OT>(y[e]);
            __builtin_nontemporal_store(o, reinterpret_cast<o8*>(op));
          } else if (row0 + in_tile < n_tokens) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (r + e < n_out) op[e] = static_cast<OT>(y[e]);
          }
        }
      }
    }
  };
  if (whole && f0 + T::BF <= n_out && t0 + T::BT <= n_tokens)
    pass(std::true_type{});
  else
    pass(std::false_type{});
}

// Tiles of features that go together: the 64 workgroups of an XCD take 8 by 8 tiles and read
// each stage of W and x from memory once (24000 x 5120 -> 5120 MXFP4: 421 us with all features
// first, 401 in panels of 4 and of 8, 411 of 16; tiles of shorter rows don't care).
constexpr int kPanel = 8;

// K16 (mx4_tile): many rows of x. W is widened to 16-bit operands in registers, x passes through
//   LDS in one part (f16, bf16) or two f16 ones (f32), and both feed 32x32x16 MFMAs. f16 holds
//   weights of scales 2^-23 to 2^13 exactly (beside two parts of x 2^-20 to 2^5), and rows of f32
//   x whose largest value is of ordinary size; a tile that meets others is formed again from bf16
//   operands, which hold any, one of x's two or three parts after the other.
//   24000 x 5120 -> 1280: f16 284 us, 1110 TFLOP/s, the matrix pipe 58% busy and the card's power
//   the bound (the library's product of f16 weights 274), bf16 265, f32 595, MXFP4 101, 3.1
//   PFLOP/s (zeros in its place a quarter less); 1280 -> 5120 MXFP4 with GELU 127, of which the
//   epilogue's 123 M outputs are about 50. 130 rows f32, 3 x 1280 -> 1280 13.1 us: ten steps of x's
//   way through LDS in two parts on one workgroup a CU (f16 9.2, MXFP4 7.4).
template <typename T, typename XT, typename OT, bool kWords>
__global__ __launch_bounds__(T::kThreads, T::KG > 1 ? 4 : 2) void mx4_tile(Mx4LinearArgs a,
                                                                           int n_f, int whole,
                                                                           int per_split) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lid = xcd_remap(blockIdx.x, gridDim.x);
  const int n_t = gridDim.x / n_f, panel = lid / (kPanel * n_t);
  const int wide = min(kPanel, n_f - kPanel * panel), in = lid - kPanel * n_t * panel;
  const int f0 = (kPanel * panel + in % wide) * T::BF, t0 = in / wide * T::BT, grp = blockIdx.y;
  const int units = (a.n_in + kUnit - 1) / kUnit;
  const int u0 = T::kSplits ? static_cast<int>(blockIdx.z) * per_split : 0;
  const int u1 = T::kSplits ? min(units, u0 + per_split) : units;
  f32x16 acc[T::WF / 32][T::WT / 32];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < T::WF / 32; ++i)
#pragma unroll
      for (int t = 0; t < T::WT / 32; ++t) acc[i][t] = f32x16{};
  };
  clear();
  float down = 1.f;
  if constexpr (sizeof(XT) == 1) {
    tile_product_mx4<T, kWords>(a, grp, f0, t0, lds, u0, u1, acc);
  } else if constexpr (__is_same(XT, __bf16)) {
    tile_product<T, XT, __bf16, 1, kWords>(a, grp, f0, t0, lds, u0, u1, 0, acc);
  } else {
    constexpr int kP = __is_same(XT, float) ? 2 : 1;
    if (kP == 2) down = kHalvesDown;
    int odd = tile_product<T, XT, _Float16, kP, kWords>(a, grp, f0, t0, lds, u0, u1, 0, acc);
    if (odd == kOddW) odd = odd_weights<T, kP>(a, grp, f0, u0, u1, lds);
    if (odd) {
      clear();
      down = 1.f;
#pragma unroll 1
      for (int part = kParts<XT> - 1; part >= 0; --part)
        tile_product<T, XT, __bf16, 1, kWords>(a, grp, f0, t0, lds, u0, u1, part, acc);
    }
  }
  tile_store<T, OT>(a, grp, f0, t0, lds, whole, down, acc);
}

// Whether output chunks of 8 features can be stored whole.
bool whole_chunks(const Mx4LinearArgs& a, DType out_dt) {
  const int64_t per = out_dt == kF32 ? 4 : 8;
  bool ok = a.out_rs % per == 0 && a.out_hs % per == 0;
  for (int g = 0; g < a.n_groups; ++g)
    ok = ok && (reinterpret_cast<uintptr_t>(a.out[g]) & 15) == 0;
  return ok;
}

// Dynamic LDS beyond 64 KB has to be asked for, once per kernel and device.
template <typename F>
hipError_t allow_lds(F fn, size_t bytes, std::atomic<uint64_t>& set) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  if (dev < 64 && (set.load(std::memory_order_acquire) & (uint64_t{1} << dev))) return hipSuccess;
  e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn),
                          hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == hipSuccess && dev < 64) set.fetch_or(uint64_t{1} << dev, std::memory_order_acq_rel);
  return e;
}

// Long rows of x over few features: a workgroup stages all of x for 16 features, so what bounds
// the call is that work on a part of the CUs, and its columns split over workgroups. The sums'
// way through memory costs 1.2 us, which staged columns x groups of `kSplitWork` make up for
// (us, split / not, 5120 -> 1280: 5 rows f32, 300: 7.3 / 9.9; 16 rows, 960: 8.7 / 16.3; 2 rows,
// 120: 7.1 / 6.4; 2048 -> 512, 8 rows f32, 192: 6.9 / 5.7; 16, 384: 8.0 / 8.6). Splits of fewer
// groups are faster down to 3 (16 rows 4096 -> 1024: 8.9 us, of 5 10.7, of 8 10.7).
constexpr int kSplitLeast = 3, kSplitWork = 200;
bool rows_split(const Mx4LinearArgs& a, int cols) {
  const int groups = (a.n_in / kMx4Block + kGroup - 1) / kGroup;
  return cols * groups >= kSplitWork && groups >= 2 * kSplitLeast &&
         (a.n_out + 15ll) / 16 * a.n_groups <= 128;
}

// Few rows: the waves that share a tile, and the groups staged at a time.
struct RowsShape {
  int ks, chunk;
  bool many;  // more than one workgroup per CU
  int splits, per_split;  // workgroups that share a row's groups, groups of each
  size_t lds;
};
RowsShape rows_shape(const Mx4LinearArgs& a, int ct, int cols) {
  int groups = (a.n_in / kMx4Block + kGroup - 1) / kGroup;
  const int64_t tiles = (a.n_out + 15ll) / 16 * a.n_groups;
  const size_t pad = 16 * cols, per = cols ? 2 * kMx4Block * kGroup * cols : 17 * 16 * kGroup;
  int ks = kRowsWaves, fit = 0;
  bool many = false;
  for (;; ks /= 2) {
    // x whole where a CU has one workgroup, else what leaves room for a second (more
    // columns than a tile's want it whole all the same: 8 f32 rows 1280 -> 51866 23.9 us in two
    // pieces, 20.6 whole).
    many = tiles * ks > 256 * kRowsWaves;
    const size_t room = (many && ct == 1 ? 78 : 156) * 1024 - kRowsWaves * kStage;
    fit = static_cast<int>((room - pad) / per);
    if (fit < groups) fit = fit / ks * ks;  // every wave has as many in a piece
    if (ks == 1 || (fit && tiles * ks <= 2048 && ks / 2 < groups)) break;
  }
  const int wide = 16 * (kRowsWaves / ks);
  const int64_t units = (a.n_out + wide - 1ll) / wide * a.n_groups;
  int splits = 1;
  if (a.part && rows_split(a, cols))
    splits = static_cast<int>(std::min<int64_t>(
        {256 / units, groups / kSplitLeast, kMx4MaxSplits,
         static_cast<int64_t>(a.part_floats) / (units * wide * a.n_tokens),
         static_cast<int64_t>(a.counter_words) / kMx4CounterStride >= units ? kMx4MaxSplits : 1}));
  splits = std::max(splits, 1);
  const int per_split = (groups + splits - 1) / splits;
  splits = (groups + per_split - 1) / per_split;
  if (splits > 1) {
    groups = per_split;
    fit = static_cast<int>((156 * 1024 - kRowsWaves * kStage - pad) / per);
    if (fit < groups) fit = fit / ks * ks;
  }
  RowsShape r{ks, std::min(groups, std::max(ks, fit)), many, splits, per_split, 0};
  r.lds = std::max<size_t>(sizeof(float) * 16 * kRowsWaves * (16 * ct + 1),
                           kRowsWaves * kStage + per * r.chunk + pad);
  return r;
}

template <typename XT, int kCT, int kBatch, bool kMany>
hipError_t launch_rows(const Mx4LinearArgs& a, const RowsShape& r, DType out_dt, hipStream_t s) {
  constexpr size_t kMost = 160 * 1024;
  if (r.lds > kMost) return hipErrorInvalidConfiguration;
  static std::atomic<uint64_t> set{0};
  const hipError_t e = allow_lds(&mx4_rows<XT, kCT, kBatch, kMany>, kMost, set);
  if (e != hipSuccess) return e;
  const int wide = 16 * (kRowsWaves / r.ks);
  const dim3 grid((a.n_out + wide - 1) / wide, a.n_groups, r.splits);
  const uint32_t inv = static_cast<uint32_t>((1ull << 32) / (4 * kGroup * r.chunk) + 1);
  hipLaunchKernelGGL((mx4_rows<XT, kCT, kBatch, kMany>), grid, dim3(64 * kRowsWaves), r.lds, s, a,
                     r.ks, r.chunk, inv, r.per_split, static_cast<int>(out_dt));
  return hipGetLastError();
}

template <typename XT, int kCT>
hipError_t launch_rows_ct(const Mx4LinearArgs& a, DType out_dt, hipStream_t s) {
  const RowsShape r = rows_shape(a, kCT, sizeof(XT) == 1 ? 0 : kParts<XT> * a.n_tokens);
  const int groups = (r.chunk + r.ks - 1) / r.ks;
  if (r.many) return launch_rows<XT, kCT, kCT == 1 ? 5 : 3, true>(a, r, out_dt, s);
  if (groups <= 1) return launch_rows<XT, kCT, 1, false>(a, r, out_dt, s);
  return launch_rows<XT, kCT, 3, false>(a, r, out_dt, s);
}

template <typename XT>
hipError_t launch_rows_of(const Mx4LinearArgs& a, DType out_dt, hipStream_t s) {
  if constexpr (sizeof(XT) == 1) {
    return launch_rows_ct<XT, 1>(a, out_dt, s);
  } else {
    const int cols = kParts<XT> * a.n_tokens;
    if (cols <= 16) return launch_rows_ct<XT, 1>(a, out_dt, s);
    if constexpr (kParts<XT> >= 2)
      if (cols <= 32) return launch_rows_ct<XT, 2>(a, out_dt, s);
    if constexpr (kParts<XT> >= 3) return launch_rows_ct<XT, 3>(a, out_dt, s);
    return hipErrorInvalidValue;
  }
}

using Small = Tile<64, 32, 32, 32, 4>;
using Mid = Tile<64, 64, 32, 32, 2>;
using Wide = Tile<128, 128, 64, 64, 1>;
template <typename T>
int64_t tile_wgs(const Mx4LinearArgs& a) {
  return static_cast<int64_t>((a.n_out + T::BF - 1) / T::BF) *
         ((a.n_tokens + T::BT - 1) / T::BT) * a.n_groups;
}
constexpr int kMidLeast = 180;  // workgroups

// Splits of the columns of small tiles that leave CUs idle over long rows, of kUnitsLeast units at
// least. The sums' way through memory costs ~2 us. us, split / not, 5120 -> 1280 (20 units): f32 17
// rows 11.3/20.7, 64 11.7/21.3, 130 15.7/21.5; f16 64 9.8/13.1, 130 11.1/13.0; MXFP4 x, whose
// units are cheap, 64 9.0/9.0. 2048 -> 512 (8 units): f32 40 rows 9.4/10.8, f16 8.0/7.7, MXFP4
// 7.2/6.4; 1280 -> 1280 (5) in units of two at least: f32 9.9/9.8, f16 8.1/7.0.
constexpr int kUnitsLeast = 4;
int tile_splits(const Mx4LinearArgs& a, DType x_dt) {
  const int64_t wgs = tile_wgs<Small>(a), units = (a.n_in + kUnit - 1) / kUnit;
  if (a.x_scales || units < (x_dt == kF32 ? 8 : 16) || tile_wgs<Mid>(a) >= kMidLeast) return 1;
  int64_t n = std::min<int64_t>(
      {256 / wgs, units / kUnitsLeast, kMx4MaxSplits});
  if (a.part)
    n = std::min<int64_t>({n, static_cast<int64_t>(a.part_floats) / (wgs * Small::BF * Small::BT),
                           static_cast<int64_t>(a.counter_words) /
                                       (kMx4CounterStride * Small::kWaves) >= wgs ? n : 1});
  return static_cast<int>(std::max<int64_t>(n, 1));
}

template <typename T, typename XT, typename OT, bool kWords = true>
hipError_t launch_tile(const Mx4LinearArgs& a, DType out_dt, hipStream_t s) {
  if constexpr (kWords) {
    // Four scales a load where the rows' scales lie on words.
    bool words =
        a.n_in % (4 * kMx4Block) == 0 && (reinterpret_cast<uintptr_t>(a.x_scales) & 3) == 0;
    for (int g = 0; g < a.n_groups; ++g)
      words = words && (reinterpret_cast<uintptr_t>(a.w_scales[g]) & 3) == 0;
    if (!words) return launch_tile<T, XT, OT, false>(a, out_dt, s);
  }
  constexpr size_t kLds = tile_lds<T, sizeof(XT) == 1 ? 0 : sizeof(XT) == 2 ? 1 : 2>();
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  static std::atomic<uint64_t> set{0};
  const hipError_t e = allow_lds(&mx4_tile<T, XT, OT, kWords>, kLds, set);
  if (e != hipSuccess) return e;
  const int n_f = (a.n_out + T::BF - 1) / T::BF;
  const int64_t wgs = static_cast<int64_t>(n_f) * ((a.n_tokens + T::BT - 1) / T::BT);
  if (wgs > 0x7fffffff) return hipErrorInvalidConfiguration;
  const int units = (a.n_in + kUnit - 1) / kUnit;
  int splits = T::kSplits && a.part ? tile_splits(a, sizeof(XT) == 4 ? kF32 : kF16) : 1;
  const int per_split = (units + splits - 1) / splits;
  splits = (units + per_split - 1) / per_split;
  hipLaunchKernelGGL((mx4_tile<T, XT, OT, kWords>),
                     dim3(static_cast<unsigned>(wgs), a.n_groups, splits), dim3(T::kThreads), kLds,
                     s, a, n_f, whole_chunks(a, out_dt) ? 1 : 0, per_split);
  return hipGetLastError();
}

template <typename XT, typename OT>
hipError_t launch_tiles(const Mx4LinearArgs& a, DType out_dt, hipStream_t s) {
  // The largest tile that fills the chip: larger ones read x and W less often, but a CU without
  // a workgroup does nothing. Both sides of each step by workgroups, us:
  //   Large, 180 (f32, 1500 rows, 3 x 1280 -> 1280): 45.6, Wide 50.3; 120 (f32, 3000 rows 5120 ->
  //   1280): 140, Wide 108.
  //   Wide, 144 (f32, 1500 rows 384 -> 1536): 13.0, Mid 14.7; 120 (f32, 1500 rows 1280 -> 1280):
  //   30.6, Mid 21.8.
  //   Mid, 180 (MXFP4, 130 rows, 3 x 1280 -> 1280): 7.4, Small 8.0; 60 (40 rows): 6.7, Small 6.1.
  // Few rows over a vocabulary's features take large tiles too, mostly empty ones (17 rows 1280 ->
  // 51866: f32 43.5, Mid 37.6; f16 24.0, Mid 21.7; MXFP4 15.9, Wide 15.3; Mid 17.3).
  using Large = Tile<256, 128, 64, 128, 1>;
  if (tile_wgs<Large>(a) >= 160) return launch_tile<Large, XT, OT>(a, out_dt, s);
  if (tile_wgs<Wide>(a) >= 144) return launch_tile<Wide, XT, OT>(a, out_dt, s);
  if (tile_wgs<Mid>(a) >= kMidLeast) return launch_tile<Mid, XT, OT>(a, out_dt, s);
  return launch_tile<Small, XT, OT>(a, out_dt, s);
}

}  // namespace

bool linear_mx4_splits(const Mx4LinearArgs& a, DType x_dt) {
  if (a.n_tokens > kMx4Rows) return tile_splits(a, x_dt) > 1;
  if (a.x_scales) return false;
  const int parts = x_dt == kF32 ? kParts<float> : x_dt == kF16 ? kParts<_Float16> : 1;
  return rows_split(a, parts * a.n_tokens);
}

hipError_t launch_linear_mx4(const Mx4LinearArgs& a, DType x_dt, DType out_dt, hipStream_t s) {
  if (a.n_tokens <= 0 || a.n_out <= 0 || a.n_groups <= 0) return hipSuccess;
  if (a.n_tokens <= kMx4Rows) {
    if (a.x_scales) return launch_rows_of<uint8_t>(a, out_dt, s);
    switch (x_dt) {
      case kF32: return launch_rows_of<float>(a, out_dt, s);
      case kF16: return launch_rows_of<_Float16>(a, out_dt, s);
      case kBF16: return launch_rows_of<__bf16>(a, out_dt, s);
      default: return hipErrorInvalidValue;
    }
  }
#define WRS_MX4_TILES(XT)                                                                    \
  switch (out_dt) {                                                                          \
    case kF32: return launch_tiles<XT, float>(a, out_dt, s);                                 \
    case kF16: return launch_tiles<XT, _Float16>(a, out_dt, s);                              \
    case kBF16: return launch_tiles<XT, __bf16>(a, out_dt, s);                               \
    default: return hipErrorInvalidValue;                                                    \
  }
  if (a.x_scales) {
    WRS_MX4_TILES(uint8_t)
  } else {
    switch (x_dt) {
      case kF32: WRS_MX4_TILES(float)
      case kF16: WRS_MX4_TILES(_Float16)
      case kBF16: WRS_MX4_TILES(__bf16)
      default: return hipErrorInvalidValue;
    }
  }
#undef WRS_MX4_TILES
  return hipGetLastError();
}

}  // namespace wrs
