// Rows of the KV arena: stored for several slots at once, read back, and the moves of an
// 8-bit arena's rows.
//
// An 8-bit arena holds each row of a head (64 values) as a byte 2^(byte - 127) and 64 codes,
// value = (code - 128) 2^(byte - 127). The power is the least that leaves no code past 127
// (1 <= byte <= 248), so a value is off by at most half a code, 1/255 to 2/255 of the row's
// largest; a row with an infinity or NaN gets byte 255 and codes of zero and reads as NaN.
// One row to a scale, because rows come one at a time, move singly (an accepted path), slide by
// any number and are cut anywhere: a scale that rows share would round the older ones again
// each time. Scaling by a power of two is exact, so what was read back stores as the same bytes.
// Scales lie in planes of their own, [layer][slot][head][pitch], a plane's rows rounded up to 64.
//
// K17 (kv_append): f32 rows of several slots into their planes, converted or quantised; 16 lanes
//   take a row of a head, 4 values each, and find its largest magnitude by DPP (as bit patterns:
//   a NaN is the largest).
// K18 (kv_read): the stored values as f32, the same way round.
//   Bound by memory. From kManyRows rows on a workgroup takes 32 rows of one head, whose codes and
//   scales are contiguous and hardly another workgroup's (rows of all heads in turn: a scale's line is
//   written by many). What is read back is written past the caches (non-temporal), and so is read what
//   is stored if it is more than they keep. 44012 rows of 12 heads to 8 bits and back (339 MB
//   each way): 62 us and 50 us, 5.4 and 6.8 TB/s; by rows of all heads 70 and 68, without the
//   non-temporal forms 68 and 67, 16 or 64 rows a workgroup 72 and 47, 64 and 50. 1500 rows of 20 heads:
//   5.2 and 4.4 us (non-temporal loads: 5.8). A step's 5 rows take 2.4 and 2.3 us, what an empty
//   launch does (64 rows of all heads a workgroup: 2.7 and 2.4).
#include "wrs_internal.hpp"

#include <algorithm>

namespace wrs {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The largest of a row of 16 lanes, in all of them.
__device__ inline uint32_t max16(uint32_t x) {
#define WRS_ROR(N)                                                                        \
  x = max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(                           \
                 0, static_cast<int>(x), 0x120 + (N), 0xF, 0xF, true)))
  WRS_ROR(8);
  WRS_ROR(4);
  WRS_ROR(2);
  WRS_ROR(1);
#undef WRS_ROR
  return x;
}

// A quarter of 16 values' codes (offset by 128) and the row's scale byte.
__device__ inline uint32_t encode4(const f32x4& x, uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float v = x[e];  // a bit cast of the element itself takes element 0
    top = max(top, __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu);
  }
  top = max16(top);
  // 2^e with the largest value in [64, 127.5) 2^e.
  const int e = static_cast<int>(top >> 23) - 133 + ((top & 0x7FFFFFu) >= 0x7F0000u ? 1 : 0);
  const int clamped = min(max(e, -126), 121);
  byte = top >= 0x7F800000u ? 255u : static_cast<uint32_t>(clamped + 127);
  const float down = __builtin_bit_cast(float, static_cast<uint32_t>(127 - clamped) << 23);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int code = min(max(static_cast<int>(__builtin_rintf(x[i] * down)), -127), 127);
    w |= static_cast<uint32_t>(byte == 255u ? 128 : code + 128) << (8 * i);
  }
  return w;
}
__device__ inline f32x4 decode4(uint32_t w, uint32_t byte) {
  // 2^(byte - 127); 255 gives infinity, and its codes are zeros: NaN.
  const float up = __builtin_bit_cast(float, byte << 23);
  f32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = (static_cast<float>((w >> (8 * i)) & 0xFFu) - 128.f) * up;
  return x;
}

constexpr int kManyRows = 16;
constexpr int64_t kOnce = 128 << 20;  // bytes that are read past the caches

// A workgroup takes rows of a head, 16 lanes each: the next 16 of all heads', or 32 of one head.
enum class Order { kAllHeads, kByHead, kByHeadOnce };
constexpr int block_rows(bool by_head) { return by_head ? 32 : 16; }
// Workgroups that a slot's K (or V) rows take.
__host__ __device__ inline int slot_blocks(bool by_head, int rows, int n_heads) {
  const int n = block_rows(by_head);
  return by_head ? (rows + n - 1) / n * n_heads : (rows * n_heads + n - 1) / n;
}
// kInTurn: the slots' workgroups follow each other; else each has as many as the longest one.
template <DType kD, bool kStore, Order kOrder, bool kInTurn, int kSlots>
__global__ __launch_bounds__(256) void kv_rows(KvSlotRows<kSlots> a) {
  constexpr bool kByHead = kOrder != Order::kAllHeads;
  constexpr int kBlockRows = block_rows(kByHead), kTurns = kBlockRows / 16;
  int u = blockIdx.z, block = blockIdx.x;
  if constexpr (kInTurn) {
    // Slots past the last one start past every workgroup.
    u = -1;
    for (int i = 0; i < a.n_slots; i += 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u += a.wg0[i + j] <= block;
    }
    block -= a.wg0[u];
  }
  const int rows_here = a.count[u], sub = threadIdx.x >> 4;
  // The block's first row of a head and that head, or its first row in turn.
  int64_t first;
  int head = 0;
  if constexpr (kByHead)
    first = static_cast<int64_t>(kBlockRows) *
            divide(block, a.n_heads, a.heads_inv, head);
  else
    first = static_cast<int64_t>(kBlockRows) * block;
  const int64_t n = kByHead ? rows_here : static_cast<int64_t>(rows_here) * a.n_heads;
  if (first >= n) return;
  float* const rows = (blockIdx.y ? a.v_rows : a.k_rows) + a.row0[u] * (blockIdx.y ? a.v_rs : a.k_rs);
  const int64_t rs = blockIdx.y ? a.v_rs : a.k_rs;
  char* const plane = static_cast<char*>(blockIdx.y ? a.v : a.k);
  uint8_t* const scale = blockIdx.y ? a.v_scale : a.k_scale;
  f32x4 x[kTurns];
  uint32_t w[kTurns], byte[kTurns];
  int64_t at[kTurns], sc[kTurns];
  float* p[kTurns];
#pragma unroll
  for (int j = 0; j < kTurns; ++j) {
    // Lanes past the end take the last row (16 lanes together).
    const int t = static_cast<int>(min(first + 16 * j + sub, n - 1));
    int col = head, row = t;
    if constexpr (!kByHead) row = divide(t, a.n_heads, a.heads_inv, col);
    const int64_t r = a.plane[u] + col;  // plane of (slot, head)
    at[j] = (r * a.plane_rows + a.pos[u] + row) * 64 + 4 * (threadIdx.x & 15);
    sc[j] = r * a.scale_rows + a.pos[u] + row;
    p[j] = rows + row * rs + col * 64 + 4 * (threadIdx.x & 15);
    if constexpr (kStore) {
      const f32x4u* const from = reinterpret_cast<const f32x4u*>(p[j]);
      if constexpr (kOrder == Order::kByHeadOnce)
        x[j] = __builtin_nontemporal_load(from);
      else
        x[j] = *from;
    } else if constexpr (kD == kF32) {
      x[j] = *reinterpret_cast<const f32x4*>(plane + 4 * at[j]);
    } else if constexpr (kD == kF16) {
      x[j] = __builtin_convertvector(*reinterpret_cast<const f16x4*>(plane + 2 * at[j]), f32x4);
    } else {
      w[j] = *reinterpret_cast<const uint32_t*>(plane + at[j]);
      byte[j] = scale[sc[j]];
    }
  }
#pragma unroll
  for (int j = 0; j < kTurns; ++j) {
    if (kStore && kD == kI8) w[j] = encode4(x[j], byte[j]);  // every lane of a row
    if (first + 16 * j + sub >= n) continue;
    if constexpr (!kStore) {
      if constexpr (kD == kI8) x[j] = decode4(w[j], byte[j]);
      f32x4u* const to = reinterpret_cast<f32x4u*>(p[j]);
      if constexpr (kByHead)
        __builtin_nontemporal_store(x[j], to);
      else
        *to = x[j];
    } else if constexpr (kD == kF32) {
      *reinterpret_cast<f32x4*>(plane + 4 * at[j]) = x[j];
    } else if constexpr (kD == kF16) {
      *reinterpret_cast<f16x4*>(plane + 2 * at[j]) = __builtin_convertvector(x[j], f16x4);
    } else {
      *reinterpret_cast<uint32_t*>(plane + at[j]) = w[j];
      if ((threadIdx.x & 15) == 0) scale[sc[j]] = static_cast<uint8_t>(byte[j]);
    }
  }
}

// Rows [0, len) of every plane of a slot, codes and scales, to another one. A workgroup takes
// pieces of kMoveRows rows, every parts-th.
constexpr int kMoveRows = 256;  // 16 KB of codes: four units of 16 bytes a thread
constexpr int kMoveParts = 32767;
__global__ __launch_bounds__(256) void kv8_copy(Kv8Planes to, Kv8Planes from, int len, int parts) {
  const int which = blockIdx.z / parts, part = blockIdx.z - which * parts, tid = threadIdx.x;
  const int64_t p = blockIdx.y * from.layer + blockIdx.x;
  const uint8_t* const s = (which ? from.v : from.k) + p * from.rows * 64;
  uint8_t* const d = (which ? to.v : to.k) + p * to.rows * 64;
  const uint8_t* const ss = (which ? from.v_scale : from.k_scale) + p * from.scale_rows;
  uint8_t* const ds = (which ? to.v_scale : to.k_scale) + p * to.scale_rows;
  for (int64_t r0 = static_cast<int64_t>(part) * kMoveRows; r0 < len;
       r0 += static_cast<int64_t>(parts) * kMoveRows) {
    u32x4 x[4];
    const int n = static_cast<int>(min(static_cast<int64_t>(kMoveRows), len - r0)) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 256 * j + tid;
      x[j] = reinterpret_cast<const u32x4*>(s + r0 * 64)[i < n ? i : 0];
    }
    const uint8_t y = ss[r0 + (4 * tid < n ? tid : 0)];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 256 * j + tid;
      if (i < n) reinterpret_cast<u32x4*>(d + r0 * 64)[i] = x[j];
    }
    if (4 * tid < n) ds[r0 + tid] = y;
  }
}

// Rows [drop, len) of every plane move down to [0, len - drop), in place: a piece is read whole
// before any thread writes, and later pieces read only rows above all that was written.
__global__ __launch_bounds__(256) void kv8_slide(Kv8Planes a, int len, int drop) {
  const int64_t p = blockIdx.y * a.layer + blockIdx.x;
  uint8_t* const codes = (blockIdx.z ? a.v : a.k) + p * a.rows * 64;
  uint8_t* const scale = (blockIdx.z ? a.v_scale : a.k_scale) + p * a.scale_rows;
  const int keep = len - drop, tid = threadIdx.x;
  for (int r0 = 0; r0 < keep; r0 += kMoveRows) {
    u32x4 x[4];
    const int n = min(kMoveRows, keep - r0) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 256 * j + tid;
      x[j] = reinterpret_cast<const u32x4*>(codes + static_cast<int64_t>(r0 + drop) * 64)[i < n ? i : 0];
    }
    const uint8_t y = scale[r0 + drop + (4 * tid < n ? tid : 0)];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 256 * j + tid;
      if (i < n) reinterpret_cast<u32x4*>(codes + static_cast<int64_t>(r0) * 64)[i] = x[j];
    }
    if (4 * tid < n) scale[r0 + tid] = y;
    __syncthreads();
  }
}

// kv_keep_rows for an 8-bit arena: one wave per plane, 8 rows a pass, their codes on lanes 0..31
// and their scales on 32..39, each pass loaded whole before it is stored.
constexpr int kKeepWaves = 4;
template <int kSlots, int kMoves>
__global__ __launch_bounds__(64 * kKeepWaves) void kv8_keep_rows(KeepArgs<kSlots, kMoves> a,
                                                                 Kv8Planes s) {
  const int p = blockIdx.x * kKeepWaves + (threadIdx.x >> 6), h = p >> 1;
  if (h >= a.n_heads) return;  // whole wave
  const int u = blockIdx.y, lane = threadIdx.x & 63;
  const int64_t plane = a.off[u] / a.plane_stride + blockIdx.z * s.layer + h;
  uint8_t* const codes = ((p & 1) ? s.v : s.k) + (plane * s.rows + a.past[u]) * 64;
  uint8_t* const scale = ((p & 1) ? s.v_scale : s.k_scale) + plane * s.scale_rows + a.past[u];
  const int n = a.count[u], first = a.first[u], dst0 = a.dst0[u];
  const bool is_code = lane < 32;
  const int sub = is_code ? lane >> 2 : lane - 32, c = lane & 3;
  for (int i = 0; i < n; i += 8) {
    const uint32_t pair = a.src[(first + i + (sub & 6)) / 2];
    const int64_t src = (sub & 1) ? pair >> 16 : pair & 0xFFFFu;
    const bool in = sub < 8 && i + sub < n;
    u32x4 x = {0, 0, 0, 0};
    uint8_t y = 0;
    if (in && is_code) x = *reinterpret_cast<const u32x4*>(codes + src * 64 + 16 * c);
    if (in && !is_code) y = scale[src];
    // Both loads are done before the stores: a destination may be another lane's source.
    asm volatile("" ::"v"(x), "v"(static_cast<int>(y)) : "memory");
    __builtin_amdgcn_s_waitcnt(0);
    if (in && is_code) *reinterpret_cast<u32x4*>(codes + (dst0 + i + sub) * 64 + 16 * c) = x;
    if (in && !is_code) scale[dst0 + i + sub] = y;
  }
}

}  // namespace

template <int kSlots>
hipError_t launch_kv_slot_rows(KvSlotRows<kSlots>& a, DType dt, bool store, hipStream_t s) {
  static_assert(kSlots % 8 == 0, "read 8 at a time");
  int most = 0;
  int64_t all = 0;
  for (int u = 0; u < a.n_slots; ++u) {
    most = std::max(most, a.count[u]);
    all += a.count[u];
  }
  if (most <= 0 || a.n_heads <= 0) return hipSuccess;
  if (static_cast<int64_t>(most) * a.n_heads > 0x7fffffff - 64) return hipErrorInvalidConfiguration;
  const bool by_head = most >= kManyRows, once = all * a.n_heads * 512 > kOnce;
  const int widest = slot_blocks(by_head, most, a.n_heads);
  int64_t sum = 0;
  for (int u = 0; u < kSlots; ++u) {
    a.wg0[u] = u < a.n_slots ? static_cast<int>(std::min<int64_t>(sum, 0x7fffffff)) : 0x7fffffff;
    if (u < a.n_slots) sum += slot_blocks(by_head, a.count[u], a.n_heads);
  }
  // A grid as wide as the longest slot for each of them has empty workgroups, of which 5000 cost 1 us; slots
  // in turn cost a search (2 to 5% where few are empty). In turn and wide, 20 heads, 8-bit: a text of
  // 8191 rows and 15 single tokens 19 and 49 us, 2 of them 19.5 and 21.5, 1500 rows and 7 single tokens
  // 5.6 and 6.7, 3 pieces of 100 rows 6.1 and 5.7; 16 slots of 1, 101, .. 1501 rows 25.1 and 24.3.
  const int64_t wide = widest * static_cast<int64_t>(a.n_slots);
  const bool in_turn = by_head && sum <= 0x7fffffff && 2 * wide > 5 * sum && wide - sum > 4096;
  const dim3 grid(static_cast<unsigned>(in_turn ? sum : widest), 2, in_turn ? 1 : a.n_slots);
#define WRS_KV_ROWS_ONE(D, S, O, T) \
  hipLaunchKernelGGL((kv_rows<D, S, Order::O, T, kSlots>), grid, dim3(256), 0, s, a)
#define WRS_KV_ROWS_STORE(D, O, T)                                            \
  if (store) {                                                                \
    WRS_KV_ROWS_ONE(D, true, O, T);                                           \
  } else {                                                                    \
    WRS_KV_ROWS_ONE(D, false, O, T);                                          \
  }
#define WRS_KV_ROWS(D)                                                        \
  if (!by_head) {                                                             \
    WRS_KV_ROWS_STORE(D, kAllHeads, false);                                   \
  } else if (store && once) {                                                 \
    if (in_turn) {                                                            \
      WRS_KV_ROWS_ONE(D, true, kByHeadOnce, true);                            \
    } else {                                                                  \
      WRS_KV_ROWS_ONE(D, true, kByHeadOnce, false);                           \
    }                                                                         \
  } else if (in_turn) {                                                       \
    WRS_KV_ROWS_STORE(D, kByHead, true);                                      \
  } else {                                                                    \
    WRS_KV_ROWS_STORE(D, kByHead, false);                                     \
  }
  switch (dt) {
    case kF32: WRS_KV_ROWS(kF32); break;
    case kF16: WRS_KV_ROWS(kF16); break;
    case kI8: WRS_KV_ROWS(kI8); break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_KV_ROWS
#undef WRS_KV_ROWS_STORE
#undef WRS_KV_ROWS_ONE
  return hipGetLastError();
}
template hipError_t launch_kv_slot_rows(KvSlotRows<kRowSlots>&, DType, bool, hipStream_t);
template hipError_t launch_kv_slot_rows(KvSlotRows<kRowFewSlots>&, DType, bool, hipStream_t);

hipError_t launch_kv8_copy(const Kv8Planes& to, const Kv8Planes& from, int n_layers, int n_heads,
                           int len, hipStream_t s) {
  if (n_layers <= 0 || n_heads <= 0 || len <= 0) return hipSuccess;
  const int parts = std::min((len + kMoveRows - 1) / kMoveRows, kMoveParts);
  hipLaunchKernelGGL(kv8_copy, dim3(n_heads, n_layers, static_cast<unsigned>(2 * parts)), dim3(256),
                     0, s, to, from, len, parts);
  return hipGetLastError();
}

hipError_t launch_kv8_slide(const Kv8Planes& a, int n_layers, int n_heads, int len, int drop,
                            hipStream_t s) {
  if (n_layers <= 0 || n_heads <= 0 || drop <= 0 || len <= drop) return hipSuccess;
  hipLaunchKernelGGL(kv8_slide, dim3(n_heads, n_layers, 2), dim3(256), 0, s, a, len, drop);
  return hipGetLastError();
}

template <int kSlots, int kMoves>
hipError_t launch_kv8_keep_rows(const KeepArgs<kSlots, kMoves>& a, const Kv8Planes& p, hipStream_t s) {
  if (a.n_slots <= 0 || a.n_layers <= 0 || a.n_heads <= 0) return hipSuccess;
  if (a.n_layers > 65535 || a.n_heads > (1 << 29)) return hipErrorInvalidConfiguration;
  const dim3 grid((2 * a.n_heads + kKeepWaves - 1) / kKeepWaves, a.n_slots, a.n_layers);
  hipLaunchKernelGGL((kv8_keep_rows<kSlots, kMoves>), grid, dim3(64 * kKeepWaves), 0, s, a, p);
  return hipGetLastError();
}
template hipError_t launch_kv8_keep_rows(const KeepArgs<kKeepSlots, kKeepMoves>&, const Kv8Planes&,
                                         hipStream_t);
template hipError_t launch_kv8_keep_rows(const KeepArgs<kKeepFewSlots, kKeepFewMoves>&,
                                         const Kv8Planes&, hipStream_t);

}  // namespace wrs
