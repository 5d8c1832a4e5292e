// Attention of drafted trees over the KV arena.
//
// K11 (tree_attend): the rows of a tree of drafted tokens against one slot's cache.
//   Row i of a tree sees the slot's `past` keys and, of the drafted rows stored
//   behind them, itself and its ancestors: s_j = q_i.k_j / 8, out_i = softmax(s) V
//   over those j only. parents[i] in [0, i) is the row's parent; anything else
//   makes it a child of the last cached token, so any parents end every walk.
//   A workgroup of four waves runs one block of 16 kRT rows of one head over one
//   chunk of the keys; wave w takes the chunk's 16-key steps w, w + 4, ... with an
//   online softmax of its own, the waves merge their (max, sum, O) in LDS, and the
//   chunks of a block merge through memory (the last workgroup to count in adds
//   the partials up in chunk order, so results do not depend on which it is).
//   Only the steps that reach past the cache test the ancestor bits.
//   The products run on the f32 matrix pipe, f16 planes widened exactly:
//   S^T = K Q^T with lane (c, g) holding key c's values d = 16 g + 0..15, so that
//   lane (r, g) gets scores of keys 4 g + 0..3 of row r, which are the B operand of
//   O^T += V^T P^T as they stand.
#include "wrs_internal.hpp"

#include <algorithm>

namespace wrs {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kStep = 16;       // keys per wave step
constexpr int kPitch = 66;      // LDS pitch (floats) of a merge row
constexpr int kCounterStride = 32;  // 128 bytes between merge counters
constexpr int kMergeLoads = 8;  // partials in flight per thread in the merge
constexpr int kRawBuffer = 0x00020000;  // buffer resource word 3: raw, 32-bit data format

// 4 values of a plane row at byte offset `o` (multiple of 4 values), zero past the range.
template <typename KT>
__device__ inline f32x4 load4(const __amdgpu_buffer_rsrc_t& rs, uint32_t o) {
  if constexpr (sizeof(KT) == 4)
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0));
  else
    return __builtin_convertvector(
        __builtin_bit_cast(f16x4, __builtin_amdgcn_raw_buffer_load_b64(rs, o, 0, 0)), f32x4);
}

template <typename KT, int kRT>
__global__ __launch_bounds__(64 * kWaves) void tree_attend(TreeArgs a) {
  constexpr int kRows = 16 * kRT;
  __shared__ float mo[kWaves][kRows * kPitch];  // a wave's O rows
  __shared__ float ml[kWaves][2][kRows];        // and their max and sum
  __shared__ int par[kTreeMaxNodes];
  __shared__ uint32_t anc[kRows][kTreeMaxNodes / 32];  // ancestors-or-self of the block's rows
  __shared__ int last_flag;

  // The workgroups of one head's chunk, which read the same rows, share an XCD's L2.
  const int lid = xcd_remap(blockIdx.x, gridDim.x);
  int t = 0;
  for (int step = kTreeMaxTrees / 2; step; step >>= 1)
    if (t + step < a.n_trees && a.wg0[t + step] <= lid) t += step;
  const int past = a.past[t], nodes = a.nodes[t], total = past + nodes;
  const int n_blk = (nodes + kRows - 1) / kRows;
  const int n_split = (total + a.chunk - 1) / a.chunk;
  const int local = lid - a.wg0[t];
  const int blk = local % n_blk, hs = local / n_blk;
  const int split = hs % n_split, h = hs / n_split;
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
  const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<KT*>(static_cast<const KT*>(a.k) + plane), 0, range, kRawBuffer);
  const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<KT*>(static_cast<const KT*>(a.v) + plane), 0, range, kRawBuffer);

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

  const bool tail = key1 > past;  // the chunk holds drafted rows
  if (tail) {
    for (int i = tid; i < nodes; i += 64 * kWaves) {
      const int p = a.parents[q_row + i];
      par[i] = static_cast<unsigned>(p) < static_cast<unsigned>(i) ? p : -1;
    }
    for (int i = tid; i < kRows * (kTreeMaxNodes / 32); i += 64 * kWaves) anc[0][i] = 0u;
    __syncthreads();
    if (tid < kRows && row0 + tid < nodes) {
      // Ancestors come in falling order: a word is whole when the walk leaves it.
      int n = row0 + tid, w = n >> 5;
      uint32_t bits = 0;
      for (; n >= 0; n = par[n]) {
        if ((n >> 5) != w) {
          anc[tid][w] = bits;
          bits = 0;
          w = n >> 5;
        }
        bits |= 1u << (n & 31);
      }
      anc[tid][w] = bits;
    }
    __syncthreads();
  }

  f32x4 o[kRT][4];
  float m[kRT], l[kRT];
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[rt] = -INFINITY;
    l[rt] = 0.f;
  }
  for (int j0 = key0 + kStep * wave; j0 < key1; j0 += kStep * kWaves) {
    f32x4 kx[4], vx[4];
    const uint32_t ko = static_cast<uint32_t>(j0 - key0 + c) * kRowBytes + 16 * g * sizeof(KT);
    const uint32_t vo = static_cast<uint32_t>(j0 - key0 + 4 * g) * kRowBytes + 4 * c * sizeof(KT);
#pragma unroll
    for (int i = 0; i < 4; ++i) kx[i] = load4<KT>(krs, ko + 4 * i * sizeof(KT));
#pragma unroll
    for (int i = 0; i < 4; ++i) vx[i] = load4<KT>(vrs, vo + i * kRowBytes);
    // Drafted values that a row does not see have weight 0, and 0 times an infinity or
    // NaN is NaN: such values leave the product and are added row by row.
    const bool masked = j0 + kStep > past;
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
      uint32_t seen = 0xF;  // bit i: the row sees key j0 + 4 g + i
      if (masked) {
        seen = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = j0 + 4 * g + i - past;
          const bool vis =
              n < 0 || (n < nodes && ((anc[16 * rt + c][(n & (kTreeMaxNodes - 1)) >> 5] >> (n & 31)) & 1));
          seen |= vis ? 1u << i : 0u;
          if (!vis) s[i] = -INFINITY;
        }
      }
      const float mx = max_x16_x32(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
      const float m_new = fmaxf(m[rt], mx);
      const float alpha = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - m_new);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      m[rt] = m_new;
      f32x4 p;
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(s[i] - m_use);
      l[rt] = __builtin_fmaf(l[rt], alpha, (p[0] + p[1]) + (p[2] + p[3]));
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o[rt][dt] *= alpha;
      if (!odd) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int dt = 0; dt < 4; ++dt)
            o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[i][dt], p[i], o[rt][dt], 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int dt = 0; dt < 4; ++dt)
            o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                __builtin_isfinite(vx[i][dt]) ? vx[i][dt] : 0.f, p[i], o[rt][dt], 0, 0, 0);
          for (int kg = 0; kg < 4; ++kg) {
            // Weight and sight of key j0 + 4 kg + i, and its row's values of this lane's
            // columns (lane group g holds d = 16 g + 4 e + dt at o[dt][e]).
            const float pk = __shfl(p[i], c + 16 * kg);
            const bool vis = (__shfl(static_cast<int>(seen), c + 16 * kg) >> i) & 1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const f32x4 vk = load4<KT>(
                  vrs, static_cast<uint32_t>(j0 - key0 + 4 * kg + i) * kRowBytes +
                           (16 * g + 4 * e) * static_cast<uint32_t>(sizeof(KT)));
#pragma unroll
              for (int dt = 0; dt < 4; ++dt)
                if (vis && !__builtin_isfinite(vk[dt])) o[rt][dt][e] += pk * vk[dt];
            }
          }
        }
      }
    }
  }

  // The waves' rows meet in LDS.
#pragma unroll
  for (int rt = 0; rt < kRT; ++rt) {
    l[rt] = sum_x16_x32(l[rt]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 16 * g + 4 * e;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) mo[wave][(16 * rt + c) * kPitch + d + dt] = o[rt][dt][e];
    }
    if (g == 0) {
      ml[wave][0][16 * rt + c] = m[rt];
      ml[wave][1][16 * rt + c] = l[rt];
    }
  }
  __syncthreads();
  const int rows = min(kRows, nodes - row0);
  float* const part =
      a.part + (static_cast<int64_t>(a.wg0[t] + h * n_split * n_blk + blk) * kRows) * kTreePart;
  const int64_t part_step = static_cast<int64_t>(n_blk) * kRows * kTreePart;  // to the next chunk
  for (int e = tid; e < rows * 64; e += 64 * kWaves) {
    const int r = e >> 6, d = e & 63;
    float M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, ml[w][0][r]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = ml[w][0][r];
      const float x = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
      L = __builtin_fmaf(ml[w][1][r], x, L);
      acc = __builtin_fmaf(mo[w][r * kPitch + d], x, acc);
    }
    if (n_split == 1) {
      a.o[(q_row + row0 + r) * a.o_rs + h * 64 + d] = L == 0.f ? 0.f : acc / L;
    } else {
      float* const p = part + split * part_step + r * kTreePart;
      st_agent(p + 2 + d, acc);
      if (d == 0) {
        st_agent(p, M);
        st_agent(p + 1, L);
      }
    }
  }
  if (n_split == 1) return;
  // Every wave's stores are performed before the chunk counts in.
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  unsigned* const counter =
      a.counters + static_cast<int64_t>(a.wg0[t] + h * n_split * n_blk + blk) * kCounterStride;
  if (tid == 0)
    last_flag = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                static_cast<unsigned>(n_split - 1);
  __syncthreads();
  if (!last_flag) return;
  for (int e = tid; e < rows * 64; e += 64 * kWaves) {
    const int r = e >> 6, d = e & 63;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int s0 = 0; s0 < n_split; s0 += kMergeLoads) {
      float ms[kMergeLoads], ls[kMergeLoads], as[kMergeLoads];
#pragma unroll
      for (int j = 0; j < kMergeLoads; ++j) {
        ms[j] = -INFINITY;
        ls[j] = as[j] = 0.f;
        if (s0 + j < n_split) {
          const float* p = part + (s0 + j) * part_step + r * kTreePart;
          ms[j] = ld_agent(p);
          ls[j] = ld_agent(p + 1);
          as[j] = ld_agent(p + 2 + d);
        }
      }
      float Mb = M;
#pragma unroll
      for (int j = 0; j < kMergeLoads; ++j) Mb = fmaxf(Mb, ms[j]);
      const float x = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - Mb);
      L *= x;
      acc *= x;
#pragma unroll
      for (int j = 0; j < kMergeLoads; ++j) {
        const float w = ms[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[j] - Mb);
        L = __builtin_fmaf(ls[j], w, L);
        acc = __builtin_fmaf(as[j], w, acc);
      }
      M = Mb;
    }
    a.o[(q_row + row0 + r) * a.o_rs + h * 64 + d] = L == 0.f ? 0.f : acc / L;
  }
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

int block_rows(const TreeArgs& a) {
  int most = 0;
  for (int t = 0; t < a.n_trees; ++t) most = std::max(most, a.nodes[t]);
  return most <= 16 ? 16 : kTreeMaxRows;
}

}  // namespace

int64_t tree_plan(TreeArgs& a, bool split) {
  const int rows = block_rows(a);
  int64_t blocks = 0, work = 0;
  int longest = 1;
  for (int t = 0; t < a.n_trees; ++t) {
    const int64_t b = static_cast<int64_t>((a.nodes[t] + rows - 1) / rows) * a.n_heads;
    const int total = a.past[t] + a.nodes[t];
    blocks += b;
    work += b * total;
    longest = std::max(longest, total);
  }
  // Workgroups of a launch: the first tree's start and the sum of all.
  auto lay = [&](int chunk) {
    int64_t n = 0;
    a.chunk = chunk;
    for (int t = 0; t < a.n_trees; ++t) {
      a.wg0[t] = static_cast<int>(std::min<int64_t>(n, 0x7fffffff));
      const int total = a.past[t] + a.nodes[t];
      n += static_cast<int64_t>((a.nodes[t] + rows - 1) / rows) * a.n_heads *
           ((static_cast<int64_t>(total) + chunk - 1) / chunk);
    }
    return n;
  };
  constexpr int kLeast = 2 * kStep * kWaves;  // keys worth a workgroup
  if (split && blocks < kTreeMaxWgs / 2 && longest > kLeast) {
    int64_t chunk = std::max<int64_t>(kLeast, (work + kTreeMaxWgs * 3 / 4 - 1) / (kTreeMaxWgs * 3 / 4));
    for (chunk = (chunk + kLeast - 1) / kLeast * kLeast; chunk < longest; chunk += kLeast) {
      const int64_t n = lay(static_cast<int>(chunk));
      if (n <= kTreeMaxWgs) return n;
    }
  }
  return lay(longest);
}

hipError_t launch_tree_attend(const TreeArgs& a, DType dt, int64_t wgs, hipStream_t s) {
  if (wgs <= 0) return hipSuccess;
  if (wgs > 0x7fffffff) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(wgs)), block(64 * kWaves);
  const bool few = block_rows(a) == 16;
#define WRS_TREE(KT, RT) hipLaunchKernelGGL((tree_attend<KT, RT>), grid, block, 0, s, a)
  switch (dt) {
    case kF16:
      if (few) WRS_TREE(_Float16, 1); else WRS_TREE(_Float16, 2);
      break;
    case kF32:
      if (few) WRS_TREE(float, 1); else WRS_TREE(float, 2);
      break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_TREE
  return hipGetLastError();
}

}  // namespace wrs
