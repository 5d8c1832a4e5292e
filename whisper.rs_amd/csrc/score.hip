// Log probabilities of given tokens, the entropy and the likeliest alternatives of rows of logits.
//
// K20 (score_rows): over the allowed entries of a row, m the largest, z_j = (x_j - m) / T:
//   lp_j = z_j - ln s,  s = sum e^z,  H = ln s - sum z e^z / s,
//   and the k largest x_j with their indices, the lowest index first among equals.
//   A row is read once: every thread keeps the maximum of its entries (and which group of 16 held it
//   first) and its sums relative to that maximum. The k largest entries then lie in the k threads
//   whose maxima are the k largest under the same order (value, then index): a bound from 64 maxima of
//   neighbouring threads leaves few threads, these look their group up again for the index, and the
//   entries of the k chosen ones, a few hundred bytes each, are read again, an entry at or above the
//   k-th chosen maximum being one of at most k * (entries of a thread) candidates. Nothing else depends
//   on values, so equal logits cost what others do.
//   s is kept without the largest entry's 1 (its thread's entries are summed again, a piece a thread),
//   and ln s = log1p of it: a token of probability 1 - 1e-7 has its log probability to 2^-22 too.
//   Few rows split over several workgroups, which merge through memory (the last to count in joins
//   the parts in order; sums and order do not depend on which it is).
#include "wrs_internal.hpp"

#include <algorithm>
#include <cfloat>

namespace wrs {
namespace {

typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32u __attribute__((aligned(1)));

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kGroup = 16;  // entries of a thread's group: 16-byte pieces, kThreads pieces apart
constexpr int kRun = kThreads / 64;  // neighbouring threads that share a maximum of the bound
constexpr int kMostPieces = kScoreChunk / kThreads / 4;  // of a thread, at most (f32: 4 entries)
constexpr int kCounterStride = 32;   // 128 bytes between merge counters
constexpr float kLow = -1e30f;       // finite: times a weight of 0 it is 0

// An entry's order as an unsigned number: by value, the lower index first among equals.
__device__ inline uint64_t key_of(float x, uint32_t index) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // one zero
  const uint32_t o = u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
  return static_cast<uint64_t>(o) << 32 | (0xFFFFFFFFu - index);
}
__device__ inline float value_of(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ inline int index_of(uint64_t key) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

template <typename T>
struct Piece {
  static constexpr int kN = 16 / sizeof(T);  // entries of 16 bytes
};
// Entry e of a 16-byte piece as f32. T: float, _Float16 or uint16_t (bf16).
template <typename T>
__device__ inline float entry(const u32x4& p, int e) {
  const uint32_t w = p[sizeof(T) == 4 ? e : e >> 1];
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(float, w);
  } else {
    if constexpr (__is_same(T, uint16_t))
      return __builtin_bit_cast(float, e & 1 ? w & 0xFFFF0000u : w << 16);
    else
      return static_cast<float>(
          __builtin_bit_cast(_Float16, static_cast<uint16_t>(e & 1 ? w >> 16 : w)));
  }
}

// A row's (or chunk's) entries: x[0 .. n), entry i allowed where ok[i] is not zero.
template <typename T, bool kMask>
struct Row {
  const T* x;
  const uint8_t* ok;
  int n;
  static constexpr int kN = Piece<T>::kN;
  // Piece p, hidden entries and those past the end at -infinity.
  template <bool kWhole>
  __device__ inline void load(int p, float (&v)[kN]) const {
    const int i0 = p * kN;
    if (kWhole || i0 + kN <= n) {
      const u32x4 w = *reinterpret_cast<const u32x4u*>(x + i0);
#pragma unroll
      for (int e = 0; e < kN; ++e) v[e] = entry<T>(w, e);
      if constexpr (kMask) {
#pragma unroll
        for (int h = 0; h < kN / 4; ++h) {
          const uint32_t m = *reinterpret_cast<const u32u*>(ok + i0 + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(m & (0xFFu << (8 * e)))) v[4 * h + e] = -INFINITY;
        }
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      v[e] = -INFINITY;
      if (i0 + e < n && (!kMask || ok[i0 + e])) {
        if constexpr (__is_same(T, uint16_t))
          v[e] = __builtin_bit_cast(float, static_cast<uint32_t>(x[i0 + e]) << 16);
        else
          v[e] = static_cast<float>(x[i0 + e]);
      }
    }
  }
};

__device__ inline float wave_max(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
__device__ inline float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}
// How many of n keys are larger than `mine`.
__device__ inline int rank_of(uint64_t mine, const uint64_t* keys, int n) {
  int r = 0;
  for (int i = 0; i < n; ++i) r += keys[i] > mine;
  return r;
}

struct Shared {
  uint64_t keys[kScoreMostTop * (kScoreChunk / kThreads)];  // candidates
  uint64_t first[kThreads];   // threads' first largest entries, and whose they are
  uint64_t best[kScoreMostTop];
  float run_max[64];
  float piece[2][kMostPieces];  // sums of the pieces of the largest entry's thread
  float sums[2][kWaves];
  float bound;
  int first_of[kThreads], chosen[kScoreMostTop];
  int n_first, n_keys, last;
};

// One chunk: its largest entry m and the sums without it, both in the exp2 domain of `scale`
// (s = sum 2^(scale (x - m)), t = sum scale (x - m) 2^(..)), and its k best entries in sh.best, keys of
// entries that are not there 0. Every thread gets m, s and t.
template <typename T, bool kMask>
__device__ inline void scan(const Row<T, kMask>& row, int index0, int k, float scale, Shared& sh,
                            float& m_out, float& s_out, float& t_out) {
  constexpr int kN = Piece<T>::kN, kTurns = kGroup / kN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int pieces = (row.n + kN - 1) / kN;
  float m = -INFINITY, s = 0.f, t = 0.f;
  int at = 0;  // the group that held m first
  auto take = [&](const float (&v)[kTurns][kN], int g) __attribute__((always_inline)) {
    float top = v[0][0];
#pragma unroll
    for (int u = 0; u < kTurns; ++u)
#pragma unroll
      for (int e = 0; e < kN; ++e) top = fmaxf(top, v[u][e]);
    if (top > m) at = g;
    const float m_new = fmaxf(fmaxf(m, top), -FLT_MAX);
    const float d = fmaxf((fmaxf(m, -FLT_MAX) - m_new) * scale, kLow);
    const float r = __builtin_amdgcn_exp2f(d);
    t = r * __builtin_fmaf(d, s, t);
    s *= r;
    m = fmaxf(m, top);
#pragma unroll
    for (int u = 0; u < kTurns; ++u)
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float z = (v[u][e] - m_new) * scale, w = __builtin_amdgcn_exp2f(z);
        s += w;
        t = __builtin_fmaf(fmaxf(z, kLow), w, t);
      }
  };
  const int groups = (pieces + kTurns * kThreads - 1) / (kTurns * kThreads);
  const int whole = row.n / (kN * kTurns * kThreads);  // groups with every entry in the row
  for (int g = 0; g < groups; ++g) {
    float v[kTurns][kN];
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int p = (g * kTurns + u) * kThreads + tid;
      if (g < whole)
        row.template load<true>(p, v[u]);
      else
        row.template load<false>(p, v[u]);
    }
    take(v, g);
  }

  // A bound under the k-th largest thread's maximum: that of 64 runs of threads.
  float run = m;
#pragma unroll
  for (int d = 1; d < kRun; d <<= 1) run = fmaxf(run, __shfl_xor(run, d));
  if (tid % kRun == 0) sh.run_max[tid / kRun] = run;
  if (tid == 0) sh.n_first = sh.n_keys = 0;
  __syncthreads();
  const float mine = sh.run_max[lane];
  const float m_all = wave_max(mine);
  if (wave == 0) {
    int r = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
      const float other = __builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), i));
      r += other > mine || (other == mine && i < lane);
    }
    if (r == k - 1) sh.bound = mine;
  }
  __syncthreads();
  if (m > -INFINITY && m >= sh.bound) {
    int index = 0;
    bool found = false;
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int p = (at * kTurns + u) * kThreads + tid;
      float v[kN];
      row.template load<false>(p, v);
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (!found && v[e] == m) {
          found = true;
          index = p * kN + e;
        }
    }
    const int i = atomicAdd(&sh.n_first, 1);
    sh.first[i] = key_of(m, index0 + index);
    sh.first_of[i] = tid;
  }
  __syncthreads();
  const int n_first = sh.n_first, n_chosen = min(n_first, k);
  if (tid < n_first) {
    const int r = rank_of(sh.first[tid], sh.first, n_first);
    if (r < k) {
      sh.chosen[r] = sh.first_of[tid];
      sh.best[r] = sh.first[tid];
    }
  }
  __syncthreads();
  // Entries of the chosen threads, a piece a thread.
  const int per = groups * kTurns;
  if (n_chosen > 0) {
    const uint64_t least = n_chosen == k ? sh.best[k - 1] : 0;
    const int top_at = index_of(sh.best[0]) - index0;
    for (int i = tid; i < n_chosen * per; i += kThreads) {
      const int j = i / per, q = i - j * per;
      const int p = q * kThreads + sh.chosen[j];
      float v[kN];
      row.template load<false>(p, v);
      float ps = 0.f, pt = 0.f;
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const uint64_t key = key_of(v[e], index0 + p * kN + e);
        if (v[e] > -INFINITY && key >= least) sh.keys[atomicAdd(&sh.n_keys, 1)] = key;
        if (j == 0 && p * kN + e != top_at) {
          const float z = (v[e] - m_all) * scale, w = __builtin_amdgcn_exp2f(z);
          ps += w;
          pt = __builtin_fmaf(fmaxf(z, kLow), w, pt);
        }
      }
      if (j == 0) {
        sh.piece[0][q] = ps;
        sh.piece[1][q] = pt;
      }
    }
  }
  // The threads' sums, without the largest entry's thread.
  {
    const float low = fmaxf(m_all, -FLT_MAX);
    const float d = fmaxf((fmaxf(m, -FLT_MAX) - low) * scale, kLow);
    const float r = __builtin_amdgcn_exp2f(d);
    const bool out = n_chosen > 0 && tid == sh.chosen[0];
    const float ws = wave_sum(out ? 0.f : r * s);
    const float wt = wave_sum(out ? 0.f : r * __builtin_fmaf(d, s, t));
    if (lane == 0) {
      sh.sums[0][wave] = ws;
      sh.sums[1][wave] = wt;
    }
  }
  __syncthreads();
  const int n_keys = sh.n_keys;
  if (tid < k) sh.best[tid] = 0;
  s = t = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    s += sh.sums[0][w];
    t += sh.sums[1][w];
  }
  if (n_chosen > 0) {
    float ps = 0.f, pt = 0.f;
    for (int q = lane; q < per; q += 64) {
      ps += sh.piece[0][q];
      pt += sh.piece[1][q];
    }
    s += wave_sum(ps);
    t += wave_sum(pt);
  }
  __syncthreads();
  for (int i = tid; i < n_keys; i += kThreads) {
    const int r = rank_of(sh.keys[i], sh.keys, n_keys);
    if (r < k) sh.best[r] = sh.keys[i];
  }
  __syncthreads();
  m_out = m_all;
  s_out = s;
  t_out = t;
}

template <typename T, bool kMask>
__global__ __launch_bounds__(kThreads) void score_rows(ScoreArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.y + static_cast<int64_t>(blockIdx.z) * 65535;
  if (r >= a.n_rows) return;
  const int i0 = blockIdx.x * a.chunk;
  const T* const x = static_cast<const T*>(a.logits) + r * a.row_stride;
  const uint8_t* const ok = kMask ? a.allowed + r * a.allowed_stride : nullptr;
  const int token = a.tokens ? a.tokens[r] : -1;
  const Row<T, kMask> row = {x + i0, kMask ? ok + i0 : nullptr, min(a.chunk, a.n_vocab - i0)};
  const int k = max(a.top_k, 1);
  float m, s, t;  // of the allowed entries; s and t without the largest entry
  scan<T, kMask>(row, i0, k, a.scale_log2, sh, m, s, t);
  if (a.n_chunks > 1) {
    float* const part = a.part + (r * a.n_chunks + blockIdx.x) * kScorePart;
    if (tid == 0) {
      st_agent(part, m);
      st_agent(part + 1, s);
      st_agent(part + 2, t);
    }
    if (tid < k)
      __hip_atomic_store(reinterpret_cast<uint64_t*>(part + 4) + tid, sh.best[tid],
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // Every wave's stores are performed before the chunk counts in.
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    unsigned* const counter = a.counters + r * kCounterStride;
    if (tid == 0)
      sh.last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                static_cast<unsigned>(a.n_chunks - 1);
    __syncthreads();
    if (!sh.last) return;
    const float* const all = a.part + r * a.n_chunks * kScorePart;
    const int n = a.n_chunks * k;
    for (int i = tid; i < n; i += kThreads) {
      const int c = i / k, j = i - c * k;
      sh.keys[i] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(all + c * kScorePart + 4) + j,
                                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (tid < k) sh.best[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t key = sh.keys[i];
      if (key == 0) continue;
      const int p = rank_of(key, sh.keys, n);
      if (p < k) sh.best[p] = key;
    }
    __syncthreads();
    // The chunks' sums in their order; the one that holds the largest entry leaves its 1 out.
    const int home = sh.best[0] ? index_of(sh.best[0]) / a.chunk : -1;
    m = -INFINITY;
    for (int c = 0; c < a.n_chunks; ++c) m = fmaxf(m, ld_agent(all + c * kScorePart));
    s = t = 0.f;
    for (int c = 0; c < a.n_chunks; ++c) {
      const float* const p = all + c * kScorePart;
      const float mc = ld_agent(p), tc = ld_agent(p + 2);
      float sc = ld_agent(p + 1);
      if (c != home && mc > -INFINITY) sc += 1.f;
      const float d =
          fmaxf((fmaxf(mc, -FLT_MAX) - fmaxf(m, -FLT_MAX)) * a.scale_log2, kLow);
      const float w = __builtin_amdgcn_exp2f(d);
      s = __builtin_fmaf(w, sc, s);
      t = __builtin_fmaf(w, __builtin_fmaf(d, sc, tc), t);
    }
    if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // A row with an allowed NaN or +infinity has no distribution; one without an entry gives none
  // of its tokens.
  const bool odd = s != s || m == INFINITY, none = !odd && m == -INFINITY;
  const float ln_s = log1pf(s);
  auto logprob = [&](float v) {
    if (odd) return NAN;
    if (none) return -INFINITY;
    return (v - m) / a.temperature - ln_s;
  };
  if (tid < a.top_k) {
    const uint64_t key = odd ? 0 : sh.best[tid];
    const int64_t o = r * a.top_k + tid;
    if (a.top_ids) a.top_ids[o] = key ? index_of(key) : -1;
    if (a.top_logprobs) a.top_logprobs[o] = key ? logprob(value_of(key)) : odd ? NAN : -INFINITY;
  }
  if (tid == 0 && a.logprobs) {
    float v = -INFINITY;
    if (token >= 0 && token < a.n_vocab && (!kMask || ok[token])) {
      if constexpr (__is_same(T, uint16_t))
        v = __builtin_bit_cast(float, static_cast<uint32_t>(x[token]) << 16);
      else
        v = static_cast<float>(x[token]);
    }
    a.logprobs[r] = logprob(v);
  }
  if (tid == 64 && a.entropy)
    a.entropy[r] = odd ? NAN : none ? 0.f : ln_s - t * 0.6931471805599453f / (1.f + s);
}

}  // namespace

void score_plan(ScoreArgs& a, bool split) {
  // Rows that fill the GPU are taken whole.
  int64_t chunks = 1;
  if (split) chunks = std::max<int64_t>(1, kScoreMaxWgs / std::max<int64_t>(a.n_rows, 1));
  // Not less than 4 groups of every thread's.. entries a workgroup.
  chunks = std::min<int64_t>(chunks, (a.n_vocab + 4095) / 4096);
  chunks = std::min<int64_t>(chunks, kScoreMostChunks);
  chunks = std::max<int64_t>(chunks, (a.n_vocab + kScoreChunk - 1) / kScoreChunk);
  a.chunk = static_cast<int>(((a.n_vocab + chunks - 1) / chunks + 63) / 64 * 64);
  a.n_chunks = (a.n_vocab + a.chunk - 1) / a.chunk;
}

hipError_t launch_score_rows(const ScoreArgs& a, DType dt, hipStream_t s) {
  if (a.n_rows <= 0) return hipSuccess;
  if (a.top_k > kScoreMostTop || a.chunk > kScoreChunk || a.n_chunks > kScoreMostChunks)
    return hipErrorInvalidValue;
  const int64_t z = (a.n_rows + 65534) / 65535;
  if (z > 65535) return hipErrorInvalidConfiguration;
  const dim3 grid(a.n_chunks, static_cast<unsigned>(std::min<int64_t>(a.n_rows, 65535)),
                  static_cast<unsigned>(z));
#define WRS_SCORE(T)                                                                       \
  if (a.allowed)                                                                           \
    hipLaunchKernelGGL((score_rows<T, true>), grid, dim3(kThreads), 0, s, a);              \
  else                                                                                     \
    hipLaunchKernelGGL((score_rows<T, false>), grid, dim3(kThreads), 0, s, a)
  switch (dt) {
    case kF32: WRS_SCORE(float); break;
    case kF16: WRS_SCORE(_Float16); break;
    case kBF16: WRS_SCORE(uint16_t); break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_SCORE
  return hipGetLastError();
}

}  // namespace wrs
