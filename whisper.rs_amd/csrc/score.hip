// Log probabilities of given tokens, the entropy and the likeliest alternatives of rows of logits.
//
// K21 (score_rows): over the allowed entries of a row, m the largest, z_j = (x_j - m) / T:
//   lp_j = z_j - ln s,  s = sum e^z,  H = ln s - sum z e^z / s,
//   and the k largest x_j with their indices, the lowest index first among equals.
//   A row is read once: every thread keeps the maximum of its entries (and which group of 16 held it
//   first) and its sums relative to that maximum. The k largest entries then lie in the k threads
//   whose maxima are the k largest under the same order (value, then index): a bound from 64 maxima of
//   neighbouring threads leaves few threads, and the entries of the chosen ones, a few hundred bytes
//   each, are read again (where the bound leaves many, after the index of their largest entry has
//   left k of them). Candidates are ranked one against all the others; of more than 256 (equal or nearly
//   equal entries, a row held down by a finite mask) only those of k threads are. 5 rows of 51866 f32
//   entries, 10 alternatives: random ones 9.0 us, equal ones 13.5, all but 1501 held down 11.8 (820 both,
//   ranked whole); 600 rows of 4096, 32 alternatives 8.1 and 18.9 (1492). One row of 262144, 32
//   alternatives, whose chunks' best ones are more than 256: 15 us, ranked whole 118.
//   s is kept without the largest entry's 1 (its thread's entries are summed again, a piece a thread),
//   and ln s = log1p of it: a token of probability 1 - 1e-7 has its log probability to 2^-22 too.
//   Few rows split over several workgroups, which merge through memory (the last to count in joins
//   the parts in order; sums and order do not depend on which it is). Chunks of at most kScoreSmall
//   entries stay in registers.
//   Bound: many rows by what a wave issues for an entry (exponent, sum, entropy: 4 instructions and a
//   half, one of them v_exp_f32) next to the bytes: 7168 rows of 51865 f16 (744 MB) 158 us, 4.7 TB/s,
//   f32 rows of the same bytes 132 us, 5.6; prefetch of 2 or 3 groups is no faster (163 and 171 us).
//   Rows of less than a workgroup a CU by latency: of the 8.9 us of 5 masked rows of 51866 f32 (13 chunks
//   of 5 rows), 0.5 are the logits, 3.5 bound, candidates and their order, 2.3 the parts' way through
//   memory, 1.9 the merge's candidates and 0.9 the results.
#include "wrs_internal.hpp"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace wrs {
namespace {

typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32u __attribute__((aligned(1)));

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kGroup = 16;  // entries of a thread's group: 16-byte pieces, kThreads pieces apart
constexpr int kSmallGroup = kScoreSmall / kThreads;  // entries of a thread of a small chunk
static_assert(kScoreSmall <= kScoreMostTop * (kScoreChunk / kThreads), "room for every one's key");
constexpr int kRun = kThreads / 64;  // neighbouring threads that share a maximum of the bound
static_assert(kRun == 8, "max8");
constexpr int kMostPieces = kScoreChunk / kThreads / 4;  // of a thread, at most (f32: 4 entries)
static_assert(kMostPieces <= 64, "a piece a lane");
constexpr int kMostKeys = kScoreMostTop * (kScoreChunk / kThreads);  // entries of that many threads
constexpr int kMostRanked = 256;  // keys that are ranked one against all the others, at most
constexpr int kCounterStride = 32;   // 128 bytes between merge counters
// Exponents below it are 0: finite, so that times a weight of 0 it is 0. References lie at or above it,
// and below -kLow where the sums against them are used.
constexpr float kLow = -0x1p24f;

// A value's order as an unsigned number, and an entry's: by value, the lower index first among
// equals.
__device__ inline uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // one zero
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ inline float value_of(uint32_t o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ inline uint64_t key_of(float x, uint32_t index) {
  return static_cast<uint64_t>(order_of(x)) << 32 | (0xFFFFFFFFu - index);
}
__device__ inline float value_of(uint64_t key) { return value_of(static_cast<uint32_t>(key >> 32)); }
__device__ inline int index_of(uint64_t key) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

// A 16-byte piece of entries. T: float, _Float16 or uint16_t (bf16).
template <typename T>
struct Piece {
  static constexpr int kN = 16 / sizeof(T);
  u32x4 w;
  __device__ inline float operator[](int e) const {
    const uint32_t x = w[sizeof(T) == 4 ? e : e >> 1];
    if constexpr (sizeof(T) == 4)
      return __builtin_bit_cast(float, x);
    else if constexpr (__is_same(T, uint16_t))
      return __builtin_bit_cast(float, e & 1 ? x & 0xFFFF0000u : x << 16);
    else
      return static_cast<float>(
          __builtin_bit_cast(_Float16, static_cast<uint16_t>(e & 1 ? x >> 16 : x)));
  }
};
template <typename T>
__device__ inline float value(T x) {
  if constexpr (__is_same(T, uint16_t))
    return __builtin_bit_cast(float, static_cast<uint32_t>(x) << 16);
  else
    return static_cast<float>(x);
}

// A row's (or chunk's) entries: x[0 .. n), entry i allowed where ok[i] is not zero.
template <typename T, bool kMask>
struct Row {
  const T* x;
  const uint8_t* ok;
  int n;
  static constexpr int kN = Piece<T>::kN;
  // Piece p, entries kN p.. : hidden ones and those past the end come as -infinity. The row's last
  // piece is read from its last kN entries on, so that nothing lies outside the row; returns the
  // index of v[0].
  __device__ inline int load(int p, float (&v)[kN]) const {
    const int i0 = p * kN, at = min(i0, n - kN);
    if (n < kN) {  // rows shorter than a piece
#pragma unroll
      for (int e = 0; e < kN; ++e)
        v[e] = i0 + e < n && (!kMask || ok[i0 + e]) ? value(x[i0 + e]) : -INFINITY;
      return i0;
    }
    Raw r;
    fetch(at, r);
    values(r, v);
#pragma unroll
    for (int e = 0; e < kN; ++e)
      if (at + e < i0) v[e] = -INFINITY;
    return at;
  }
  // A piece that lies within the row, from entry `at` on, in two steps.
  struct Raw {
    Piece<T> x;
    uint32_t ok[kMask ? kN / 4 : 1];
  };
  __device__ inline void fetch(int at, Raw& r) const {
    r.x.w = *reinterpret_cast<const u32x4u*>(x + at);
    if constexpr (kMask) {
#pragma unroll
      for (int h = 0; h < kN / 4; ++h) r.ok[h] = *reinterpret_cast<const u32u*>(ok + at + 4 * h);
    }
  }
  static __device__ inline void values(const Raw& r, float (&v)[kN]) {
#pragma unroll
    for (int e = 0; e < kN; ++e) v[e] = r.x[e];
    if constexpr (kMask) {
#pragma unroll
      for (int e = 0; e < kN; ++e)
        if (!(r.ok[e / 4] & (0xFFu << (8 * (e & 3))))) v[e] = -INFINITY;
    }
  }
};

// The largest of the 16 f16 entries of two pieces, two at a time (widened first: 16 conversions).
template <typename R>
__device__ inline float max_of_halves(const R (&r)[2]) {
  uint32_t m = r[0].x.w[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    const uint32_t w = r[i >> 2].x.w[i & 3];
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(m) : "v"(m), "v"(w));
  }
  return fmaxf(static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(m))),
               static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(m >> 16))));
}

template <int kCtrl>
__device__ inline float dpp(float x) {
  const int i = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, kCtrl, 0xF, 0xF, false));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kRor8 = 0x128;  // lanes of 16
__device__ inline float max8(float x) {  // of 8 neighbouring lanes
  x = fmaxf(x, dpp<kXor1>(x));
  x = fmaxf(x, dpp<kXor2>(x));
  return fmaxf(x, dpp<kHalfMirror>(x));
}
__device__ inline float wave_max(float x) {
  x = max8(x);
  return max_x16_x32(fmaxf(x, dpp<kRor8>(x)));
}
__device__ inline float wave_sum(float x) {
  x += dpp<kXor1>(x);
  x += dpp<kXor2>(x);
  x += dpp<kHalfMirror>(x);
  return sum_x16_x32(x + dpp<kRor8>(x));
}
// The sum over 8 neighbouring lanes.
__device__ inline int sum8(int x) {
  x += __builtin_amdgcn_update_dpp(x, x, kXor1, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(x, x, kXor2, 0xF, 0xF, false);
  return x + __builtin_amdgcn_update_dpp(x, x, kHalfMirror, 0xF, 0xF, false);
}
// Calls f(rank, key) for each of n keys, 8 lanes to a key, with how many keys are larger; in one lane
// of the 8. The array goes on for 31 more.
template <typename F>
__device__ inline void rank_all(const uint64_t* keys, int n, F f) {
  const int part = threadIdx.x & 7;
  for (int q = threadIdx.x >> 3; q - static_cast<int>(threadIdx.x >> 3) < n; q += kThreads / 8) {
    const uint64_t mine = keys[min(q, n - 1)];
    int r = 0;
    for (int i = part; i < n; i += 32) {
#pragma unroll
      for (int j = 0; j < 32; j += 8) r += keys[i + j] > mine && i + j < n;
    }
    r = sum8(r);
    if (part == 0 && q < n) f(r, mine);
  }
}
// Puts the kCount keys of each lane that `in` names behind those in the list.
template <int kCount>
__device__ inline void append(const uint64_t (&key)[kCount], const bool (&in)[kCount], uint64_t* list,
                              int* n) {
  uint64_t who[kCount];
  int all = 0;
#pragma unroll
  for (int e = 0; e < kCount; ++e) {
    who[e] = __ballot(in[e]);
    all += __popcll(who[e]);
  }
  if (all == 0) return;  // the whole wave
  int at = 0;
  if ((threadIdx.x & 63) == 0) at = atomicAdd(n, all);
  at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
  for (int e = 0; e < kCount; ++e) {
    const int before = __builtin_amdgcn_mbcnt_hi(
        static_cast<uint32_t>(who[e] >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who[e]), 0));
    if (in[e]) list[at + before] = key[e];
    at += __popcll(who[e]);
  }
}

struct Shared {
  uint64_t keys[kMostKeys + 32];  // candidates
  uint64_t best[kScoreMostTop], bound_key;
  uint32_t least;
  uint32_t run_max[64];  // in order_of's numbers, the low bits a number of the run's own
  float wave_max[kWaves];
  float sums[2][kWaves];
  float piece[2][kMostPieces];  // sums of the pieces of the thread that holds the largest entry
  float bound;
  int chosen[kThreads];    // threads whose entries are read again (-1 - thread: holds the largest)
  int equals[kMostPieces];  // entries of those pieces that equal it
  int tops[kWaves];
  int n_first, n_chosen, n_keys, last;
};

// The k-th best of the threads' keys (0: none), 0 if there are fewer. Takes the room of the candidates
// and leaves none of them. Keys lie in the k runs of 8 threads whose best ones are the k best, so that
// 8 k of them are ranked, however many there are.
static_assert(kScoreMostTop * kRun <= kMostRanked, "runs of k");
__device__ inline uint64_t kth_best(uint64_t mine, int k, Shared& sh) {
  const int tid = threadIdx.x;
  unsigned long long run = mine;
#pragma unroll
  for (int x = 1; x < kRun; x <<= 1) run = max(run, __shfl_xor(run, x));
  __syncthreads();  // what was listed is read
  if (tid % kRun == 0) sh.keys[tid / kRun] = run;
  if (tid == 0) {
    sh.bound_key = 0;
    sh.n_keys = sh.n_first = 0;
  }
  __syncthreads();
  int r = 0;
#pragma unroll
  for (int i = 0; i < kRun; ++i) r += sh.keys[kRun * (tid % kRun) + i] > run;
  r = sum8(r);
  if (tid % kRun == 0 && r == k - 1) sh.bound_key = run;
  __syncthreads();
  uint64_t* const list = sh.keys + kThreads / kRun;
  const uint64_t key[1] = {mine};
  const bool in[1] = {mine != 0 && mine >= sh.bound_key};
  append(key, in, list, &sh.n_first);
  __syncthreads();
  const int n = sh.n_first;
  rank_all(list, n, [&](int r, uint64_t key) __attribute__((always_inline)) {
    if (r == k - 1) sh.best[r] = key;
  });
  __syncthreads();
  return n < k ? 0 : sh.best[k - 1];
}
// Leaves the candidates that may be among the k best: those of k threads, 8 each.
__device__ inline void cut(int k, Shared& sh) {
  constexpr int kMine = kMostKeys / kThreads;
  static_assert(kMine * kScoreMostTop <= kMostRanked, "keys that are left");
  const int n = sh.n_keys;
  uint64_t key[kMine], mine = 0;
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    const int i = threadIdx.x + kThreads * j;
    key[j] = i < n ? sh.keys[i] : 0;
    mine = key[j] > mine ? key[j] : mine;
  }
  const uint64_t least = kth_best(mine, k, sh);
  bool in[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) in[j] = key[j] != 0 && key[j] >= least;
  append(key, in, sh.keys, &sh.n_keys);
  __syncthreads();
}

// One chunk: its largest entry m, the sums of the others (s = sum 2^z, t = sum z 2^z with z = scale (x
// - m)) and its k best entries in sh.best, keys of entries that are not there 0. Every thread gets
// m, s and t.
//
// Sums are kept against a reference r of the thread's, its maximum times scale as f32 rounds it, so that
// a term's exponent is one fma (rounded once, whatever r is); what r is off by, half a unit of f32 at
// 2^24 at most, is taken back at the end. Farther out it is off by more than a sum's range takes (2^9
// at 2^33), so a thread whose entries all lie below -2^24 adds 0 against that, and where the largest
// entry of all lies outside `plain` takes a second pass over differences.
// early() is called while few other loads are on their way.
template <typename T, bool kMask, bool kSmall, typename F>
__device__ inline void scan(const Row<T, kMask>& row, int index0, int k, float scale, Shared& sh,
                            F early, float& m_out, float& s_out, float& t_out) {
  constexpr int kN = Piece<T>::kN, kTurns = (kSmall ? kSmallGroup : kGroup) / kN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int pieces = (row.n + kN - 1) / kN;
  float m = -INFINITY, s = 0.f, t = 0.f, ref = kLow;
  int at = 0;  // the group that held m first
  float v[kTurns][kN];
  // Entries of the group g, `top` the largest. kClean: -infinity is unlikely among them.
  auto take = [&](int g, const auto& x, float top, auto kClean) __attribute__((always_inline)) {
    constexpr int kPieces = sizeof(x) / sizeof(x[0]);
    if (top > m) at = g;
    m = fmaxf(m, top);
    const float r = fmaxf(m * scale, kLow), d = ref - r, w0 = __builtin_amdgcn_exp2f(d);
    ref = r;
    t = w0 * __builtin_fmaf(d, s, t);
    s *= w0;
    const float t0 = t;
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const float z = __builtin_fmaf(x[u][e], scale, -r), w = __builtin_amdgcn_exp2f(z);
        s += w;
        t = __builtin_fmaf(kClean.value ? z : fmaxf(z, kLow), w, t);
      }
    if (kClean.value && __any(t != t)) {
      // An entry of -infinity, whose weight of 0 times its exponent is no number: again without.
      t = t0;
#pragma unroll
      for (int u = 0; u < kPieces; ++u)
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float z = __builtin_fmaf(x[u][e], scale, -r);
          t = __builtin_fmaf(fmaxf(z, kLow), __builtin_amdgcn_exp2f(z), t);
        }
    }
  };
  const int groups = kSmall ? 1 : (pieces + kTurns * kThreads - 1) / (kTurns * kThreads);
  const int whole = row.n / (kN * kTurns * kThreads);  // groups with every entry in the row
  int index[kTurns] = {};  // of v[u][0], in a small chunk
  if constexpr (!kSmall) {
    if (whole > 0) {
      typename Row<T, kMask>::Raw raw[kTurns];
      auto fetch = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kTurns; ++u)
          row.fetch(((g * kTurns + u) * kThreads + tid) * kN, raw[u]);
      };
      fetch(0);
      for (int g = 0; g < whole; ++g) {
#pragma unroll
        for (int u = 0; u < kTurns; ++u) row.values(raw[u], v[u]);
        float top = v[0][0];
        if constexpr (__is_same(T, _Float16) && !kMask) {
          top = max_of_halves(raw);
        } else {
#pragma unroll
          for (int u = 0; u < kTurns; ++u)
#pragma unroll
            for (int e = 0; e < kN; ++e) top = fmaxf(top, v[u][e]);
        }
        if (g + 1 < whole) fetch(g + 1);
        take(g, v, top, std::integral_constant<bool, !kMask>{});
      }
    }
  }
  if constexpr (kSmall) {
#pragma unroll
    for (int u = 0; u < kTurns; ++u) index[u] = row.load(u * kThreads + tid, v[u]);
    float top = v[0][0];
#pragma unroll
    for (int u = 0; u < kTurns; ++u)
#pragma unroll
      for (int e = 0; e < kN; ++e) top = fmaxf(top, v[u][e]);
    take(0, v, top, std::false_type{});
  } else if (whole < groups) {
    for (int q = whole * kTurns; q * kThreads + 64 * wave < pieces; ++q) {
      float x[1][kN];
      row.load(q * kThreads + tid, x[0]);
      float top = x[0][0];
#pragma unroll
      for (int e = 0; e < kN; ++e) top = fmaxf(top, x[0][e]);
      take(whole, x, top, std::false_type{});
    }
  }

  // A bound at or below the k-th largest thread's maximum: that of 64 runs of threads.
  // The 64 are told apart by their low bits; the bound has none of them, so it lies at or below.
  const uint32_t run = (order_of(max8(m)) & ~63u) | (63u - (tid / kRun));
  if (tid % kRun == 0) sh.run_max[tid / kRun] = run;
  const float wave_top = wave_max(m);
  if (lane == 0) sh.wave_max[wave] = wave_top;
  if (tid == 0) sh.n_first = sh.n_chosen = sh.n_keys = 0;
  early();
  __syncthreads();
  {
    int r = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) r += sh.run_max[kRun * (tid % kRun) + i] > run;
    r = sum8(r);
    // Cut down, -infinity is a NaN.
    if (tid % kRun == 0 && r == k - 1) sh.bound = fmaxf(value_of(run & ~63u), -INFINITY);
  }
  float m_all = sh.wave_max[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m_all = fmaxf(m_all, sh.wave_max[w]);
  const bool odd = !(m_all * scale > kLow && m_all * scale < -kLow);  // the same in all threads
  if (odd && m_all > -INFINITY) {
    // plain: the sums against the largest entry, from differences.
    s = t = ref = 0.f;
    for (int g = 0; g < groups; ++g)
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        float x[kN];
        row.load((g * kTurns + u) * kThreads + tid, x);
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float z = (x[e] - m_all) * scale, w = __builtin_amdgcn_exp2f(z);
          s += w;
          t = __builtin_fmaf(fmaxf(z, kLow), w, t);
        }
      }
  }
  const bool is_top = m > -INFINITY && m == m_all;
  // A piece's terms without the entries that equal the largest, which are counted.
  auto others = [&](const float (&x)[kN], float& a, float& b, int& n) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const float z = (x[e] - m_all) * scale, w = __builtin_amdgcn_exp2f(z);
      n += x[e] == m_all;
      a += x[e] == m_all ? 0.f : w;
      b = __builtin_fmaf(fmaxf(z, kLow), w, b);
    }
  };
  // A thread's sums s and t, against m_all.
  auto joined = [&](float& a, float& b) __attribute__((always_inline)) {
    const float r_all = odd ? 0.f : m_all * scale;
    // scale m_all - r_all, which the sums lie too high by
    const float off = odd ? 0.f : __builtin_fmaf(m_all, scale, -r_all);
    const float d = fmaxf(ref - r_all - off, kLow), w0 = __builtin_amdgcn_exp2f(d);
    a = w0 * s;
    b = w0 * __builtin_fmaf(d, s, t);
  };
  auto add_up = [&](float a, float b) __attribute__((always_inline)) {
    const float ws = wave_sum(a), wt = wave_sum(b);
    if (lane == 0) {
      sh.sums[0][wave] = ws;
      sh.sums[1][wave] = wt;
    }
  };
  int n_top = 0;
  const int per = groups * kTurns;  // pieces of a thread
  if constexpr (kSmall) {
    // Threads that hold the largest entry leave out all that equal it, and count them.
    float a, b;
    int equal = 0;
    joined(a, b);
    if (is_top) {
      a = b = 0.f;
#pragma unroll
      for (int u = 0; u < kTurns; ++u) others(v[u], a, b, equal);
    }
    add_up(a, b);
    int of_wave = 0;
    if (__any(is_top)) of_wave = static_cast<int>(wave_sum(static_cast<float>(equal)));
    if (lane == 0) sh.tops[wave] = of_wave;
    __syncthreads();
    const float bound = sh.bound;
    uint64_t key[kTurns * kN];
    bool with[kTurns * kN];
#pragma unroll
    for (int u = 0; u < kTurns; ++u)
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        key[u * kN + e] = key_of(v[u][e], index0 + index[u] + e);
        with[u * kN + e] = v[u][e] > -INFINITY && v[u][e] >= bound;
      }
    append(key, with, sh.keys, &sh.n_keys);
  } else {
    const int of_wave = __popcll(__ballot(is_top));
    if (lane == 0) sh.tops[wave] = of_wave;
    __syncthreads();
    const float bound = sh.bound;
    const bool in = m > -INFINITY && m >= bound;
    if (in) sh.chosen[atomicAdd(&sh.n_chosen, 1)] = is_top ? -1 - tid : tid;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) n_top += sh.tops[w];
    // Entries at or above the bound, whatever their index..
    uint64_t least = key_of(bound == -INFINITY ? -FLT_MAX : bound, 0xFFFFFFFFu);
    int n_chosen = sh.n_chosen;
    if (n_chosen * per * kN > kMostKeys) {
      // .. or, where that could be too many, those of the k threads whose first largest entries are the
      // k best.
      uint64_t mine = 0;
      if (in) {
        int first = 0;
#pragma unroll
        for (int u = kTurns - 1; u >= 0; --u) {
          float x[kN];
          const int i0 = row.load((at * kTurns + u) * kThreads + tid, x);
#pragma unroll
          for (int e = kN - 1; e >= 0; --e)
            if (x[e] == m) first = i0 + e;
        }
        mine = key_of(m, index0 + first);
      }
      least = kth_best(mine, k, sh);
      if (tid == 0) sh.n_chosen = 0;
      __syncthreads();
      if (in && mine >= least) sh.chosen[atomicAdd(&sh.n_chosen, 1)] = is_top ? -1 - tid : tid;
      __syncthreads();
      n_chosen = sh.n_chosen;
    }
    // The chosen threads' entries again, a piece a thread.
    for (int i = tid; i < n_chosen * per; i += kThreads) {
      const int j = i / per, q = i - j * per;
      const int who = sh.chosen[j];
      float x[kN];
      const int i0 = row.load(q * kThreads + (who < 0 ? -1 - who : who), x);
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const uint64_t key = key_of(x[e], index0 + i0 + e);
        if (x[e] > -INFINITY && key >= least) sh.keys[atomicAdd(&sh.n_keys, 1)] = key;
      }
      if (who < 0 && n_top == 1) {
        float a = 0.f, b = 0.f;
        int equal = 0;
        others(x, a, b, equal);
        sh.piece[0][q] = a;
        sh.piece[1][q] = b;
        sh.equals[q] = equal;
      }
    }
    // The threads' sums, without the one that alone holds the largest entry, whose pieces follow.
    float a, b;
    joined(a, b);
    const bool apart = is_top && n_top == 1;
    add_up(apart ? 0.f : a, apart ? 0.f : b);
  }
  __syncthreads();
  if (sh.n_keys > kMostRanked) cut(k, sh);
  const int n_keys = sh.n_keys;
  if (tid < k && tid >= n_keys) sh.best[tid] = 0;
  rank_all(sh.keys, n_keys, [&](int r, uint64_t key) __attribute__((always_inline)) {
    if (r < k) sh.best[r] = key;
  });
  s = t = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    s += sh.sums[0][w];
    t += sh.sums[1][w];
  }
  if constexpr (kSmall) {
    int equal = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) equal += sh.tops[w];
    s += static_cast<float>(max(equal - 1, 0));
  } else if (n_top == 1) {
    const bool mine_too = lane < per;
    s += wave_sum(mine_too ? sh.piece[0][lane] : 0.f) +
         (wave_sum(mine_too ? static_cast<float>(sh.equals[lane]) : 0.f) - 1.f);
    t += wave_sum(mine_too ? sh.piece[1][lane] : 0.f);
  } else if (n_top > 1) {
    s -= 1.f;
  }
  __syncthreads();
  m_out = m_all;
  s_out = s;
  t_out = t;
}

template <typename T, bool kMask, bool kSmall>
__global__ __launch_bounds__(kThreads, 8) void score_rows(ScoreArgs a) {
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
  float given = 0.f;  // the token's logit
  uint8_t given_ok = 1;
  scan<T, kMask, kSmall>(row, i0, k, a.scale_log2, sh, [&]() __attribute__((always_inline)) {
    if (tid == 0 && a.logprobs) {
      const int at = min(max(token, 0), a.n_vocab - 1);
      given = value(x[at]);
      if (kMask) given_ok = ok[at];
    }
  }, m, s, t);
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
    // A chunk a lane: their sums, and the best entries j = wave, wave + 8, .. of each.
    const int c = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    float mc = -INFINITY, sc = 0.f, tc = 0.f;
    if (c < a.n_chunks) {
      const float* const p = all + c * kScorePart;
      mc = ld_agent(p);
      sc = ld_agent(p + 1);
      tc = ld_agent(p + 2);
    }
    constexpr int kMine = (kScoreMostTop + kWaves - 1) / kWaves;
    uint64_t mine[kMine] = {};
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      const int j = wave + kWaves * q;
      if (j < k && c < a.n_chunks)
        mine[q] = __hip_atomic_load(reinterpret_cast<const uint64_t*>(all + c * kScorePart + 4) + j,
                                    __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (tid == 0) sh.n_keys = sh.least = 0;
    if (tid < k) sh.best[tid] = 0;
    __syncthreads();
    // The k best are at or above the largest of the chunks' k-th ones.
#pragma unroll
    for (int q = 0; q < kMine; ++q)
      if (wave + kWaves * q == k - 1 && mine[q])
        atomicMax(&sh.least, static_cast<uint32_t>(mine[q] >> 32));
    __syncthreads();
    const uint32_t least = sh.least;
    bool with[kMine];
#pragma unroll
    for (int q = 0; q < kMine; ++q)
      with[q] = mine[q] && static_cast<uint32_t>(mine[q] >> 32) >= least;
    append(mine, with, sh.keys, &sh.n_keys);
    __syncthreads();
    if (sh.n_keys > kMostRanked) cut(k, sh);
    const int n_keys = sh.n_keys;
    rank_all(sh.keys, n_keys, [&](int p, uint64_t key) __attribute__((always_inline)) {
      if (p < k) sh.best[p] = key;
    });
    __syncthreads();
    // The chunk that holds the largest entry leaves its 1 out.
    const int home = sh.best[0] ? index_of(sh.best[0]) / a.chunk : -1;
    if (c != home && mc > -INFINITY) sc += 1.f;
    m = wave_max(mc);
    const float d = fmaxf((fmaxf(mc, -FLT_MAX) - fmaxf(m, -FLT_MAX)) * a.scale_log2, kLow);
    const float w = __builtin_amdgcn_exp2f(d);
    s = wave_sum(w * sc);
    t = wave_sum(w * __builtin_fmaf(d, sc, tc));
    if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // A row with an allowed NaN or +infinity has no distribution; one without an entry gives none
  // of its tokens.
  const bool odd = s != s || m == INFINITY, none = !odd && m == -INFINITY;
  if (tid >= 128) return;  // two waves write
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
    const bool is_entry = token >= 0 && token < a.n_vocab && given_ok != 0;
    a.logprobs[r] = logprob(is_entry ? given : -INFINITY);
  }
  if (tid == 64 && a.entropy)
    a.entropy[r] = odd ? NAN : none ? 0.f : ln_s - t * 0.6931471805599453f / (1.f + s);
}

}  // namespace

void score_plan(ScoreArgs& a, bool split) {
  // A workgroup a CU and no more: f32 rows of 51865 entries, a workgroup a row, up to 256 and up to
  // 520 workgroups: 16 rows 9.0, 8.1, 8.2 us, 40 rows 9.8, 9.4, 11.1 us, 130 rows 11.2, 11.2, 15.9 us. With
  // one, two and three workgroups a row 86 rows take 8.5, 9.5 and 10.2 us, 130 9.0, 11.7 and 11.0, 200 10.9,
  // 14.0 and 15.7 (with a mask each 10.5, 10.9, 11.7; 10.9, 14.3, 12.8; 13.0, 17.0, 18.0).
  int64_t chunks = 1;
  if (split) chunks = std::max<int64_t>(1, kScoreMaxWgs / std::max<int64_t>(a.n_rows, 1));
  chunks = std::min<int64_t>(chunks, (a.n_vocab + kScoreSmall - 1) / kScoreSmall);
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
  const bool small = a.chunk <= kScoreSmall;
#define WRS_SCORE_ONE(T, M, S) hipLaunchKernelGGL((score_rows<T, M, S>), grid, dim3(kThreads), 0, s, a)
#define WRS_SCORE(T)                                                      \
  if (a.allowed) {                                                        \
    if (small) { WRS_SCORE_ONE(T, true, true); } else { WRS_SCORE_ONE(T, true, false); }   \
  } else {                                                                \
    if (small) { WRS_SCORE_ONE(T, false, true); } else { WRS_SCORE_ONE(T, false, false); } \
  }
  switch (dt) {
    case kF32: WRS_SCORE(float); break;
    case kF16: WRS_SCORE(_Float16); break;
    case kBF16: WRS_SCORE(uint16_t); break;
    default: return hipErrorInvalidValue;
  }
#undef WRS_SCORE
#undef WRS_SCORE_ONE
  return hipGetLastError();
}

}  // namespace wrs
