// qlin_token_logprobs: log probabilities of given tokens, the entropy and the top alternatives of rows of logits, and the gradient.
//
//   m = max x,  S = sum exp(x - m),  T = sum exp(x - m) (x - m):   log p(t) = (x_t - m) - log S,   H = log S - T / S
//   dx_j = dl ([j = t] - p_j) - dh p_j (log p_j + H)
//
// What bounds it: HBM, the logits once (the gradient: once more, and its own bytes).  A thread keeps its own m, S and T over pieces of
// eight 16-byte loads and moves m once a piece at most; they are joined in the block and, where rows are few, in a cluster of blocks that share
// a row.  An element costs one exponential and four or five other operations, which 16-bit logits just leave time for.
//
// The top alternatives come out of the same pass.  The k-th largest of the maxima of the block's 64 groups of threads is at most the k-th largest element, and for
// elements in no special order nearly as large (k = 20: 24 elements expected above it); each piece's maximum stays in shared
// memory, so only the few pieces that reach that threshold are listed and read again, from L2, by whole warps.  What they hold above it is ordered by counting for
// each element how many are larger.  Elements are ordered by value, then by the lower id, so results do not depend on timing.
//
// Measured (device time, bf16): 4096 x 128256 165 us, 6.4 TB/s, 0.97 of the copy rate, with the exponentials' unit busy for 77 % of it; 2048 x 128256 forward and backward 261 us,
// 6.0 TB/s (188 and 276 a call in a long run, whose clock falls); 64 x 128256 with 20 alternatives 11 us and one row with five 8 us (12 a call, on the host), which are the latency of the row, its sums, the pieces and the cluster behind one another; 333 x 50257 in
// fp32 with all but nine logits minus infinity 21 us (18 where L2 holds them).  Tried and no faster, 4096 x 128256: every fourth or eighth pair of exponentials by a polynomial on the FMA pipe 179 and 167 us (the
// instructions are what there is no room for), pieces without the guard for minus infinity, which are done again where they held one, 170.
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qlin_internal.h"
#include "qlin_ptx.cuh"

namespace qlin {

constexpr int kScoreThreads = 256;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kPieceLoads = 8;       // 16-byte loads of a piece
constexpr int kMostTop = 32;
constexpr int kMostParts = 8;        // blocks that share a row
constexpr int kCandidates = 1024;
constexpr int kHits = 512;
constexpr int kMostVocab = 1 << 20;
constexpr float kLog2e = 1.4426950408889634f;

struct ScoreParams {
  qlin_token_logprobs_args a;
  int32_t parts;   // blocks of a row, a cluster
  int32_t pieces;  // of a thread at most
};

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (std::is_same<T, float>::value) return v;
  if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(v);
}
template <typename T>
__device__ __forceinline__ float2 word_pair(uint32_t w) {  // the two 16-bit elements of a word
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint4 packed(const float (&e)[16 / sizeof(T)]) {  // 16 bytes of the type, rounded to nearest
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (std::is_same<T, float>::value) {
      w[j] = __float_as_uint(e[j]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(e[2 * j], e[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(e[2 * j], e[2 * j + 1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// The larger of two, NaN if one is NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t max_words(uint32_t a, uint32_t b) {
  if constexpr (std::is_same<T, float>::value) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  } else {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t lowest_word() {  // minus infinity, twice in 16 bits
  return std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
}
__device__ __forceinline__ float exp2_ftz(float x) {  // 2 ulp; below 2^-126 zero
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A number whose unsigned order is that of the values: NaN above all, both zeros the same.  0 stands for no element.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order); }
// Value first, then the lower id.
__device__ __forceinline__ uint64_t ranked(uint32_t order, uint32_t id) { return static_cast<uint64_t>(order) << 32 | (0xffffffffu - id); }

// Sums of exp(x - ref) and exp(x - ref) (x - ref) where ref is the maximum, or 0 where that is minus infinity.
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ Sums moved(Sums v, float m) {  // the same sums about a maximum m >= v.m
  const float d = reference(v.m) - reference(m);
  const float f = exp2_ftz(d * kLog2e);
  // a sum of nothing stays one: d may be infinite
  return v.s == 0.0f ? Sums{m, 0.0f, 0.0f} : Sums{m, v.s * f, f == 0.0f ? 0.0f : f * fmaf(d, v.s, v.t)};
}
__device__ __forceinline__ Sums joined(Sums a, Sums b) {
  const float m = max_nan(a.m, b.m);
  a = moved(a, m);
  b = moved(b, m);
  return Sums{m, a.s + b.s, a.t + b.t};
}

// How a row lies in memory: elements before the first 16-byte boundary, whole pieces of 16 bytes, elements behind them.
template <typename T>
struct Row {
  static constexpr int PER = 16 / sizeof(T);
  const T* x;
  int vocab, head, vectors, tail;
  __device__ __forceinline__ Row(const T* row, int n) : x(row), vocab(n) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T));
    head = min((PER - off) & (PER - 1), n);
    vectors = (n - head) / PER;
    tail = n - head - vectors * PER;
  }
  __device__ __forceinline__ uint4 vector(int i) const { return __ldg(reinterpret_cast<const uint4*>(x + head) + i); }
  __device__ __forceinline__ int id(int i) const { return head + i * PER; }  // of a vector's first element
  __device__ __forceinline__ int edge_id(int e) const { return e < head ? e : vocab - tail + (e - head); }
};

template <typename T>
__device__ __forceinline__ void orders_of(const uint4& v, uint32_t (&o)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      o[i] = order_of(__uint_as_float(w[i]));
    } else {
      const float2 f = word_pair<T>(w[i]);
      o[2 * i] = order_of(f.x);
      o[2 * i + 1] = order_of(f.y);
    }
  }
}

// Shared memory of a block: what the threads and pieces found, and the elements that may be among the top ones.
constexpr int kGroups = kScoreThreads / 4;
struct ScoreShared {
  Sums warp[kScoreWarps], block;
  uint4 best[kGroups / 4];  // of four threads each
  uint64_t candidate[kCandidates];
  uint64_t chosen[kMostTop];
  uint32_t hit[kHits];  // pieces that are looked at again: piece * threads + thread
  uint32_t threshold;
  int found, hits, scan[kScoreWarps];
};

// Elements of this block's share from `least` on, as many as there are places for; returns how many there are.  The pieces that reach it are listed first and
// then read by whole warps, a word a lane; -1, and nothing read, where they are too many to list.
template <typename T>
__device__ __forceinline__ int gather(const Row<T>& row, ScoreShared& sh, const uint32_t* piece_best, int pieces, int first, int last, int edges, uint32_t least) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __syncthreads();
  if (tid == 0) sh.found = sh.hits = 0;
  __syncthreads();
  for (int p = 0; p < pieces; ++p)
    if (piece_best[p * kScoreThreads + tid] >= least) {
      const int at = atomicAdd(&sh.hits, 1);
      if (at < kHits) sh.hit[at] = static_cast<uint32_t>(p * kScoreThreads + tid);
    }
  const auto offer = [&](uint32_t order, int id) {
    if (order < least) return;
    const int at = atomicAdd(&sh.found, 1);
    if (at < kCandidates) sh.candidate[at] = ranked(order, static_cast<uint32_t>(id));
  };
  if (tid < edges) offer(order_of(to_float(row.x[row.edge_id(tid)])), row.edge_id(tid));
  __syncthreads();
  const int hits = sh.hits;
  if (hits > kHits) return -1;
  constexpr int AHEAD = 4;
  for (int h0 = warp * AHEAD; h0 < hits; h0 += kScoreWarps * AHEAD) {
    uint32_t word[AHEAD];
    int id[AHEAD];
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {  // lane: load lane / 4 of the piece, word lane % 4 of it
      const uint32_t hit = h0 + e < hits ? sh.hit[h0 + e] : 0u;
      const int i = first + (static_cast<int>(hit / kScoreThreads) * kPieceLoads + (lane >> 2)) * kScoreThreads + static_cast<int>(hit % kScoreThreads);
      id[e] = h0 + e < hits && i < last ? row.id(i) + (lane & 3) * static_cast<int>(4 / sizeof(T)) : -1;
      word[e] = id[e] >= 0 ? __ldg(reinterpret_cast<const uint32_t*>(row.x + id[e])) : 0u;
    }
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      if (id[e] < 0) continue;
      if constexpr (std::is_same<T, float>::value) {
        offer(order_of(__uint_as_float(word[e])), id[e]);
      } else {
        const float2 f = word_pair<T>(word[e]);
        offer(order_of(f.x), id[e]);
        offer(order_of(f.y), id[e] + 1);
      }
    }
  }
  __syncthreads();
  return sh.found;
}
// After a call of gather that found too much: a value that at least `want` elements reach, from the listed pieces' maxima (n < 0) or the elements that found a
// place.  The least of these at first, which is the answer for rows of few values; then the `want`-th largest.
__device__ __forceinline__ uint32_t raised(ScoreShared& sh, const uint32_t* piece_best, int n, int want, bool again) {
  const int tid = threadIdx.x, all = n < 0 ? kHits : kCandidates;
  const auto value = [&](int i) { return n < 0 ? piece_best[sh.hit[i]] : static_cast<uint32_t>(sh.candidate[i] >> 32); };
  __syncthreads();
  if (!again) {
    uint32_t low = 0xffffffffu;
    for (int i = tid; i < all; i += kScoreThreads) low = min(low, value(i));
    low = __reduce_min_sync(0xffffffffu, low);
    if ((tid & 31) == 0) sh.scan[tid >> 5] = static_cast<int>(low);
    __syncthreads();
    for (int w = 0; w < kScoreWarps; ++w) low = min(low, static_cast<uint32_t>(sh.scan[w]));
    return low;
  }
  for (int i = tid; i < all; i += kScoreThreads) {
    const uint32_t mine = value(i);
    int above = 0;
    for (int j = 0; j < all; ++j) above += value(j) > mine || (value(j) == mine && j < i) ? 1 : 0;
    if (above == want - 1) sh.threshold = mine;
  }
  __syncthreads();
  return sh.threshold;
}
// The `want` first of n candidates, in order, to `to`; returns how many there are.
__device__ __forceinline__ int rank_candidates(ScoreShared& sh, int n, int want, uint64_t* to) {
  for (int i = threadIdx.x; i < n; i += kScoreThreads) {
    const uint64_t mine = sh.candidate[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += sh.candidate[j] > mine ? 1 : 0;
    if (above < want) to[above] = mine;
  }
  __syncthreads();
  return min(n, want);
}
// The first elements that equal `order`, by id, behind `have` chosen ones: a row of vectors a turn.
template <typename T>
__device__ __forceinline__ int take_ties(const Row<T>& row, ScoreShared& sh, int first, int last, int edges, uint32_t order, int have, int want) {
  constexpr int PER = Row<T>::PER;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int turns = (last - first + kScoreThreads - 1) / kScoreThreads;
  // turn -1: the elements before the first vector; turn `turns`: those behind the last one
#pragma unroll 1
  for (int turn = -1; turn <= turns && have < want; ++turn) {
    uint32_t equal = 0;
    int id = 0;
    if (turn < 0 || turn == turns) {
      const bool mine = turn < 0 ? tid < min(edges, row.head) : tid < edges - row.head;
      if (mine) {
        id = row.edge_id(turn < 0 ? tid : row.head + tid);
        equal = order_of(to_float(row.x[id])) == order ? 1u : 0u;
      }
    } else if (first + turn * kScoreThreads + tid < last) {
      const int i = first + turn * kScoreThreads + tid;
      uint32_t o[PER];
      orders_of<T>(row.vector(i), o);
      id = row.id(i);
#pragma unroll
      for (int e = 0; e < PER; ++e) equal |= o[e] == order ? 1u << e : 0u;
    }
    const int n = __popc(equal);
    int before = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before += other;
    }
    if (lane == 31) sh.scan[warp] = before;
    __syncthreads();
    int all = 0;
    before -= n;
#pragma unroll
    for (int w = 0; w < kScoreWarps; ++w) {
      if (w < warp) before += sh.scan[w];
      all += sh.scan[w];
    }
    for (int at = have + before; equal != 0 && at < want; ++at, equal &= equal - 1) sh.chosen[at] = ranked(order, static_cast<uint32_t>(id + __ffs(equal) - 1));
    have = min(want, have + all);
    __syncthreads();
  }
  return have;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads) score_kernel(const __grid_constant__ ScoreParams p) {
  extern __shared__ __align__(16) uint32_t piece_best[];  // [pieces][threads]
  __shared__ ScoreShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t r = blockIdx.x / p.parts;
  const int part = blockIdx.x % p.parts;
  const T* base = static_cast<const T*>(p.a.logits) + r * p.a.ld;
  const Row<T> row(base, p.a.vocab);
  // the given token's logit is on its way while the row is read
  int64_t token = -1;
  float given = 0.0f;
  if (part == 0 && tid == 0) {
    token = p.a.tokens[r];
    if (token >= 0 && token < p.a.vocab) given = to_float(base[token]);
  }
  const int share = (row.vectors + p.parts - 1) / p.parts;
  const int first = min(part * share, row.vectors), last = min(first + share, row.vectors);
  const int edges = part == 0 ? row.head + row.tail : 0;

  Sums mine{-INFINITY, 0.0f, 0.0f};
  const int pieces = (last - first + kPieceLoads * kScoreThreads - 1) / (kPieceLoads * kScoreThreads);
#pragma unroll 1
  for (int q = 0; q < pieces; ++q) {
    uint4 v[kPieceLoads];
#pragma unroll
    for (int u = 0; u < kPieceLoads; ++u) {
      const int i = first + (q * kPieceLoads + u) * kScoreThreads + tid;
      v[u] = i < last ? row.vector(i) : make_uint4(lowest_word<T>(), lowest_word<T>(), lowest_word<T>(), lowest_word<T>());
    }
    uint32_t top = lowest_word<T>();
#pragma unroll
    for (int u = 0; u < kPieceLoads; ++u) top = max_words<T>(max_words<T>(top, max_words<T>(v[u].x, v[u].y)), max_words<T>(v[u].z, v[u].w));
    float most;
    if constexpr (std::is_same<T, float>::value) {
      most = __uint_as_float(top);
    } else {
      const float2 f = word_pair<T>(top);
      most = max_nan(f.x, f.y);
    }
    if constexpr (TOP) {
      const bool any = first + q * kPieceLoads * kScoreThreads + tid < last;
      piece_best[q * kScoreThreads + tid] = any ? order_of(most) : 0u;
    }
    if (!(most <= mine.m)) mine = moved(mine, max_nan(most, mine.m));
    const float ref = reference(mine.m);
    const uint64_t minus_ref = pair64(-ref, -ref), log2e = pair64(kLog2e, kLog2e);
    uint64_t s2 = pair64(mine.s, 0.0f), t2 = pair64(mine.t, 0.0f);
    const auto take = [&](float a, float b) {
      // the difference first: exact near the maximum, however large that is
      const uint64_t d2 = add2(pair64(a, b), minus_ref);
      float da, db, ea, eb;
      unpair64(mul2(d2, log2e), ea, eb);
      unpair64(d2, da, db);
      const uint64_t e2 = pair64(exp2_ftz(ea), exp2_ftz(eb));
      s2 = add2(s2, e2);
      // a logit of minus infinity has no weight: 0 times a finite difference
      t2 = fma2(e2, pair64(fmaxf(da, -1e30f), fmaxf(db, -1e30f)), t2);
    };
#pragma unroll
    for (int u = 0; u < kPieceLoads; ++u) {
      if constexpr (std::is_same<T, float>::value) {
        take(__uint_as_float(v[u].x), __uint_as_float(v[u].y));
        take(__uint_as_float(v[u].z), __uint_as_float(v[u].w));
      } else {
        const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = word_pair<T>(w[i]);
          take(f.x, f.y);
        }
      }
    }
    float a, b;
    unpair64(s2, a, b);
    mine.s = a + b;
    unpair64(t2, a, b);
    mine.t = a + b;
  }
  const float body = mine.m;  // of the pieces alone
  if (tid < edges) {
    const float x = to_float(row.x[row.edge_id(tid)]);
    mine = joined(mine, x == -INFINITY ? Sums{x, 0.0f, 0.0f} : Sums{x, x - x == 0.0f ? 1.0f : x - x, 0.0f});
  }

  // ---------------------------------------------------------------- the row's sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    mine = joined(mine, Sums{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.t, o)});
  if (lane == 0) sh.warp[warp] = mine;
  if constexpr (TOP) {
    uint32_t best = pieces > 0 && first + tid < last ? order_of(body) : 0u;
    best = max(best, __shfl_xor_sync(0xffffffffu, best, 1));
    best = max(best, __shfl_xor_sync(0xffffffffu, best, 2));
    // the group takes the place of the last bits: no two are equal, and the threshold is not above the true one
    if ((lane & 3) == 0) reinterpret_cast<uint32_t*>(sh.best)[tid >> 2] = (best & ~static_cast<uint32_t>(kGroups - 1)) | static_cast<uint32_t>(tid >> 2);
  }
  __syncthreads();
  if (tid == 0) {
    Sums all = sh.warp[0];
#pragma unroll
    for (int w = 1; w < kScoreWarps; ++w) all = joined(all, sh.warp[w]);
    sh.block = all;
  }

  // ---------------------------------------------------------------- the block's top elements
  int have = 0;
  if constexpr (TOP) {
    const int want = p.a.top;
    if (tid < kGroups) {
      const uint32_t best = reinterpret_cast<const uint32_t*>(sh.best)[tid];
      int above = 0;
#pragma unroll
      for (int j = 0; j < kGroups / 4; ++j) {
        const uint4 o = sh.best[j];
        above += (o.x > best ? 1 : 0) + (o.y > best ? 1 : 0) + (o.z > best ? 1 : 0) + (o.w > best ? 1 : 0);
      }
      if (above == want - 1) sh.threshold = best & ~static_cast<uint32_t>(kGroups - 1);  // 0 where fewer groups have elements: all of these are looked at
    }
    __syncthreads();
    uint32_t least = max(sh.threshold, 1u);
    int n = gather<T>(row, sh, piece_best, pieces, first, last, edges, least);
    if (n >= 0 && n <= kCandidates) {
      have = rank_candidates(sh, n, want, sh.chosen);
    } else {
      // More than there are places for, by many equal elements or by their order.  The threshold rises to one that enough elements reach; what lies above it is wanted, and of
      // what lies at it, in order, as many as are left.  If the former is too much as well, once more.
      for (bool again = false; n < 0 || n > kCandidates; again = true) {
        least = raised(sh, piece_best, n, want, again);
        n = least == 0xffffffffu ? 0 : gather<T>(row, sh, piece_best, pieces, first, last, edges, least + 1);
      }
      have = rank_candidates(sh, n, want, sh.chosen);
      if (have < want) have = take_ties<T>(row, sh, first, last, edges, least, have, want);
    }
  }

  // ---------------------------------------------------------------- the cluster joins
  if (p.parts > 1) {
    if constexpr (TOP) {
      if (tid >= have && tid < p.a.top) sh.chosen[tid] = 0;
    }
    cluster_arrive_wait();
    if (part == 0) {
      if (tid == 0) {
        Sums all = sh.block;
        const uint32_t at = smem_u32(&sh.block);
#pragma unroll 1
        for (int o = 1; o < p.parts; ++o) all = joined(all, Sums{__uint_as_float(ld_cluster_u32(in_block(at, o))), __uint_as_float(ld_cluster_u32(in_block(at + 4, o))), __uint_as_float(ld_cluster_u32(in_block(at + 8, o)))});
        sh.block = all;
      }
      if constexpr (TOP) {
        const int n = p.parts * p.a.top;  // at most 8 x 32
        if (tid < n) {
          const uint32_t at = in_block(smem_u32(&sh.chosen[tid % p.a.top]), tid / p.a.top);
          sh.candidate[tid] = static_cast<uint64_t>(ld_cluster_u32(at + 4)) << 32 | ld_cluster_u32(at);
        }
      }
    }
    cluster_arrive_wait();  // nobody leaves, and nobody's choice changes, while it is read
    if (part != 0) return;
    if constexpr (TOP) {
      // empty places are 0 and stand behind all others; no two others are equal
      const int n = p.parts * p.a.top;
      if (tid < n) {
        const uint64_t own = sh.candidate[tid];
        int above = 0;
        for (int j = 0; j < n; ++j) above += sh.candidate[j] > own ? 1 : 0;
        if (own != 0 && above < p.a.top) sh.chosen[above] = own;
      }
    }
  }
  __syncthreads();

  // ---------------------------------------------------------------- results
  const Sums all = sh.block;
  const float ref = reference(all.m), log_s = logf(all.s);
  if (tid == 0) {
    if (token >= p.a.vocab && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
    p.a.logprobs[r] = token < 0 || token >= p.a.vocab ? 0.0f : (given - ref) - log_s;
    p.a.entropy[r] = log_s - all.t / all.s;
    if (p.a.stats != nullptr) {
      p.a.stats[2 * r] = ref;
      p.a.stats[2 * r + 1] = log_s;
    }
  }
  if constexpr (TOP) {
    if (tid < p.a.top) {
      const uint64_t one = sh.chosen[tid];
      p.a.top_ids[r * p.a.top + tid] = static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(one));
      p.a.top_logprobs[r * p.a.top + tid] = (value_of(static_cast<uint32_t>(one >> 32)) - ref) - log_s;
    }
  }
}

// ------------------------------------------------------------------------------------------------ the gradient
// 16-byte pieces of a thread.  Blocks that go over four times as much with the next loads under way are slower: 2048 x 128256, forward and backward, 311 us, 263 so.
constexpr int kGradLoads = 4;

template <typename T>
__global__ void __launch_bounds__(kScoreThreads) score_grad_kernel(const __grid_constant__ ScoreParams p) {
  constexpr int PER = 16 / sizeof(T);
  const int64_t r = blockIdx.x / p.parts;
  const int part = blockIdx.x % p.parts;
  const int vocab = p.a.vocab;
  const T* x = static_cast<const T*>(p.a.logits) + r * p.a.ld;
  T* out = static_cast<T*>(p.a.d_logits) + r * vocab;
  const int64_t token = p.a.tokens[r];
  const bool known = token >= 0 && token < vocab;
  const float dl = known && p.a.d_logprobs != nullptr ? p.a.d_logprobs[r] : 0.0f, dh = p.a.d_entropy != nullptr ? p.a.d_entropy[r] : 0.0f;
  const float ref = p.a.stats[2 * r], log_s = p.a.stats[2 * r + 1], entropy = p.a.entropy[r];
  const bool none = dl == 0.0f && dh == 0.0f;
  // p (a + b log p) for two logits, with the [j = t] term left out; where there is no probability log p is finite: 0 times a finite number
  const float a = -fmaf(dh, entropy, dl), b = -dh;
  const uint64_t minus_ref = pair64(-ref, -ref), minus_log_s = pair64(-log_s, -log_s), log2e = pair64(kLog2e, kLog2e), a2 = pair64(a, a), b2 = pair64(b, b);
  const auto gradient = [&](float& u, float& w) {
    float lu, lw, eu, ew;
    unpair64(add2(add2(pair64(u, w), minus_ref), minus_log_s), lu, lw);
    const uint64_t log_p = pair64(fmaxf(lu, -1e30f), fmaxf(lw, -1e30f));
    unpair64(mul2(pair64(lu, lw), log2e), eu, ew);
    unpair64(mul2(pair64(exp2_ftz(eu), exp2_ftz(ew)), fma2(log_p, b2, a2)), u, w);
  };
  const Row<T> row(reinterpret_cast<const T*>(out), vocab);  // pieces by where the gradient lies
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const auto vector_of = [&](int u) { return (part * kGradLoads + u) * kScoreThreads + static_cast<int>(threadIdx.x); };
  uint4 v[kGradLoads];
#pragma unroll
  for (int u = 0; u < kGradLoads; ++u) {
    const int i = vector_of(u);
    if (i >= row.vectors || none) continue;
    const T* at = x + row.id(i);
    if (same) {
      v[u] = __ldg(reinterpret_cast<const uint4*>(at));
    } else {
      float e[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) e[j] = to_float(at[j]);
      v[u] = packed<T>(e);
    }
  }
#pragma unroll
  for (int u = 0; u < kGradLoads; ++u) {
    const int i = vector_of(u);
    if (i >= row.vectors) continue;
    const int id = row.id(i);
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (!none) {
      const uint32_t in[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      float e[PER];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (std::is_same<T, float>::value) {
          e[j] = __uint_as_float(in[j]);
        } else {
          const float2 f = word_pair<T>(in[j]);
          e[2 * j] = f.x;
          e[2 * j + 1] = f.y;
        }
      }
#pragma unroll
      for (int j = 0; j < PER; j += 2) gradient(e[j], e[j + 1]);
      if (token >= id && token < id + PER) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (token == id + j) e[j] += dl;
      }
      w = packed<T>(e);
    }
    reinterpret_cast<uint4*>(out + row.head)[i] = w;
  }
  if (part == 0 && static_cast<int>(threadIdx.x) < row.head + row.tail) {
    const int id = row.edge_id(threadIdx.x);
    float e = to_float(x[id]), twice = e;
    gradient(e, twice);
    out[id] = from_float<T>(none ? 0.0f : id == token ? e + dl : e);
  }
}

// ------------------------------------------------------------------------------------------------ host
static int check_score(const qlin_token_logprobs_args* a, const char* what) {
  if (a == nullptr) return fail(QLIN_ERR_NULL, "%s: args is NULL", what);
  if (a->rows < 0 || a->vocab < 1 || a->top < 0) return fail(QLIN_ERR_BAD_SHAPE, "%s: rows and top must not be negative, vocab must be positive", what);
  if (a->vocab > kMostVocab) return fail(QLIN_ERR_TOO_LARGE, "%s: at most %d logits a row", what, kMostVocab);
  if (a->top > kMostTop || a->top > a->vocab) return fail(QLIN_ERR_BAD_SHAPE, "%s: top must be at most %d and at most vocab", what, kMostTop);
  if (a->dtype != QLIN_DT_F32 && a->dtype != QLIN_DT_F16 && a->dtype != QLIN_DT_BF16) return fail(QLIN_ERR_BAD_DTYPE, "%s: logits must be fp32, fp16 or bf16", what);
  if (a->ld < 0) return fail(QLIN_ERR_BAD_SHAPE, "%s: ld must not be negative", what);
  return QLIN_OK;
}

// Blocks of a row: as many as fill the SMs, with two pieces of a thread each at least.
static int parts_of(int64_t rows, int vectors) {
  int parts = 1;
  while (parts < kMostParts && rows * parts * 2 <= 2 * sm_count() && vectors >= parts * 2 * kScoreThreads * 2) parts *= 2;
  return parts;
}

template <typename T, bool TOP>
static int launch_score(ScoreParams p, cudaStream_t stream) {
  const auto kernel = score_kernel<T, TOP>;
  const int vectors = p.a.vocab / (16 / static_cast<int>(sizeof(T)));
  p.parts = parts_of(p.a.rows, vectors);
  const int share = (vectors + p.parts - 1) / p.parts;
  p.pieces = (share + kPieceLoads * kScoreThreads - 1) / (kPieceLoads * kScoreThreads);
  const int smem = TOP ? p.pieces * kScoreThreads * 4 : 0;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(QLIN_ERR_DEVICE, "device ordinal %d out of range", dev);
  if (TOP && !configured[dev]) {
    constexpr int most = (kMostVocab / (16 / static_cast<int>(sizeof(T))) + kPieceLoads * kScoreThreads - 1) / (kPieceLoads * kScoreThreads) * kScoreThreads * 4;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return fail(QLIN_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  if (static_cast<int64_t>(p.a.rows) * p.parts > 0x7fffffff) return fail(QLIN_ERR_TOO_LARGE, "qlin_token_logprobs: too many rows");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.a.rows) * p.parts, 1, 1);
  cfg.blockDim = dim3(kScoreThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.parts);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.parts > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(QLIN_ERR_LAUNCH, "qlin_token_logprobs: %s", cudaGetErrorString(e));
  }
  return QLIN_OK;
}

template <typename T>
static int launch_score_grad(ScoreParams p, cudaStream_t stream) {
  const int vectors = p.a.vocab / (16 / static_cast<int>(sizeof(T)));
  p.parts = vectors / (kGradLoads * kScoreThreads) + 1;
  const int64_t blocks = static_cast<int64_t>(p.a.rows) * p.parts;
  if (blocks > 0x7fffffff) return fail(QLIN_ERR_TOO_LARGE, "qlin_token_logprobs_bwd: too many rows");
  score_grad_kernel<T><<<static_cast<unsigned>(blocks), kScoreThreads, 0, stream>>>(p);
  QLIN_CHECK_LAUNCH("qlin_token_logprobs_bwd");
  return QLIN_OK;
}

}  // namespace qlin

extern "C" int qlin_token_logprobs(const qlin_token_logprobs_args* a, void* stream) {
  using namespace qlin;
  const int rc = check_score(a, "qlin_token_logprobs");
  if (rc != QLIN_OK) return rc;
  if (a->rows == 0) return QLIN_OK;
  if (a->logits == nullptr || a->tokens == nullptr || a->logprobs == nullptr || a->entropy == nullptr || (a->top > 0 && (a->top_logprobs == nullptr || a->top_ids == nullptr)))
    return fail(QLIN_ERR_NULL, "qlin_token_logprobs: logits, tokens or an output is NULL");
  if (reinterpret_cast<uintptr_t>(a->logits) % dtype_size(a->dtype) != 0) return fail(QLIN_ERR_BAD_ALIGN, "qlin_token_logprobs: logits must be aligned to their type");
  const ScoreParams p{*a, 1, 0};
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool top = a->top > 0;
  if (a->dtype == QLIN_DT_F32) return top ? launch_score<float, true>(p, s) : launch_score<float, false>(p, s);
  if (a->dtype == QLIN_DT_F16) return top ? launch_score<__half, true>(p, s) : launch_score<__half, false>(p, s);
  return top ? launch_score<__nv_bfloat16, true>(p, s) : launch_score<__nv_bfloat16, false>(p, s);
}

extern "C" int qlin_token_logprobs_bwd(const qlin_token_logprobs_args* a, void* stream) {
  using namespace qlin;
  const int rc = check_score(a, "qlin_token_logprobs_bwd");
  if (rc != QLIN_OK) return rc;
  if (a->rows == 0) return QLIN_OK;
  if (a->logits == nullptr || a->tokens == nullptr || a->entropy == nullptr || a->stats == nullptr || a->d_logits == nullptr)
    return fail(QLIN_ERR_NULL, "qlin_token_logprobs_bwd: logits, tokens, entropy, stats or d_logits is NULL");
  const int size = dtype_size(a->dtype);
  if (reinterpret_cast<uintptr_t>(a->logits) % size != 0 || reinterpret_cast<uintptr_t>(a->d_logits) % size != 0)
    return fail(QLIN_ERR_BAD_ALIGN, "qlin_token_logprobs_bwd: logits and d_logits must be aligned to their type");
  const ScoreParams p{*a, 1, 0};
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == QLIN_DT_F32) return launch_score_grad<float>(p, s);
  if (a->dtype == QLIN_DT_F16) return launch_score_grad<__half>(p, s);
  return launch_score_grad<__nv_bfloat16>(p, s);
}
