// Attention of one new token of every sequence over a paged cache: the kernels behind qlin_paged_attention (qlin_paged.cu says what they do and
// what they measured) and, with a prefix that sequences share, behind qlin_prefix_attention (qlin_prefix.cu).
#pragma once
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qlin_internal.h"
#include "qlin_ptx.cuh"

namespace qlin {

constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = kPagedWarps * 32;
constexpr int kTileKeys = 16;
constexpr int kMinTiles = 4;       // tiles of a block at least, one a warp (with eight 1 x 2048 keys take 0.9 us more)

// Sequences that share a prefix (qlin_prefix_attention): what all of a group's see of it is read once for all of them, kShared, and everything else
// of a sequence with its own tokens, kOwn, whose blocks take the former's sums in as one more part of the split.
enum PagedMode { kSingle, kOwn, kShared };
struct SharedPrefix {
  const int32_t* table;   // [groups, max_pages], row stride table_stride
  const int32_t* lens;    // [groups]
  const int32_t* groups;  // [count + 1]: first sequence of each
  int64_t table_stride;
  int32_t count, max_pages, splits;
  int32_t blocks;         // of the launch
  int32_t align;          // a power of two: the keys that are read for a group begin and end at multiples of it
  float* part_o;          // [batch * q_heads, splits, head_dim]
  float2* part_ml;        // [batch * q_heads, splits]: maximum and sum
};

struct PagedParams {
  qlin_paged_attention_args a;
  int32_t splits, head_blocks, group;  // blocks of query heads per kv head, query heads per kv head
  int32_t page_shift;                  // log2 of the page size, or -1
  int32_t cluster;                     // the splits of a head are a cluster of blocks and join in shared memory
  float* part_o;                       // [batch * q_heads, splits, head_dim]
  float2* part_ml;                     // [batch * q_heads, splits]: maximum and sum
  SharedPrefix pre;
};

// The visible keys of a sequence in order: `sinks` first ones, then those from `start` on.
struct Visible {
  int sinks, start, n;
  __device__ __forceinline__ int key(int u) const { return u < sinks ? u : start + (u - sinks); }
};
__device__ __forceinline__ Visible visible_keys(int len, int window, int sinks) {
  Visible v;
  v.start = window > 0 && len > window ? len - window : 0;
  v.sinks = min(max(sinks, 0), v.start);
  v.n = v.sinks + len - v.start;
  return v;
}
// `shared`: tokens of the prefix that the sequence may hold whatever the width of its own table.
__device__ __forceinline__ int sequence_length(const PagedParams& p, int b, bool report, int shared = 0) {
  const int64_t own = p.a.num_pages > 0 ? static_cast<int64_t>(p.a.max_pages) * p.a.page_size : 0, most = own > shared ? own : shared;
  const int len = p.a.lens[b];
  if (len < 0 || len > most) {
    if (report && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
    return len < 0 ? 0 : static_cast<int>(most);
  }
  return len;
}
// Tiles of each split, and how many splits have any.
__device__ __forceinline__ int tiles_per_split(int tiles, int splits) { return max(kMinTiles, (tiles + splits - 1) / splits); }
__device__ __forceinline__ int splits_used(int tiles, int per) { return max(1, (tiles + per - 1) / per); }

// The keys [from, to) of a group's prefix that each of its sequences sees (those of length 0 aside); none where to is 0.
struct Common {
  int first, sequences, prefix, from, to;
};
// Reported by one block of a launch: groups that do not rise from 0 to the batch.
__device__ __forceinline__ void check_groups(const PagedParams& p) {
  bool bad = p.pre.groups[0] != 0 || p.pre.groups[p.pre.count] != p.a.batch;
  for (int g = threadIdx.x; g < p.pre.count; g += blockDim.x) bad |= p.pre.groups[g] > p.pre.groups[g + 1];
  if (bad && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
}
__device__ __forceinline__ Common common_keys(const PagedParams& p, int g, int g0, int g1, bool report) {  // by a whole warp
  const int given = p.pre.lens[g];  // beside the lengths, before anything waits for it
  const bool rises = g0 >= 0 && g0 <= g1 && g1 <= p.a.batch;
  const int64_t most = p.a.num_pages > 0 ? static_cast<int64_t>(p.pre.max_pages) * p.a.page_size : 0;
  const int64_t wide = p.a.num_pages > 0 ? static_cast<int64_t>(p.a.max_pages) * p.a.page_size : 0;
  Common c{rises ? g0 : 0, rises ? g1 - g0 : 0, 0, 0, 0};
  int longest = 0, shortest = 0x7fffffff;  // of the lengths as they are given
  for (int i = threadIdx.x & 31; i < c.sequences; i += 32) {
    const int len = p.a.lens[c.first + i];
    if (len > 0) {
      longest = max(longest, len);
      shortest = min(shortest, len);
    }
  }
  c.prefix = given < 0 ? 0 : given > most ? static_cast<int>(most) : given;
  if (report && c.prefix != given && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
  longest = __reduce_max_sync(0xffffffffu, longest);
  shortest = __reduce_min_sync(0xffffffffu, shortest);
  if (longest == 0) return c;
  const int cut = static_cast<int>(wide > c.prefix ? wide : c.prefix);  // lengths above it are cut there
  longest = min(longest, cut);
  const int first = p.a.window > 0 && longest > p.a.window ? longest - p.a.window : 0, past = p.pre.align - 1;
  const int from = (first + past) & ~past, to = min(min(shortest, cut), c.prefix) & ~past;
  c.from = from < to ? from : 0;
  c.to = from < to ? to : 0;
  return c;
}
// Keys of a split of n common keys, and how many splits have any.
constexpr int kSharedStep = 128;
__device__ __forceinline__ int keys_per_split(int n, int splits) { return max(1, (n + kSharedStep * splits - 1) / (kSharedStep * splits)) * kSharedStep; }
__device__ __forceinline__ int shared_splits(const SharedPrefix& pre, const Common& c) {
  const int n = c.to - c.from, per = keys_per_split(n, pre.splits);
  return (n + per - 1) / per;
}
// The kv head, the group and the block of `columns` of its rows of a unit, by a whole warp, 32 groups a look; false: there is no such unit.
__device__ __forceinline__ bool shared_unit(const PagedParams& p, int unit, int columns, int& kvh, int& g, int& block) {
  const int lane = threadIdx.x & 31;
  kvh = unit % p.a.kv_heads;
  int left = unit / p.a.kv_heads;
  for (int base = 0; base < p.pre.count; base += 32) {
    int blocks = 0;
    if (base + lane < p.pre.count) {
      const int rows = max(0, min(p.pre.groups[base + lane + 1], p.a.batch) - max(p.pre.groups[base + lane], 0)) * p.group;
      blocks = (rows + columns - 1) / columns;
    }
    int upto = blocks;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += other;
    }
    const int here = __shfl_sync(0xffffffffu, upto, 31);
    if (left < here) {
      const int owner = __ffs(__ballot_sync(0xffffffffu, left < upto)) - 1;
      g = base + owner;
      block = left - __shfl_sync(0xffffffffu, upto - blocks, owner);
      return true;
    }
    left -= here;
  }
  return false;
}
// What is left to a sequence: its first keys and those of its window before the common ones, then what follows these.
struct Rest {
  int sinks, start, mid, after, n;
  __device__ __forceinline__ int key(int u) const { return u < sinks ? u : u < sinks + mid ? start + (u - sinks) : after + (u - sinks - mid); }
};
__device__ __forceinline__ Rest rest_of(const Visible& v, const Common& c, int len) {
  Rest r{v.sinks, v.start, 0, v.start, v.n};
  if (c.to > 0 && len > 0) {
    r.mid = c.from - v.start;
    r.after = c.to;
    r.n = v.sinks + r.mid + (len - c.to);
  }
  return r;
}
// The group of a sequence and its bounds, by a whole warp: 32 bounds a look.  g is -1 where the groups do not say.
struct Group {
  int g, first, end;
};
__device__ __forceinline__ Group group_of(const SharedPrefix& pre, int b) {
  const int lane = threadIdx.x & 31;
  for (int base = 0; base < pre.count; base += 31) {
    const int at = min(base + lane, pre.count), bound = pre.groups[at];
    const uint32_t under = __ballot_sync(0xffffffffu, bound <= b && base + lane < pre.count);
    const int i = under == 0 ? 0 : 31 - __clz(under);
    const int first = __shfl_sync(0xffffffffu, bound, i), end = __shfl_sync(0xffffffffu, bound, min(i + 1, 31));
    if (under != 0 && i < 31 && first <= b && b < end) return Group{base + i, first, end};
  }
  return Group{-1, 0, 0};
}
// The sums over the prefix join those of a sequence's own keys, which carry a factor of `shift`, sixteen splits at a time in order.  Sixteen lanes that have outputs of one head
// (d: the first of four) share the work on maxima and sums, a split each: done by every lane for itself, with the library's exponential, a turn took 4000 cycles.
constexpr int kJoinAtOnce = 16;
__device__ __forceinline__ float exp2_or_zero(float x) {  // 2 ulp
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void join_prefix(const PagedParams& p, int64_t row, int d, int used, float shift, float& top, float& sum, float (&acc)[4]) {
  const int lane = threadIdx.x & 31, base = lane & 16;
  const uint32_t group = 0xffffu << base;
  const float2* ml = p.pre.part_ml + row * p.pre.splits;
  const float* o = p.pre.part_o + row * p.pre.splits * p.a.head_dim + min(d, p.a.head_dim - 4);
#pragma unroll 1
  for (int s0 = 0; s0 < used; s0 += kJoinAtOnce) {
    const int mine = s0 + (lane & 15);
    float4 v[kJoinAtOnce];
    float2 one = __ldcg(ml + min(mine, used - 1));
#pragma unroll
    for (int i = 0; i < kJoinAtOnce; ++i)  // past the last one it is read again: loads behind branches would wait for one another
      v[i] = __ldcg(reinterpret_cast<const float4*>(o + static_cast<int64_t>(min(s0 + i, used - 1)) * p.a.head_dim));
    if (mine >= used) one = make_float2(-INFINITY, 0.0f);
    float most = one.x;
#pragma unroll
    for (int w = 1; w < kJoinAtOnce; w <<= 1) most = fmaxf(most, __shfl_xor_sync(group, most, w));
    most = fmaxf(most, top);
    const float ref = most == -INFINITY ? 0.0f : most, keep = exp2_or_zero(top - ref), f = exp2_or_zero(one.x - ref) * shift;
    float total = one.y * f;
#pragma unroll
    for (int w = 1; w < kJoinAtOnce; w <<= 1) total += __shfl_xor_sync(group, total, w);
    top = most;
    sum = fmaf(sum, keep, total);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= keep;
#pragma unroll
    for (int i = 0; i < kJoinAtOnce; ++i) {
      const float fi = __shfl_sync(group, f, base + i);
      if (s0 + i < used) {  // not 0 times what is read again
        acc[0] = fmaf(v[i].x, fi, acc[0]);
        acc[1] = fmaf(v[i].y, fi, acc[1]);
        acc[2] = fmaf(v[i].z, fi, acc[2]);
        acc[3] = fmaf(v[i].w, fi, acc[3]);
      }
    }
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Two e4m3 codes (the low or the high half of a register) as fp16.
__device__ __forceinline__ uint32_t widen_lo(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Four outputs from their sums; zeros where there is no weight at all, whatever the values hold.
template <bool BF16>
__device__ __forceinline__ uint2 outputs4(const float (&acc)[4], float sum, float v_scale) {
  if (sum == 0.0f) return make_uint2(0u, 0u);
  const float r = v_scale / sum;
  return make_uint2(pack16<BF16>(acc[0] * r, acc[1] * r), pack16<BF16>(acc[2] * r, acc[3] * r));
}
__device__ __forceinline__ float max_of_rows(float v) {  // over the eight lanes that hold one column
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

template <typename QT, bool F8, int DP, int NT, bool OWN = false>
struct PagedCfg {
  static constexpr bool BF16 = std::is_same<QT, __nv_bfloat16>::value && !F8;  // type of the products
  static constexpr int ES = F8 ? 1 : 2;
  static constexpr int RB = DP * ES;                   // bytes of a row
  static constexpr int CH = RB / 16;                   // 16-byte pieces of a row
  static constexpr int STAGE = 2 * kTileKeys * RB;     // keys, then values
  // Three stages at least; where they are small, 16 KB a warp, so that a third block fits the SM: its warps cover the latency of the
  // chain from a tile's keys to its outputs (3 x up to 30000 keys in e4m3 32 us, 37 with two).  16-bit rows of 128 run as fast as
  // memory does with two blocks of three stages (61 x 2050 keys 78 us, three blocks of two stages 95).
  // A sequence's own keys behind a prefix are few: three blocks of two stages there.
  static constexpr int RING = STAGE >= 8192 && !OWN ? 24576 : 16384;
  static constexpr int STAGES = RING / STAGE;
  static constexpr int BLOCKS = NT == 1 && RING == 16384 ? 3 : 2;  // an SM
  static constexpr int LOADS = kTileKeys * CH / 32;    // pieces of K a lane copies, and as many of V
  static constexpr int HEADS = 8 * NT;
  static constexpr int OROW = DP + 4;                  // floats of a row of the joined outputs
  static constexpr int SMEM = kPagedWarps * STAGES * STAGE;
  static constexpr float SHIFT = BF16 ? 0.0f : 12.0f;
  static_assert((kPagedWarps + 1) * HEADS * (OROW + 2) * 4 <= SMEM, "the join reuses the stages");
};

template <int RB>
__device__ __forceinline__ uint32_t piece(int row, int c) {
  return static_cast<uint32_t>(row * RB + ((RB >= 128 ? c ^ (row & 7) : c ^ ((row >> 1) & 3)) << 4));
}

// WARPS: of a unit, a kv head of a sequence (up to 8 or 16 query heads of it).  Fewer than the block's four where there are more units than blocks fit the SMs at once: a block
// then has two or four units, and each unit fewer warps to join.
template <typename QT, bool F8, int DP, int NT, PagedMode MODE, int WARPS>
__global__ void __launch_bounds__(kPagedThreads, (PagedCfg<QT, F8, DP, NT, MODE == kOwn>::BLOCKS)) paged_kernel(const __grid_constant__ PagedParams p) {
  using C = PagedCfg<QT, F8, DP, NT, MODE == kOwn>;
  extern __shared__ __align__(128) uint8_t smem[];
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int splits = MODE == kShared ? p.pre.splits : p.splits;
  const int split = WARPS == kPagedWarps ? blockIdx.x % splits : 0, sub = warp % WARPS;
  const int units = p.a.batch * p.a.kv_heads * p.head_blocks, given = WARPS == kPagedWarps ? blockIdx.x / splits : blockIdx.x * (kPagedWarps / WARPS) + warp / WARPS;
  const bool idle = WARPS != kPagedWarps && given >= units;
  const int unit = idle ? units - 1 : given;
  int b, kvh, head0, heads;  // head0: first query head of the block within the kv head's, kShared: first of the group's rows
  Common common{0, 0, 0, 0, 0};
  if constexpr (MODE == kShared) {
    if (blockIdx.x == 0) check_groups(p);
    int g_, left;
    if (!shared_unit(p, unit, C::HEADS, kvh, g_, left)) return;
    common = common_keys(p, g_, p.pre.groups[g_], p.pre.groups[g_ + 1], threadIdx.x == 0);
    b = g_;
    head0 = left * C::HEADS;
    heads = min(C::HEADS, common.sequences * p.group - head0);
    if (heads <= 0) return;
  } else {
    const int hb = unit % (p.a.kv_heads * p.head_blocks);
    b = unit / (p.a.kv_heads * p.head_blocks);
    kvh = hb / p.head_blocks;
    head0 = hb % p.head_blocks * C::HEADS;
    heads = min(C::HEADS, p.group - head0);
  }
  const int D = p.a.head_dim;
  // a column's row among all [batch, q_heads], and where its query is
  const auto sequence_of = [&](int h) { return MODE == kShared ? common.first + (head0 + h) / p.group : b; };
  const auto head_of = [&](int h) { return kvh * p.group + (MODE == kShared ? (head0 + h) % p.group : head0 + h); };
  int len = 0, group = 0;
  if constexpr (MODE == kSingle) len = sequence_length(p, b, threadIdx.x == 0);
  if constexpr (MODE == kOwn) {
    const bool alone = p.pre.blocks == 0;  // no launch for the prefixes, which would have reported
    if (alone && blockIdx.x == 0) check_groups(p);
    const Group of = group_of(p.pre, b);
    group = of.g;
    if (group >= 0) common = common_keys(p, group, of.first, of.end, alone && lane == 0);
    else if (lane == 0 && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
    len = sequence_length(p, b, lane == 0, common.prefix);
    if (idle) len = 0;
  }
  const auto vis = [&]() {
    if constexpr (MODE == kShared) return Visible{0, common.from, common.to - common.from};
    else if constexpr (MODE == kOwn) return rest_of(visible_keys(len, p.a.window, p.a.sinks), common, len);
    else return visible_keys(len, p.a.window, p.a.sinks);
  }();
  const int tiles = (vis.n + kTileKeys - 1) / kTileKeys;
  const int per = MODE == kShared ? keys_per_split(vis.n, splits) / kTileKeys : tiles_per_split(tiles, splits);
  const int used = MODE == kShared ? shared_splits(p.pre, common) : splits_used(tiles, per);
  if (split >= used && (MODE == kShared || !p.cluster)) {
    if constexpr (MODE == kOwn) griddep_wait();
    return;
  }
  const int first = split * per + sub, last = min(tiles, (split + 1) * per);

  // ---------------------------------------------------------------- loads
  const int32_t* table = MODE == kShared ? p.pre.table + b * p.pre.table_stride : p.a.block_table + static_cast<int64_t>(b) * p.a.table_stride;
  const int32_t* before = MODE == kOwn && group >= 0 ? p.pre.table + group * p.pre.table_stride : nullptr;  // the pages of keys under common.prefix
  const uint8_t* kbase = static_cast<const uint8_t*>(p.a.k_pages);
  const uint8_t* vbase = static_cast<const uint8_t*>(p.a.v_pages);
  const int64_t head_off = kvh * p.a.head_stride;
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::STAGE;
  const int lrow = lane / C::CH, lc = lane % C::CH;  // of the first piece this lane copies
  const bool piece_real = lc * 16 < D * C::ES;
  bool bad_page = false;
  // lane r < 16 finds row r of a tile: its page is read one turn ahead of its copies
  struct Place {
    int page, offset;
  };
  const auto look_up = [&](int tile) {
    const int u = tile * kTileKeys + (lane & 15);
    Place at{0, 0};
    if (tile < last && u < vis.n) {
      const int key = vis.key(u), pg = p.page_shift >= 0 ? key >> p.page_shift : key / p.a.page_size;
      at.offset = key - pg * p.a.page_size;
      if constexpr (MODE == kOwn) at.page = (key < common.prefix ? before : table)[pg];
      else at.page = table[pg];
    }
    return at;
  };
  const auto load_tile = [&](int tile, int stage, Place where) {
    if (tile < last) {
      const bool real = tile * kTileKeys + (lane & 15) < vis.n;
      if (real && (where.page < 0 || where.page >= p.a.num_pages)) {
        bad_page = true;
        where.page = 0;
      }
      const int64_t off = real ? (where.page * p.a.page_stride + where.offset * p.a.slot_stride + head_off) * C::ES : 0;
      const uint32_t reals = __ballot_sync(0xffffffffu, real);
      const uint32_t dst = ring + stage * C::STAGE;
#pragma unroll
      for (int i = 0; i < C::LOADS; ++i) {
        const int row = i * (32 / C::CH) + lrow;
        const int64_t at = __shfl_sync(0xffffffffu, off, row) + lc * 16;
        const uint32_t bytes = piece_real && ((reals >> row) & 1u) ? 16u : 0u;
        cp_async16(dst + piece<C::RB>(row, lc), bytes ? kbase + at : kbase, bytes);
        cp_async16(dst + kTileKeys * C::RB + piece<C::RB>(row, lc), bytes ? vbase + at : vbase, bytes);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  {
    Place ahead[C::STAGES - 1];  // all of them are read together
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) ahead[s] = look_up(first + s * WARPS);
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) load_tile(first + s * WARPS, s, ahead[s]);
  }
  Place place = look_up(first + (C::STAGES - 1) * WARPS);

  // ---------------------------------------------------------------- queries, as columns g of the product's second operand
  uint32_t qf[DP / 16][NT][2];
  float logit_scale[NT][2];  // of the columns 2t and 2t + 1
  {
    const QT* q = static_cast<const QT*>(p.a.q);
    const float base = p.a.scale * 1.4426950408889634f * (F8 ? p.a.k_scale[kvh] : 1.0f);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const bool real = h < heads;
      const QT* row = q + sequence_of(real ? h : 0) * p.a.q_batch + head_of(real ? h : 0) * p.a.q_head;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = 16 * kk + (F8 ? 4 * t + 2 * i : 2 * t + 8 * i);
          qf[kk][nt][i] = real && d < D ? *reinterpret_cast<const uint32_t*>(row + d) : 0u;
        }
      float up = 1.0f;
      if constexpr (F8 && std::is_same<QT, __nv_bfloat16>::value) {
        float top = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(qf[kk][nt][i] << 16)), fabsf(__uint_as_float(qf[kk][nt][i] & 0xffff0000u))));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(13 - exponent), where that and its inverse are normal numbers
        const int e = static_cast<int>(__float_as_uint(top) >> 23);
        const int up_e = min(max(127 + 13 - (e - 127), 1), 253);
        if (top > 0.0f && e < 255) up = __uint_as_float(static_cast<uint32_t>(up_e) << 23);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            qf[kk][nt][i] = pack16<false>(__uint_as_float(qf[kk][nt][i] << 16) * up, __uint_as_float(qf[kk][nt][i] & 0xffff0000u) * up);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) logit_scale[nt][i] = base / __shfl_sync(0xffffffffu, up, (2 * t + i) * 4);
    }
  }

  // ---------------------------------------------------------------- the loop
  float o[DP / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dt][nt][i] = 0.0f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.0f;
  }
  int stage = 0, stage_in = C::STAGES - 1;
  const int krow = (lane & 7) + ((lane >> 3) & 1) * 8, kc = lane >> 4;   // ldmatrix: rows, then pieces
  const int vrow = (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;   // ldmatrix.trans of 16-bit values: pieces, then rows
  for (int tile = first; tile < last; tile += WARPS) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    __syncwarp();
    load_tile(tile + (C::STAGES - 1) * WARPS, stage_in, place);  // into the stage of the tile before this one
    place = look_up(tile + C::STAGES * WARPS);
    const uint32_t ks = ring + stage * C::STAGE, vs = ks + kTileKeys * C::RB;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
    if constexpr (F8) {
#pragma unroll
      for (int c = 0; c < DP / 16; c += 2) {
        uint32_t r[4];
        ldsm4(ks + piece<C::RB>(krow, c + kc), r);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a0 = widen_lo(r[2 * i]), a1 = widen_lo(r[2 * i + 1]), a2 = widen_hi(r[2 * i]), a3 = widen_hi(r[2 * i + 1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<C::BF16>(s[nt], a0, a1, a2, a3, qf[c + i][nt][0], qf[c + i][nt][1]);
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        uint32_t r[4];
        ldsm4(ks + piece<C::RB>(krow, 2 * kk + kc), r);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<C::BF16>(s[nt], r[0], r[1], r[2], r[3], qf[kk][nt][0], qf[kk][nt][1]);
      }
    }
    const int left = vis.n - tile * kTileKeys;
    uint32_t pf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] *= logit_scale[nt][i & 1];
      if (left < kTileKeys) {
        if (g >= left) s[nt][0] = s[nt][1] = -INFINITY;
        if (g + 8 >= left) s[nt][2] = s[nt][3] = -INFINITY;
      }
      float ref[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float top = fmaxf(m[nt][i], max_of_rows(fmaxf(s[nt][i], s[nt][i + 2])));
        const float keep = top == m[nt][i] ? 1.0f : exp2f(m[nt][i] - top);
        m[nt][i] = top;
        ref[i] = top == -INFINITY ? 0.0f : top;
        if (__any_sync(0xffffffffu, keep != 1.0f)) {
          l[nt][i] *= keep;
#pragma unroll
          for (int dt = 0; dt < DP / 16; ++dt) {
            o[dt][nt][i] *= keep;
            o[dt][nt][i + 2] *= keep;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[nt][i] = exp2f((s[nt][i] - ref[i & 1]) + C::SHIFT);  // the difference first: exact near the maximum, however large that is
        l[nt][i & 1] += s[nt][i];
        // not to zero in fp16, so that an infinite value stays one (e4m3 has none); NaN is in the sum
        if constexpr (!F8 && !C::BF16) s[nt][i] = fmaxf(s[nt][i], 0x1p-24f);
      }
      pf[nt][0] = transpose8x8(pack16<C::BF16>(s[nt][0], s[nt][1]));
      pf[nt][1] = transpose8x8(pack16<C::BF16>(s[nt][2], s[nt][3]));
    }
    if constexpr (F8) {
#pragma unroll
      for (int c = 0; c < DP / 16; c += 2) {
        uint32_t r[4];
        ldsm4_t(vs + piece<C::RB>(krow, c + kc), r);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = __byte_perm(r[2 * i], 0, 0x3120), y = __byte_perm(r[2 * i + 1], 0, 0x3120);
          const uint32_t a0 = widen_lo(x), a1 = widen_hi(x), a2 = widen_lo(y), a3 = widen_hi(y);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<C::BF16>(o[c + i][nt], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
        }
      }
    } else {
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) {
        uint32_t r[4];
        ldsm4_t(vs + piece<C::RB>(vrow, 2 * dt + vc), r);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<C::BF16>(o[dt][nt], r[0], r[1], r[2], r[3], pf[nt][0], pf[nt][1]);
      }
    }
    __syncwarp();  // every lane has read this stage before the next turn's copies go into it
    if (++stage == C::STAGES) stage = 0;
    if (++stage_in == C::STAGES) stage_in = 0;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (bad_page && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
  __syncthreads();

  // ---------------------------------------------------------------- the block's warps join
  float* warp_o = reinterpret_cast<float*>(smem);                                   // [warps][heads][OROW]
  float2* warp_ml = reinterpret_cast<float2*>(warp_o + kPagedWarps * C::HEADS * C::OROW);  // [warps][heads]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float sum = l[nt][i];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int h = nt * 8 + 2 * t + i;
      if (g == 0) warp_ml[warp * C::HEADS + h] = make_float2(m[nt][i], sum);
      float* row = warp_o + (warp * C::HEADS + h) * C::OROW;
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) {
        row[16 * dt + (F8 ? 2 * g : g)] = o[dt][nt][i];
        row[16 * dt + (F8 ? 2 * g + 1 : g + 8)] = o[dt][nt][i + 2];
      }
    }
  __syncthreads();
  const float v_scale = F8 ? p.a.v_scale[kvh] : 1.0f;
  float* block_o = reinterpret_cast<float*>(warp_ml + kPagedWarps * C::HEADS);  // [heads][OROW]
  float2* block_ml = reinterpret_cast<float2*>(block_o + C::HEADS * C::OROW);   // [heads]
  const auto store_out = [&](int h, int d, const float (&acc)[4], float sum) {
    constexpr bool bf16 = std::is_same<QT, __nv_bfloat16>::value;
    QT* out = static_cast<QT*>(p.a.out) + (static_cast<int64_t>(b) * p.a.q_heads + kvh * p.group + head0 + h) * D + d;
    *reinterpret_cast<uint2*>(out) = outputs4<bf16>(acc, sum, v_scale);
  };
  const int pre_used = MODE == kOwn && len > 0 ? shared_splits(p.pre, common) : 0;
  const auto with_prefix = [&](int h, int d, float (&acc)[4], float& sum, float top) {
    if constexpr (MODE == kOwn) join_prefix(p, static_cast<int64_t>(b) * p.a.q_heads + head_of(h), d, pre_used, C::BF16 ? 1.0f : 4096.0f, top, sum, acc);
  };
  if constexpr (MODE == kOwn) griddep_wait();  // the sums over the prefix are there
  const int warp0 = warp - sub;  // the unit's first
  for (int i = sub * 32 + lane; i < heads * (DP / 4); i += WARPS * 32) {
    const int h = i / (DP / 4), d = i % (DP / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = warp0; w < warp0 + WARPS; ++w) top = fmaxf(top, warp_ml[w * C::HEADS + h].x);
    float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = warp0; w < warp0 + WARPS; ++w) {
      const float2 ml = warp_ml[w * C::HEADS + h];
      const float f = ml.x == top ? 1.0f : exp2f(ml.x - top);
      sum += ml.y * f;
      const float4 v = *reinterpret_cast<const float4*>(warp_o + (w * C::HEADS + h) * C::OROW + d);
      acc[0] += v.x * f;
      acc[1] += v.y * f;
      acc[2] += v.z * f;
      acc[3] += v.w * f;
    }
    if ((MODE != kOwn && d >= D) || idle) continue;
    const bool real = d < D;  // the lanes of a head stay together until the sums over the prefix have joined
    if constexpr (MODE == kShared) {
      constexpr float down = C::BF16 ? 1.0f : 1.0f / 4096.0f;  // without the factor that fp16 weights carry
      const int64_t row = (static_cast<int64_t>(sequence_of(h)) * p.a.q_heads + head_of(h)) * splits + split;
      *reinterpret_cast<float4*>(p.pre.part_o + row * D + d) = make_float4(acc[0] * down, acc[1] * down, acc[2] * down, acc[3] * down);
      if (d == 0) p.pre.part_ml[row] = make_float2(top, sum * down);
      continue;
    }
    const int64_t row = static_cast<int64_t>(b) * p.a.q_heads + kvh * p.group + head0 + h;
    if (p.cluster) {
      if (!real) continue;
      *reinterpret_cast<float4*>(block_o + h * C::OROW + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) block_ml[h] = make_float2(top, sum);
    } else if (used == 1) {
      with_prefix(h, d, acc, sum, top);
      if (real) store_out(h, d, acc, sum);
    } else if (real) {
      *reinterpret_cast<float4*>(p.part_o + (row * p.splits + split) * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) p.part_ml[row * p.splits + split] = make_float2(top, sum);
    }
  }
  if (MODE != kShared && p.cluster) {
    // the blocks of the cluster share out the outputs and read each other's sums, in the order of the splits
    cluster_arrive_wait();
    const uint32_t o_base = smem_u32(block_o), ml_base = smem_u32(block_ml);
    for (int i = static_cast<int>(cluster_cta_rank()) * kPagedThreads + threadIdx.x; i < heads * (DP / 4); i += p.splits * kPagedThreads) {
      const int h = i / (DP / 4), d = i % (DP / 4) * 4;
      if (MODE != kOwn && d >= D) continue;
      float2 ml[8];
      float4 v[8];
      float top = -INFINITY;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < used) {
          ml[r] = ld_cluster_f2(ml_base + h * 8, r);
          v[r] = ld_cluster_f4(o_base + (h * C::OROW + d) * 4, r);
          top = fmaxf(top, ml[r].x);
        }
      float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < used) {
          const float f = ml[r].x == top ? 1.0f : exp2f(ml[r].x - top);
          sum += ml[r].y * f;
          acc[0] += v[r].x * f;
          acc[1] += v[r].y * f;
          acc[2] += v[r].z * f;
          acc[3] += v[r].w * f;
        }
      with_prefix(h, d, acc, sum, top);
      if (d < D) store_out(h, d, acc, sum);
    }
    cluster_arrive_wait();  // nobody leaves while its sums are read
  }
}

// The splits of one query head, in order.  One block a head: its warps take every kJoinWarps-th split, a lane four outputs, and are
// added up in turn.
constexpr int kJoinWarps = 8;
template <typename QT, PagedMode MODE>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const __grid_constant__ PagedParams p, bool f8) {
  __shared__ float warp_top[kJoinWarps], warp_sum[kJoinWarps];
  __shared__ float4 warp_o[kJoinWarps][32];
  const int64_t row = blockIdx.x;
  const int b = static_cast<int>(row / p.a.q_heads), h = static_cast<int>(row % p.a.q_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane * 4, D = p.a.head_dim;
  Common common{0, 0, 0, 0, 0};
  if constexpr (MODE == kOwn) {
    const Group of = group_of(p.pre, b);
    if (of.g >= 0) common = common_keys(p, of.g, of.first, of.end, false);
  }
  const int len = sequence_length(p, b, false, common.prefix);
  const Visible all = visible_keys(len, p.a.window, p.a.sinks);
  const int n = MODE == kOwn ? rest_of(all, common, len).n : all.n;
  const int tiles = (n + kTileKeys - 1) / kTileKeys;
  const int used = splits_used(tiles, tiles_per_split(tiles, p.splits));
  griddep_wait();
  if (used == 1) return;
  const float2* ml = p.part_ml + row * p.splits;
  const float* part = p.part_o + row * p.splits * D;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < used; s += kJoinWarps * 32) top = fmaxf(top, ml[s].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, warp_top[w]);
  float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = warp; s < used; s += kJoinWarps) {
    const float2 v = ml[s];
    const float4 o = d < D ? *reinterpret_cast<const float4*>(part + static_cast<int64_t>(s) * D + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float f = v.x == top ? 1.0f : exp2f(v.x - top);
    sum += v.y * f;
    acc[0] += o.x * f;
    acc[1] += o.y * f;
    acc[2] += o.z * f;
    acc[3] += o.w * f;
  }
  warp_o[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  if (lane == 0) warp_sum[warp] = sum;
  __syncthreads();
  if (warp != 0 || (MODE != kOwn && d >= D)) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) {
    sum += warp_sum[w];
    const float4 o = warp_o[w][lane];
    acc[0] += o.x;
    acc[1] += o.y;
    acc[2] += o.z;
    acc[3] += o.w;
  }
  constexpr bool bf16 = std::is_same<QT, __nv_bfloat16>::value;
  if constexpr (MODE == kOwn) join_prefix(p, row, d, len > 0 ? shared_splits(p.pre, common) : 0, bf16 && !f8 ? 1.0f : 4096.0f, top, sum, acc);
  if (d < D) *reinterpret_cast<uint2*>(static_cast<QT*>(p.a.out) + row * D + d) = outputs4<bf16>(acc, sum, f8 ? p.a.v_scale[h / p.group] : 1.0f);
}

// Splits of the keys: blocks for every SM, none with fewer than kMinTiles tiles where the page table is as wide as its longest
// sequence.  Up to kClusterSplits of them (a power of two) are a cluster of blocks, which joins without a second launch and without
// a workspace; few heads with long tables take more.  Blocks an SM, device time: 16-bit caches two (1 x 131072 keys 86 us, with
// three 90, with six 94; 61 x 2050 78, 78, 93; 61 x up to 4099 79, 79, 86; 16 x up to 8000 47, 47, 59); e4m3 three, and up to nine where they
// join in a cluster, which evens out ragged batches (61 x up to 4099 keys 60 us unsplit, 53 in pairs, 67 in fours; 32 x up to 8000 58 in
// pairs and in fours, 77 in eights; 3 x up to 30000, which join over the workspace, 37 with two blocks, 32 with three and six).
constexpr int kClusterSplits = 8;
struct Splits {
  int32_t n, cluster;
};
inline Splits choose_splits(const qlin_paged_attention_args& a, int head_blocks) {
  int64_t most = static_cast<int64_t>(a.max_pages) * a.page_size;
  if (a.window > 0 && most > static_cast<int64_t>(a.window) + a.sinks) most = static_cast<int64_t>(a.window) + (a.sinks > 0 ? a.sinks : 0);
  const int64_t tiles = (most + kTileKeys - 1) / kTileKeys, rows = static_cast<int64_t>(a.batch) * a.kv_heads * head_blocks;
  const bool f8 = a.cache_dtype == QLIN_DT_F8E4M3;
  const int64_t cap = (tiles + kMinTiles - 1) / kMinTiles, blocks = (f8 ? 3 : 2) * sm_count();
  int64_t want = (blocks + rows - 1) / rows;
  if (want > kClusterSplits && cap > 2 * kClusterSplits) return Splits{static_cast<int32_t>(want < cap ? want : cap), 0};
  if (f8) want = (3 * blocks / 2 + rows - 1) / rows;
  int32_t n = 1;
  while (n < kClusterSplits && n < want && n < cap) n *= 2;
  return Splits{n, n > 1};
}
inline int heads_per_block(int group) { return group <= 8 ? 8 : 16; }

inline int check_paged(const qlin_paged_attention_args* a, const char* what) {
  if (a == nullptr) return fail(QLIN_ERR_NULL, "%s: args is NULL", what);
  if (a->batch < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads != 0)
    return fail(QLIN_ERR_BAD_SHAPE, "%s: q_heads must be a multiple of kv_heads", what);
  if (a->page_size < 1 || a->num_pages < 0 || a->max_pages < 0) return fail(QLIN_ERR_BAD_SHAPE, "%s: bad cache dimensions", what);
  if (!(a->scale > 0.0f) || a->scale > 3.0e38f) return fail(QLIN_ERR_UNSUPPORTED, "%s: scale must be positive and finite", what);
  if (static_cast<int64_t>(a->max_pages) * a->page_size > (1 << 30)) return fail(QLIN_ERR_TOO_LARGE, "%s: at most 2^30 keys a sequence", what);
  if (a->dtype != QLIN_DT_F16 && a->dtype != QLIN_DT_BF16) return fail(QLIN_ERR_BAD_DTYPE, "%s: q must be fp16 or bf16", what);
  if (a->cache_dtype != a->dtype && a->cache_dtype != QLIN_DT_F8E4M3) return fail(QLIN_ERR_BAD_DTYPE, "%s: the cache must have the type of q, or e4m3", what);
  const int step = a->cache_dtype == QLIN_DT_F8E4M3 ? 16 : 8;
  if (a->head_dim < step || a->head_dim % step != 0 || a->head_dim > 128)
    return fail(QLIN_ERR_BAD_SHAPE, "%s: head_dim must be a multiple of %d up to 128", what, step);
  const int head_blocks = (a->q_heads / a->kv_heads + 7) / 8;
  if (static_cast<int64_t>(a->batch) * a->kv_heads * head_blocks > (1 << 24) || static_cast<int64_t>(a->batch) * a->q_heads > (1 << 28))
    return fail(QLIN_ERR_TOO_LARGE, "%s: too many sequences and heads", what);
  return QLIN_OK;
}
inline int check_paged_pointers(const qlin_paged_attention_args* a, const char* what) {
  const bool f8 = a->cache_dtype == QLIN_DT_F8E4M3;
  if (a->q == nullptr || a->out == nullptr || a->lens == nullptr) return fail(QLIN_ERR_NULL, "%s: q, out or lens is NULL", what);
  if (a->max_pages > 0 && a->num_pages > 0 && (a->k_pages == nullptr || a->v_pages == nullptr || a->block_table == nullptr))
    return fail(QLIN_ERR_NULL, "%s: k_pages, v_pages or block_table is NULL", what);
  if (f8 && (a->k_scale == nullptr || a->v_scale == nullptr)) return fail(QLIN_ERR_NULL, "%s: an e4m3 cache needs k_scale and v_scale", what);
  const int cs = f8 ? 1 : 2;
  if (!aligned16(a->q) || !aligned16(a->out) || !aligned16(a->k_pages) || !aligned16(a->v_pages) || a->q_batch * 2 % 16 != 0 || a->q_head * 2 % 16 != 0 ||
      a->page_stride * cs % 16 != 0 || a->head_stride * cs % 16 != 0 || a->slot_stride * cs % 16 != 0)
    return fail(QLIN_ERR_BAD_ALIGN, "%s: every row of q, out and the cache must start on 16 bytes", what);
  return QLIN_OK;
}

template <typename QT, bool F8, int DP, int NT, PagedMode MODE, int WARPS = kPagedWarps>
static int launch_paged(const PagedParams& p, cudaStream_t stream) {
  using C = PagedCfg<QT, F8, DP, NT, MODE == kOwn>;
  const auto kernel = paged_kernel<QT, F8, DP, NT, MODE, WARPS>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(QLIN_ERR_DEVICE, "device ordinal %d out of range", dev);
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return fail(QLIN_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  const bool shared = MODE == kShared, cluster = !shared && p.cluster;
  constexpr unsigned units_of_block = kPagedWarps / WARPS;
  const unsigned blocks = shared ? static_cast<unsigned>(p.pre.blocks) : (static_cast<unsigned>(p.a.batch) * p.a.kv_heads * p.head_blocks * p.splits + units_of_block - 1) / units_of_block;
  cudaLaunchConfig_t main = {};
  main.gridDim = dim3(blocks, 1, 1);
  main.blockDim = dim3(kPagedThreads, 1, 1);
  main.dynamicSmemBytes = C::SMEM;
  main.stream = stream;
  cudaLaunchAttribute how[2];
  if (cluster) {
    how[main.numAttrs].id = cudaLaunchAttributeClusterDimension;
    how[main.numAttrs].val.clusterDim.x = static_cast<unsigned>(p.splits);
    how[main.numAttrs].val.clusterDim.y = how[main.numAttrs].val.clusterDim.z = 1;
    ++main.numAttrs;
  }
  if (MODE == kOwn && p.pre.blocks > 0) {  // beside the end of the launch for the prefix; it waits before it reads what that one wrote
    how[main.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    how[main.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++main.numAttrs;
  }
  main.attrs = how;
  const cudaError_t launched = cudaLaunchKernelEx(&main, kernel, p);
  if (launched != cudaSuccess) {
    cudaGetLastError();
    return fail(QLIN_ERR_LAUNCH, "%s: %s", MODE == kSingle ? "qlin_paged_attention" : "qlin_prefix_attention", cudaGetErrorString(launched));
  }
  if (!shared && p.splits > 1 && !p.cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.a.batch) * p.a.q_heads, 1, 1);
    cfg.blockDim = dim3(kJoinWarps * 32, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_join_kernel<QT, MODE>, p, F8);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(QLIN_ERR_LAUNCH, "%s: %s", MODE == kSingle ? "qlin_paged_attention" : "qlin_prefix_attention", cudaGetErrorString(e));
    }
  }
  return QLIN_OK;
}

// The prefix's part on tcgen05, tiles of 128 rows (qlin_prefix_tc.cu): two tiles a block where `pair`, otherwise one tile and two splits.
// Only where prefix_box says how many keys of a page a copy takes, which `align` then is.
int launch_prefix_tc(const PagedParams& p, bool pair, cudaStream_t stream);
int prefix_box(const qlin_paged_attention_args& a);

}  // namespace qlin
