// qlin_paged_attention: one new token of every sequence against its keys in a paged cache, split over the keys and joined.
//
//   o[h] = sum_j w_j v_j / sum_j w_j,   w_j = 2^(x_j - max x),   x_j = q[h].k_j scale log2(e),   j over the visible keys
//
// What bounds it: HBM, every visible key and value once.  The G = q_heads / kv_heads queries of a kv head share its keys, so a
// block takes up to eight (or sixteen) of them: S^T = K Q^T with the keys as the rows of the tensor core's m16n8k16 tile and the
// queries as its eight columns, then O^T += V^T P^T, whose second operand is the first one's result after a transposition of 8x8
// matrices in registers.  One query against one key is 4 operations per 2 bytes; the instruction for full tiles (tcgen05, 128
// rows) would not make the loads any faster, and this one leaves keys, sums and outputs in the registers of the warp that loaded them.
//
// A warp works alone: 16 keys at a time, its own ring of stages filled by 16-byte asynchronous copies, its own running maximum and
// sums.  No barrier stands in the loop; the four warps of a block join once, at its end, in shared memory.  Rows are found one by
// one through the page table, so a page may have any size and end anywhere in a tile; the table entries of the next tile are read
// while this one is loaded.  Rows behind the last key are zeros in shared memory (never what the page holds there).
//
// e4m3 codes become fp16 in registers (exactly).  The eight 16-byte pieces that ldmatrix hands out hold sixteen codes then, so the
// order of the 16 head dimensions of a step is permuted, the same way in Q (keys) and in the rows of O^T (values).  A bf16 query
// meets them as fp16 times a power of two that brings its largest element to 2^13..2^14: no digit of it is lost above 2^-27 of the largest.
//
// Measured (device time): 1 x 131072 keys of 8 heads of 128 in bf16 87 us, 6.1 TB/s; 61 x 2050 78 us, 6.5 TB/s; 61 x up to 4099 79 us, 6.6 TB/s,
// and in e4m3 53 us, 4.9 TB/s, where the chain of conversions, products and shuffles of a tile is as long as its loads; 1 x 2048 6.9 us,
// which is the latency of the length, the page table, the keys and the join behind one another.  A batch of very unequal lengths takes as long as
// its longest sequence does in the few blocks that the split of all leaves it: 63 x 500 and one of 100000 1128 us, the bytes 82.
//
// Statistics, sums and the join are fp32.  Weights are rounded to the cache's 16-bit type (fp16 with an e4m3 cache) as operands of
// the product; fp16 weights carry a factor of 2^12, so that weights down to 2^-26 of the largest keep 11 bits.
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

struct PagedParams {
  qlin_paged_attention_args a;
  int32_t splits, head_blocks, group;  // blocks of query heads per kv head, query heads per kv head
  int32_t page_shift;                  // log2 of the page size, or -1
  int32_t cluster;                     // the splits of a head are a cluster of blocks and join in shared memory
  float* part_o;                       // [batch * q_heads, splits, head_dim]
  float2* part_ml;                     // [batch * q_heads, splits]: maximum and sum
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
__device__ __forceinline__ int sequence_length(const PagedParams& p, int b, bool report) {
  const int64_t most = p.a.num_pages > 0 ? static_cast<int64_t>(p.a.max_pages) * p.a.page_size : 0;
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

template <typename QT, bool F8, int DP, int NT>
struct PagedCfg {
  static constexpr bool BF16 = std::is_same<QT, __nv_bfloat16>::value && !F8;  // type of the products
  static constexpr int ES = F8 ? 1 : 2;
  static constexpr int RB = DP * ES;                   // bytes of a row
  static constexpr int CH = RB / 16;                   // 16-byte pieces of a row
  static constexpr int STAGE = 2 * kTileKeys * RB;     // keys, then values
  // Three stages at least; where they are small, 16 KB a warp, so that a third block fits the SM: its warps cover the latency of the
  // chain from a tile's keys to its outputs (3 x up to 30000 keys in e4m3 32 us, 37 with two).  16-bit rows of 128 run as fast as
  // memory does with two blocks of three stages (61 x 2050 keys 78 us, three blocks of two stages 95).
  static constexpr int RING = STAGE >= 8192 ? 24576 : 16384;
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

template <typename QT, bool F8, int DP, int NT>
__global__ void __launch_bounds__(kPagedThreads, (PagedCfg<QT, F8, DP, NT>::BLOCKS)) paged_kernel(const __grid_constant__ PagedParams p) {
  using C = PagedCfg<QT, F8, DP, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % p.splits;
  const int hb = blockIdx.x / p.splits % (p.a.kv_heads * p.head_blocks), b = blockIdx.x / p.splits / (p.a.kv_heads * p.head_blocks);
  const int kvh = hb / p.head_blocks, head0 = hb % p.head_blocks * C::HEADS;  // first query head of the block within the kv head's
  const int heads = min(C::HEADS, p.group - head0);
  const int D = p.a.head_dim;
  const int len = sequence_length(p, b, threadIdx.x == 0);
  const Visible vis = visible_keys(len, p.a.window, p.a.sinks);
  const int tiles = (vis.n + kTileKeys - 1) / kTileKeys;
  const int per = tiles_per_split(tiles, p.splits), used = splits_used(tiles, per);
  if (split >= used && !p.cluster) return;
  const int first = split * per + warp, last = min(tiles, (split + 1) * per);

  // ---------------------------------------------------------------- loads
  const int32_t* table = p.a.block_table + static_cast<int64_t>(b) * p.a.table_stride;
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
      at.page = table[pg];
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
    for (int s = 0; s < C::STAGES - 1; ++s) ahead[s] = look_up(first + s * kPagedWarps);
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) load_tile(first + s * kPagedWarps, s, ahead[s]);
  }
  Place place = look_up(first + (C::STAGES - 1) * kPagedWarps);

  // ---------------------------------------------------------------- queries, as columns g of the product's second operand
  uint32_t qf[DP / 16][NT][2];
  float logit_scale[NT][2];  // of the columns 2t and 2t + 1
  {
    const QT* q = static_cast<const QT*>(p.a.q) + b * p.a.q_batch;
    const float base = p.a.scale * 1.4426950408889634f * (F8 ? p.a.k_scale[kvh] : 1.0f);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const bool real = h < heads;
      const QT* row = q + (kvh * p.group + head0 + (real ? h : 0)) * p.a.q_head;
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
  for (int tile = first; tile < last; tile += kPagedWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    __syncwarp();
    load_tile(tile + (C::STAGES - 1) * kPagedWarps, stage_in, place);  // into the stage of the tile before this one
    place = look_up(tile + C::STAGES * kPagedWarps);
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
  for (int i = threadIdx.x; i < heads * (DP / 4); i += kPagedThreads) {
    const int h = i / (DP / 4), d = i % (DP / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) top = fmaxf(top, warp_ml[w * C::HEADS + h].x);
    float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      const float2 ml = warp_ml[w * C::HEADS + h];
      const float f = ml.x == top ? 1.0f : exp2f(ml.x - top);
      sum += ml.y * f;
      const float4 v = *reinterpret_cast<const float4*>(warp_o + (w * C::HEADS + h) * C::OROW + d);
      acc[0] += v.x * f;
      acc[1] += v.y * f;
      acc[2] += v.z * f;
      acc[3] += v.w * f;
    }
    if (d >= D) continue;
    const int64_t row = static_cast<int64_t>(b) * p.a.q_heads + kvh * p.group + head0 + h;
    if (p.cluster) {
      *reinterpret_cast<float4*>(block_o + h * C::OROW + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) block_ml[h] = make_float2(top, sum);
    } else if (used == 1) {
      store_out(h, d, acc, sum);
    } else {
      *reinterpret_cast<float4*>(p.part_o + (row * p.splits + split) * D + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (d == 0) p.part_ml[row * p.splits + split] = make_float2(top, sum);
    }
  }
  if (p.cluster) {
    // the blocks of the cluster share out the outputs and read each other's sums, in the order of the splits
    cluster_arrive_wait();
    const uint32_t o_base = smem_u32(block_o), ml_base = smem_u32(block_ml);
    for (int i = static_cast<int>(cluster_cta_rank()) * kPagedThreads + threadIdx.x; i < heads * (DP / 4); i += p.splits * kPagedThreads) {
      const int h = i / (DP / 4), d = i % (DP / 4) * 4;
      if (d >= D) continue;
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
      store_out(h, d, acc, sum);
    }
    cluster_arrive_wait();  // nobody leaves while its sums are read
  }
}

// The splits of one query head, in order.  One block a head: its warps take every kJoinWarps-th split, a lane four outputs, and are
// added up in turn.
constexpr int kJoinWarps = 8;
template <typename QT>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const __grid_constant__ PagedParams p, bool f8) {
  __shared__ float warp_top[kJoinWarps], warp_sum[kJoinWarps];
  __shared__ float4 warp_o[kJoinWarps][32];
  const int64_t row = blockIdx.x;
  const int b = static_cast<int>(row / p.a.q_heads), h = static_cast<int>(row % p.a.q_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = lane * 4, D = p.a.head_dim;
  const Visible vis = visible_keys(sequence_length(p, b, false), p.a.window, p.a.sinks);
  const int tiles = (vis.n + kTileKeys - 1) / kTileKeys;
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
  if (warp != 0 || d >= D) return;
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
  *reinterpret_cast<uint2*>(static_cast<QT*>(p.a.out) + row * D + d) = outputs4<bf16>(acc, sum, f8 ? p.a.v_scale[h / p.group] : 1.0f);
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
static Splits choose_splits(const qlin_paged_attention_args& a, int head_blocks) {
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
static int heads_per_block(int group) { return group <= 8 ? 8 : 16; }

static int check_paged(const qlin_paged_attention_args* a) {
  if (a == nullptr) return fail(QLIN_ERR_NULL, "qlin_paged_attention: args is NULL");
  if (a->batch < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads != 0)
    return fail(QLIN_ERR_BAD_SHAPE, "qlin_paged_attention: q_heads must be a multiple of kv_heads");
  if (a->page_size < 1 || a->num_pages < 0 || a->max_pages < 0) return fail(QLIN_ERR_BAD_SHAPE, "qlin_paged_attention: bad cache dimensions");
  if (!(a->scale > 0.0f) || a->scale > 3.0e38f) return fail(QLIN_ERR_UNSUPPORTED, "qlin_paged_attention: scale must be positive and finite");
  if (static_cast<int64_t>(a->max_pages) * a->page_size > (1 << 30)) return fail(QLIN_ERR_TOO_LARGE, "qlin_paged_attention: at most 2^30 keys a sequence");
  if (a->dtype != QLIN_DT_F16 && a->dtype != QLIN_DT_BF16) return fail(QLIN_ERR_BAD_DTYPE, "qlin_paged_attention: q must be fp16 or bf16");
  if (a->cache_dtype != a->dtype && a->cache_dtype != QLIN_DT_F8E4M3) return fail(QLIN_ERR_BAD_DTYPE, "qlin_paged_attention: the cache must have the type of q, or e4m3");
  const int step = a->cache_dtype == QLIN_DT_F8E4M3 ? 16 : 8;
  if (a->head_dim < step || a->head_dim % step != 0 || a->head_dim > 128)
    return fail(QLIN_ERR_BAD_SHAPE, "qlin_paged_attention: head_dim must be a multiple of %d up to 128", step);
  const int head_blocks = (a->q_heads / a->kv_heads + 7) / 8;
  if (static_cast<int64_t>(a->batch) * a->kv_heads * head_blocks > (1 << 24) || static_cast<int64_t>(a->batch) * a->q_heads > (1 << 28))
    return fail(QLIN_ERR_TOO_LARGE, "qlin_paged_attention: too many sequences and heads");
  return QLIN_OK;
}

template <typename QT, bool F8, int DP, int NT>
static int launch_paged(const PagedParams& p, cudaStream_t stream) {
  using C = PagedCfg<QT, F8, DP, NT>;
  const auto kernel = paged_kernel<QT, F8, DP, NT>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(QLIN_ERR_DEVICE, "device ordinal %d out of range", dev);
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return fail(QLIN_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  const unsigned blocks = static_cast<unsigned>(p.a.batch) * p.a.kv_heads * p.head_blocks * p.splits;
  cudaLaunchConfig_t main = {};
  main.gridDim = dim3(blocks, 1, 1);
  main.blockDim = dim3(kPagedThreads, 1, 1);
  main.dynamicSmemBytes = C::SMEM;
  main.stream = stream;
  cudaLaunchAttribute size[1];
  size[0].id = cudaLaunchAttributeClusterDimension;
  size[0].val.clusterDim.x = static_cast<unsigned>(p.cluster ? p.splits : 1);
  size[0].val.clusterDim.y = size[0].val.clusterDim.z = 1;
  main.attrs = size;
  main.numAttrs = p.cluster ? 1 : 0;
  const cudaError_t launched = cudaLaunchKernelEx(&main, kernel, p);
  if (launched != cudaSuccess) {
    cudaGetLastError();
    return fail(QLIN_ERR_LAUNCH, "qlin_paged_attention: %s", cudaGetErrorString(launched));
  }
  if (p.splits > 1 && !p.cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.a.batch) * p.a.q_heads, 1, 1);
    cfg.blockDim = dim3(kJoinWarps * 32, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_join_kernel<QT>, p, F8);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(QLIN_ERR_LAUNCH, "qlin_paged_attention: %s", cudaGetErrorString(e));
    }
  }
  return QLIN_OK;
}
template <typename QT, bool F8>
static int pick_paged(const PagedParams& p, cudaStream_t s) {
  const bool wide = heads_per_block(p.group) == 16;
  if (p.a.head_dim <= 64) return wide ? launch_paged<QT, F8, 64, 2>(p, s) : launch_paged<QT, F8, 64, 1>(p, s);
  return wide ? launch_paged<QT, F8, 128, 2>(p, s) : launch_paged<QT, F8, 128, 1>(p, s);
}

}  // namespace qlin

extern "C" int64_t qlin_paged_attention_workspace_bytes(const qlin_paged_attention_args* a) {
  using namespace qlin;
  const int rc = check_paged(a);
  if (rc != QLIN_OK) return rc;
  if (a->batch == 0) return 0;
  const int group = a->q_heads / a->kv_heads;
  const Splits splits = choose_splits(*a, (group + heads_per_block(group) - 1) / heads_per_block(group));
  if (splits.n == 1 || splits.cluster) return 0;
  const int64_t rows = static_cast<int64_t>(a->batch) * a->q_heads * splits.n;
  return rows * a->head_dim * 4 + rows * 8;
}

extern "C" int qlin_paged_attention(const qlin_paged_attention_args* a, void* stream) {
  using namespace qlin;
  const int rc = check_paged(a);
  if (rc != QLIN_OK) return rc;
  if (a->batch == 0) return QLIN_OK;
  const bool f8 = a->cache_dtype == QLIN_DT_F8E4M3;
  if (a->q == nullptr || a->out == nullptr || a->lens == nullptr) return fail(QLIN_ERR_NULL, "qlin_paged_attention: q, out or lens is NULL");
  if (a->max_pages > 0 && a->num_pages > 0 && (a->k_pages == nullptr || a->v_pages == nullptr || a->block_table == nullptr))
    return fail(QLIN_ERR_NULL, "qlin_paged_attention: k_pages, v_pages or block_table is NULL");
  if (f8 && (a->k_scale == nullptr || a->v_scale == nullptr)) return fail(QLIN_ERR_NULL, "qlin_paged_attention: an e4m3 cache needs k_scale and v_scale");
  const int cs = f8 ? 1 : 2;
  if (!aligned16(a->q) || !aligned16(a->out) || !aligned16(a->k_pages) || !aligned16(a->v_pages) || a->q_batch * 2 % 16 != 0 || a->q_head * 2 % 16 != 0 ||
      a->page_stride * cs % 16 != 0 || a->head_stride * cs % 16 != 0 || a->slot_stride * cs % 16 != 0)
    return fail(QLIN_ERR_BAD_ALIGN, "qlin_paged_attention: every row of q, out and the cache must start on 16 bytes");
  PagedParams p;
  p.a = *a;
  p.group = a->q_heads / a->kv_heads;
  p.head_blocks = (p.group + heads_per_block(p.group) - 1) / heads_per_block(p.group);
  const Splits splits = choose_splits(*a, p.head_blocks);
  p.splits = splits.n;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a->page_size == 1 << i) p.page_shift = i;
  p.cluster = splits.cluster;
  p.part_o = nullptr;
  p.part_ml = nullptr;
  if (p.splits > 1 && !p.cluster) {
    if (a->workspace == nullptr) return fail(QLIN_ERR_NULL, "qlin_paged_attention: workspace is NULL");
    if (!aligned16(a->workspace)) return fail(QLIN_ERR_BAD_ALIGN, "qlin_paged_attention: workspace must start on 16 bytes");
    p.part_o = static_cast<float*>(a->workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<int64_t>(a->batch) * a->q_heads * p.splits * a->head_dim);
  }
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == QLIN_DT_BF16) return f8 ? pick_paged<__nv_bfloat16, true>(p, s) : pick_paged<__nv_bfloat16, false>(p, s);
  return f8 ? pick_paged<__half, true>(p, s) : pick_paged<__half, false>(p, s);
}
