// qlin_lora: low-rank adapters of many requests added to the output of a projection that they share.
//
//   v = x[t] a[i]^T  (rank numbers),   y[t] += scale[i] v b[i]^T       for every row t of adapter i
//
// What bounds it: HBM, x and the adapters read once, y read and written once; a row of x against an adapter of rank 16 is 16 operations a byte.
// One launch does both products.  A tile is 16 or more rows of one adapter, wherever they stand; its block (or cluster of blocks, where tiles are few)
// shares out the width of x for v and the columns of y afterwards, warp by warp, and joins the parts of v in shared memory in between, in order.
//
// Both products are m16n8k16 with the rows as the tile's rows.  No lane needs what another one loads, but for v: the order of the terms of a product is free, so a lane
// takes 16 bytes of a row of x and 16 of a row of a where the instruction wants four pairs of terms, and the columns of y are dealt so that
// the four n = 8 products of 32 columns leave a lane with 16 bytes of y in a row.  Asynchronous copies bring them to places of the lane's own in shared memory, several
// steps ahead; a lane waits for its own copies only.  Rows of 128 (tcgen05) would not make the loads faster.
//
// Measured (device time): 8 prompts of 2048 rows, rank 16, 4096 -> 4096 in bf16 80 us, 5.0 TB/s, 0.77 of the copy rate (registers instead of the copies 86, a tile of 16 rows 104 and
// of 64 82); 1999 rows of rank 64, 14336 -> 4096 in fp16 32 to 36 us, 2.2 TB/s: 112 blocks of 64 rows that go through 1.2 MB each, a step's copies and products behind one another; 1999 rows of
// rank 128, 4096 -> 4096 in bf16 45 us; 64 rows of 16 adapters, rank 16, 4096 -> 14336 9 us; one row 5.9: the latency of starts, rows, x, the join of v in the cluster, and y behind one another.
//
// v goes into the second product as two 16-bit numbers whose sum has 16 (bf16) or 22 (fp16) of its bits; in fp16 a row of v is brought to
// 1 <= max < 2 first, by a power of two that comes back with the scale, since its sums may leave fp16's range where y does not.
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qlin_internal.h"
#include "qlin_ptx.cuh"

namespace qlin {

constexpr int kLoraWarps = 8;
constexpr int kLoraThreads = kLoraWarps * 32;
constexpr int kMostCluster = 8;

struct LoraParams {
  qlin_lora_args a;
  int32_t cluster;  // blocks of a tile
};

template <typename T, int R16, int MT>
struct LoraCfg {
  static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int RP = 16 * R16;        // the rank, padded
  static constexpr int ROWS = 16 * MT;
  static constexpr int PITCH = RP + 4;       // floats of a row of v
  static constexpr int PITCH16 = RP + 8;     // 16-bit numbers of a row of v
  static constexpr int QUADS = RP >= 32 ? RP / 32 : 1;  // 16-byte (8-byte for rank 16) pieces of a row of b a lane has
  static constexpr bool HOLD = R16 * MT <= 8;           // v stays in registers while the columns go by
  // A stage of a warp: 32 terms of the tile's rows of x and of the rows of a, or 32 columns of y and the rows of b behind them.  Stages for two blocks
  // an SM, or for one where they are large.
  static constexpr int B_BYTES = R16 == 1 ? 4 * 256 : 4 * QUADS * 512;
  static constexpr int FIRST = (2 * MT + 2 * R16) * 512, SECOND = 2 * MT * 512 + B_BYTES;
  static constexpr int STAGE = FIRST > SECOND ? FIRST : SECOND;
  static constexpr int BLOCKS = STAGE <= 4096 ? 2 : 1;
  static constexpr int STAGES = STAGE <= 2048 ? 6 : STAGE <= 4096 ? 3 : STAGE <= 6144 ? 4 : STAGE <= 8192 ? 3 : 2;
  static constexpr int RING = kLoraWarps * STAGES * STAGE;
  static constexpr int PARTS = RING;                       // [warps][rows][PITCH], in the room of the stages where those are not needed yet
  static constexpr int PART_BYTES = kLoraWarps * ROWS * PITCH * 4;
  static constexpr bool APART = RING + PART_BYTES + ROWS * PITCH * 4 + 4 * ROWS * PITCH16 + ROWS * 4 <= (BLOCKS == 2 ? 114 : 226) * 1024;
  static constexpr int BLOCK_V = APART ? PARTS + PART_BYTES : PART_BYTES;  // [rows][PITCH]: the block's, then everybody's
  static constexpr int V_END = BLOCK_V + ROWS * PITCH * 4;
  static constexpr int V16 = APART || V_END > RING ? V_END : RING;  // [2][rows][PITCH16]
  static constexpr int BACK = V16 + 2 * ROWS * PITCH16 * 2;  // [rows]
  static constexpr int SMEM = BACK + ROWS * 4;
  static_assert(SMEM <= (BLOCKS == 2 ? 114 : 227) * 1024, "fits");
};

// Adapter and first listed row of a tile; adapter -1: there is no such tile.  Every warp looks for itself.
struct LoraTile {
  int adapter, first, count;
};
__device__ __forceinline__ LoraTile lora_tile(const LoraParams& p, int tile, int rows, bool report) {
  const int lane = threadIdx.x & 31;
  int passed = 0;
  for (int i0 = 0; i0 < p.a.adapters; i0 += 32) {
    const int i = i0 + lane;
    int s0 = 0, n = 0;
    bool bad = false;
    if (i < p.a.adapters) {
      s0 = p.a.starts[i];
      const int s1 = p.a.starts[i + 1];
      bad = s0 < 0 || s1 < s0 || s1 > p.a.listed || (i == 0 && s0 != 0);
      n = bad ? 0 : s1 - s0;
    }
    if (report && bad && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
    const int tiles = (n + rows - 1) / rows;
    int upto = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += other;
    }
    const int here = __shfl_sync(0xffffffffu, upto, 31);
    if (tile < passed + here && !report) {
      const int owner = __ffs(__ballot_sync(0xffffffffu, tile < passed + upto)) - 1;
      const int within = (tile - passed - (__shfl_sync(0xffffffffu, upto - tiles, owner))) * rows;
      return LoraTile{i0 + owner, __shfl_sync(0xffffffffu, s0, owner) + within, min(rows, __shfl_sync(0xffffffffu, n, owner) - within)};
    }
    passed += here;
  }
  return LoraTile{-1, 0, 0};
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
  if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Adds 0 times two numbers: a zero stays one unless they, or what was added before, are infinite or NaN.
template <bool BF16>
__device__ __forceinline__ uint32_t zero_unless_infinite(uint32_t w, uint32_t before) {
  uint32_t r;
  if constexpr (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(before));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(before));
  return r;
}

template <typename T, int R16, int MT>
__global__ void __launch_bounds__(kLoraThreads, (LoraCfg<T, R16, MT>::BLOCKS)) lora_kernel(const __grid_constant__ LoraParams p) {
  using C = LoraCfg<T, R16, MT>;
  extern __shared__ __align__(16) uint8_t smem[];
  float* parts = reinterpret_cast<float*>(smem + (C::APART ? C::PARTS : 0));
  float* block_v = reinterpret_cast<float*>(smem + C::BLOCK_V);
  T* v16 = reinterpret_cast<T*>(smem + C::V16);
  float* back = reinterpret_cast<float*>(smem + C::BACK);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % p.cluster;
  const LoraTile tile = lora_tile(p, blockIdx.x / p.cluster, C::ROWS, false);
  if (tile.adapter < 0) {  // the whole cluster
    if (blockIdx.x == 0 && warp == 0) lora_tile(p, 0x7fffffff, C::ROWS, true);
    return;
  }
  const int share = rank * kLoraWarps + warp, shares = p.cluster * kLoraWarps;  // of the width, then of the columns

  // the rows g and g + 8 of each sixteen that this lane loads and stores
  const T* x_row[2 * MT];
  T* y_row[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const int at = 8 * i + g;
    int row = at < tile.count ? p.a.rows[tile.first + at] : -1;
    if (at < tile.count && (row < 0 || row >= p.a.tokens)) {
      if (p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
      row = -1;
    }
    x_row[i] = row < 0 ? nullptr : static_cast<const T*>(p.a.x) + row * p.a.x_row;
    y_row[i] = row < 0 ? nullptr : static_cast<T*>(p.a.y) + row * p.a.y_row;
  }
  // ---------------------------------------------------------------- copies: this warp's steps of 32 terms, then its steps of 32 columns
  const T* a = static_cast<const T*>(p.a.a) + tile.adapter * p.a.a_adapter;
  const T* b = static_cast<const T*>(p.a.b) + tile.adapter * p.a.b_adapter;
  const int terms = (p.a.width + 31) / 32, columns = (p.a.out + 31) / 32;
  const int terms_each = (terms + shares - 1) / shares, columns_each = (columns + shares - 1) / shares;
  const int term0 = share * terms_each, column0 = share * columns_each;
  const int n1 = max(0, min(terms_each, terms - term0)), n2 = max(0, min(columns_each, columns - column0));
  const uint32_t ring = smem_u32(smem) + warp * C::STAGES * C::STAGE + lane * 16;
  const auto copy = [&](uint32_t to, const void* from, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(real ? from : p.a.x), "r"(real ? 16 : 0) : "memory");
  };
  const auto copy_terms = [&](int i, uint32_t to) {
    const int k = (term0 + i) * 32 + 8 * t;
    const bool in = k < p.a.width;
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) copy(to + j * 512, x_row[j] + k, in && x_row[j] != nullptr);
#pragma unroll
    for (int j = 0; j < 2 * R16; ++j) copy(to + (2 * MT + j) * 512, a + (8 * j + g) * p.a.a_row + k, in && 8 * j < p.a.rank);
  };
  const auto copy_columns = [&](int i, uint32_t to) {
    const int n0 = (column0 + i) * 32;
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) copy(to + j * 512, y_row[j] + n0 + 8 * t, y_row[j] != nullptr && n0 + 8 * t < p.a.out);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + 8 * (g >> 1) + 2 * q + (g & 1);
      if constexpr (R16 == 1) {
        const bool real = n < p.a.out && 4 * t < p.a.rank;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to - lane * 8 + 2 * MT * 512 + q * 256), "l"(real ? static_cast<const void*>(b + n * p.a.b_row + 4 * t) : p.a.x),
                     "r"(real ? 8 : 0)
                     : "memory");
      } else {
#pragma unroll
        for (int c = 0; c < C::QUADS; ++c) copy(to + (2 * MT + q * C::QUADS + c) * 512, b + n * p.a.b_row + 32 * c + 8 * t, n < p.a.out && 32 * c + 8 * t < p.a.rank);
      }
    }
  };
  const auto stage_of = [&](int i) { return ring + static_cast<uint32_t>(i % C::STAGES) * C::STAGE; };
  // The i-th copies of the warp.  Where the warps' parts of v lie over the stages, those of the columns begin behind the join.
  const int first_total = C::APART ? n1 + n2 : n1;
  const auto issue = [&](int i, int total) {
    if (i < total) {
      if (i < n1) copy_terms(i, stage_of(i));
      else copy_columns(i - n1, stage_of(i));
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const auto held = [&](uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
  };
#pragma unroll 1
  for (int i = 0; i < C::STAGES - 1; ++i) issue(i, first_total);

  // ---------------------------------------------------------------- v, this warp's share of the terms
  float acc[MT][2 * R16][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < 2 * R16; ++j) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.0f;
#pragma unroll 1
  for (int i = 0; i < n1; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    const uint32_t at = stage_of(i);
    uint4 xv[2 * MT];
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) xv[j] = held(at + j * 512);
#pragma unroll
    for (int j = 0; j < 2 * R16; ++j) {
      const uint4 av = held(at + (2 * MT + j) * 512);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        mma16816<C::BF16>(acc[m][j], xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y, av.x, av.y);
        mma16816<C::BF16>(acc[m][j], xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w, av.z, av.w);
      }
    }
    issue(i + C::STAGES - 1, first_total);  // over the step before this one, which has been read
  }
  if constexpr (!C::APART) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < 2 * R16; ++j) {
      float* to = parts + (warp * C::ROWS + 16 * m + g) * C::PITCH + 8 * j + 2 * t;
      *reinterpret_cast<float2*>(to) = make_float2(acc[m][j][0], acc[m][j][1]);
      *reinterpret_cast<float2*>(to + 8 * C::PITCH) = make_float2(acc[m][j][2], acc[m][j][3]);
    }

  // ---------------------------------------------------------------- v of all warps, then of all blocks, in order
  __syncthreads();
  for (int i = threadIdx.x; i < C::ROWS * C::RP / 4; i += kLoraThreads) {
    const int row = i / (C::RP / 4), c = i % (C::RP / 4) * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kLoraWarps; ++w) {
      const float4 one = *reinterpret_cast<const float4*>(parts + (w * C::ROWS + row) * C::PITCH + c);
      sum = make_float4(sum.x + one.x, sum.y + one.y, sum.z + one.z, sum.w + one.w);
    }
    *reinterpret_cast<float4*>(block_v + row * C::PITCH + c) = sum;
  }
  float* v = block_v;
  if (p.cluster > 1) {
    cluster_arrive_wait();
    v = parts;  // the warps' parts are no longer needed
    const uint32_t base = smem_u32(block_v);
    for (int i = threadIdx.x; i < C::ROWS * C::RP / 4; i += kLoraThreads) {
      const int row = i / (C::RP / 4), c = i % (C::RP / 4) * 4;
      float4 one[kMostCluster];
#pragma unroll
      for (int o = 0; o < kMostCluster; ++o) one[o] = o < p.cluster ? ld_cluster_f4(base + (row * C::PITCH + c) * 4, o) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float4 sum = one[0];
#pragma unroll
      for (int o = 1; o < kMostCluster; ++o) sum = make_float4(sum.x + one[o].x, sum.y + one[o].y, sum.z + one[o].z, sum.w + one[o].w);
      *reinterpret_cast<float4*>(v + row * C::PITCH + c) = sum;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  __syncthreads();
  const float scale = p.a.scale[tile.adapter];
  for (int row = warp; row < C::ROWS; row += kLoraWarps) {
    float up = 1.0f, down = 1.0f;
    if constexpr (!C::BF16) {
      float top = 0.0f;
      for (int c = lane; c < C::RP; c += 32) {
        const float one = fabsf(v[row * C::PITCH + c]);
        top = one < INFINITY ? fmaxf(top, one) : top;  // an infinity needs no room, those beside it do
      }
      const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
      const int e = static_cast<int>(bits >> 23);
      if (e > 0 && e < 254) {  // 2^-(e - 127) and its inverse are normal numbers
        up = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
        down = __uint_as_float(static_cast<uint32_t>(e) << 23);
      }
    }
    if (lane == 0) back[row] = down * scale;
    for (int c = 2 * lane; c < C::RP; c += 64) {
      const float a0 = v[row * C::PITCH + c] * up, a1 = v[row * C::PITCH + c + 1] * up;
      uint32_t hi = pack_pair<C::BF16>(a0, a1);
      // not to zero, so that an infinite weight of b meets a number: the least one, which the second part takes off again
      if (a0 != 0.0f && (hi & 0x7fffu) == 0u) hi |= 1u;
      if (a1 != 0.0f && (hi & 0x7fff0000u) == 0u) hi |= 0x10000u;
      const float2 h = unpack_pair<C::BF16>(hi);
      // what is infinite or NaN is so in the first part alone
      const uint32_t lo = pack_pair<C::BF16>(isfinite(h.x) ? a0 - h.x : 0.0f, isfinite(h.y) ? a1 - h.y : 0.0f);
      *reinterpret_cast<uint32_t*>(v16 + row * C::PITCH16 + c) = hi;
      *reinterpret_cast<uint32_t*>(v16 + (C::ROWS + row) * C::PITCH16 + c) = lo;
    }
  }
  __syncthreads();

  // ---------------------------------------------------------------- y
  float factor[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) factor[i] = back[8 * i + g];
  const auto part_of_v = [&](int part, int m, int h, int c) {  // of row g or g + 8 of the sixteen
    const T* at = v16 + (part * C::ROWS + 16 * m + 8 * h + g) * C::PITCH16;
    if constexpr (R16 == 1) {
      const uint2 w = *reinterpret_cast<const uint2*>(at + 4 * t);
      return make_uint4(w.x, w.y, 0u, 0u);
    } else {
      return *reinterpret_cast<const uint4*>(at + 32 * c + 8 * t);
    }
  };
  uint4 vf[C::HOLD ? 2 : 1][C::HOLD ? MT : 1][2][C::QUADS];
  if constexpr (C::HOLD) {
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < C::QUADS; ++c) vf[part][m][h][c] = part_of_v(part, m, h, c);
  }
  const auto leave = [&]() {  // nobody leaves, or copies over its part of v, while that is read
    if (p.cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  };
  if constexpr (!C::APART) {
    leave();
    __syncthreads();  // v has been read
#pragma unroll 1
    for (int i = 0; i < C::STAGES - 1; ++i) issue(n1 + i, n1 + n2);
  }
#pragma unroll 1
  for (int i = n1; i < n1 + n2; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
    const uint32_t at = stage_of(i);
    const auto weights = [&](int q, int c) {
      uint4 w = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (R16 == 1) {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w.x), "=r"(w.y) : "r"(at - lane * 8 + 2 * MT * 512 + q * 256) : "memory");
      } else {
        w = held(at + (2 * MT + q * C::QUADS + c) * 512);
      }
      return w;
    };
    uint4 bv[4][C::QUADS];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int c = 0; c < C::QUADS; ++c) bv[q][c] = weights(q, c);
    // The second part of v has any sign, or is zero: where it meets an infinite weight the first part alone says what becomes of it.  To look for one takes 0.1 to 0.4 us a call
    // (64 rows of 16 adapters 8.7 -> 9.0, 8 prompts of 2048 rows 78.6 -> 78.8, of rank 32 83.1 -> 85.5); a look at the sums instead, which waits for them, up to 4.
    uint32_t nan[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int c = 0; c < C::QUADS; ++c) {
        nan[q] = zero_unless_infinite<C::BF16>(bv[q][c].y, zero_unless_infinite<C::BF16>(bv[q][c].x, nan[q]));
        if constexpr (R16 > 1) nan[q] = zero_unless_infinite<C::BF16>(bv[q][c].w, zero_unless_infinite<C::BF16>(bv[q][c].z, nan[q]));
      }
    const bool odd = __any_sync(0xffffffffu, ((nan[0] | nan[1] | nan[2] | nan[3]) & 0x7fff7fffu) != 0u);
    const int n = (column0 + i - n1) * 32 + 8 * t;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float o[4][4];
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q][0] = o[q][1] = o[q][2] = o[q][3] = 0.0f;
#pragma unroll
      for (int part = 1; part >= 0; --part)  // the small part first
#pragma unroll
        for (int c = 0; c < C::QUADS; ++c) {
          const uint4 r0 = C::HOLD ? vf[part % (C::HOLD ? 2 : 1)][m % (C::HOLD ? MT : 1)][0][c] : part_of_v(part, m, 0, c);
          const uint4 r1 = C::HOLD ? vf[part % (C::HOLD ? 2 : 1)][m % (C::HOLD ? MT : 1)][1][c] : part_of_v(part, m, 1, c);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            mma16816<C::BF16>(o[q], r0.x, r1.x, r0.y, r1.y, bv[q][c].x, bv[q][c].y);
            if constexpr (R16 > 1) mma16816<C::BF16>(o[q], r0.z, r1.z, r0.w, r1.w, bv[q][c].z, bv[q][c].w);
          }
        }
      if (odd) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float first[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < C::QUADS; ++c) {
            const uint4 w = weights(q, c);
            const uint4 r0 = C::HOLD ? vf[0][m % (C::HOLD ? MT : 1)][0][c] : part_of_v(0, m, 0, c);
            const uint4 r1 = C::HOLD ? vf[0][m % (C::HOLD ? MT : 1)][1][c] : part_of_v(0, m, 1, c);
            mma16816<C::BF16>(first, r0.x, r1.x, r0.y, r1.y, w.x, w.y);
            if constexpr (R16 > 1) mma16816<C::BF16>(first, r0.z, r1.z, r0.w, r1.w, w.z, w.w);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) o[q][e] = o[q][e] != o[q][e] ? first[e] : o[q][e];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 y4 = held(at + (2 * m + h) * 512);
        const uint32_t old[4] = {y4.x, y4.y, y4.z, y4.w};
        uint32_t sum[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 y = unpack_pair<C::BF16>(old[q]);
          sum[q] = pack_pair<C::BF16>(fmaf(o[q][2 * h], factor[2 * m + h], y.x), fmaf(o[q][2 * h + 1], factor[2 * m + h], y.y));
        }
        if (y_row[2 * m + h] != nullptr && n < p.a.out) *reinterpret_cast<uint4*>(y_row[2 * m + h] + n) = make_uint4(sum[0], sum[1], sum[2], sum[3]);
      }
    }
    issue(i + C::STAGES - 1, n1 + n2);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if constexpr (C::APART) leave();
  if (blockIdx.x == 0 && warp == 0) lora_tile(p, 0x7fffffff, C::ROWS, true);
}

// Sixteens of rows of a tile: as many as an adapter has rows for on average, and no more than leave a cluster of blocks for every eighth SM.
static int64_t tiles_at_most(const qlin_lora_args& a, int rows) {
  // every adapter has at most one tile that is not full, every tile a row
  const int64_t most = static_cast<int64_t>(a.listed) / rows + a.adapters;
  return most < a.listed ? most : a.listed;
}
static int sixteens(const qlin_lora_args& a, int most) {
  int mt = 1;
  while (mt < most && a.listed / a.adapters >= 32 * mt && tiles_at_most(a, 32 * mt) * kMostCluster >= sm_count()) mt *= 2;
  return mt;
}

template <typename T, int R16, int MT>
static int launch_lora(LoraParams p, cudaStream_t stream) {
  using C = LoraCfg<T, R16, MT>;
  const auto kernel = lora_kernel<T, R16, MT>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(QLIN_ERR_DEVICE, "device ordinal %d out of range", dev);
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return fail(QLIN_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    configured[dev] = true;
  }
  const int64_t tiles = tiles_at_most(p.a, C::ROWS);
  p.cluster = 1;  // as many blocks a tile as are resident at once: a second wave costs more than they save (1999 rows of rank 64 36 us in fours, 74 in eights)
  while (p.cluster < kMostCluster && tiles * p.cluster * 2 <= static_cast<int64_t>(C::BLOCKS) * sm_count()) p.cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles) * p.cluster, 1, 1);
  cfg.blockDim = dim3(kLoraThreads, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(QLIN_ERR_LAUNCH, "qlin_lora: %s", cudaGetErrorString(e));
  }
  return QLIN_OK;
}
template <typename T, int R16, int MOST>
static int pick_rows(const LoraParams& p, cudaStream_t s) {
  const int mt = sixteens(p.a, MOST);
  if constexpr (MOST >= 4) {
    if (mt == 4) return launch_lora<T, R16, 4>(p, s);
  }
  if (mt == 2) return launch_lora<T, R16, 2>(p, s);
  return launch_lora<T, R16, 1>(p, s);
}
template <typename T>
static int pick_lora(const LoraParams& p, cudaStream_t s) {
  if (p.a.rank <= 16) return pick_rows<T, 1, 2>(p, s);
  if (p.a.rank <= 32) return pick_rows<T, 2, 2>(p, s);
  if (p.a.rank <= 64) return pick_rows<T, 4, 4>(p, s);
  return pick_rows<T, 8, 2>(p, s);
}

}  // namespace qlin

extern "C" int qlin_lora(const qlin_lora_args* a, void* stream) {
  using namespace qlin;
  if (a == nullptr) return fail(QLIN_ERR_NULL, "qlin_lora: args is NULL");
  if (a->tokens < 0 || a->listed < 0 || a->adapters < 0 || a->width < 0 || a->out < 0 || a->rank < 1) return fail(QLIN_ERR_BAD_SHAPE, "qlin_lora: a dimension is negative");
  if (a->rank > 128 || a->rank % 8 != 0 || a->width % 8 != 0 || a->out % 8 != 0)
    return fail(QLIN_ERR_BAD_SHAPE, "qlin_lora: width, out and rank must be multiples of 8, rank at most 128");
  if (a->listed > (1 << 27)) return fail(QLIN_ERR_TOO_LARGE, "qlin_lora: at most 2^27 rows");
  if (a->dtype != QLIN_DT_F16 && a->dtype != QLIN_DT_BF16) return fail(QLIN_ERR_BAD_DTYPE, "qlin_lora: x, a, b and y must be fp16 or bf16");
  if (a->listed == 0 || a->adapters == 0 || a->out == 0 || a->width == 0) return QLIN_OK;
  if (a->x == nullptr || a->y == nullptr || a->a == nullptr || a->b == nullptr || a->rows == nullptr || a->starts == nullptr || a->scale == nullptr)
    return fail(QLIN_ERR_NULL, "qlin_lora: x, y, a, b, rows, starts or scale is NULL");
  if (!aligned16(a->x) || !aligned16(a->y) || !aligned16(a->a) || !aligned16(a->b) || a->x_row % 8 != 0 || a->y_row % 8 != 0 || a->a_adapter % 8 != 0 ||
      a->a_row % 8 != 0 || a->b_adapter % 8 != 0 || a->b_row % 8 != 0)
    return fail(QLIN_ERR_BAD_ALIGN, "qlin_lora: every row of x, y, a and b must start on 16 bytes");
  const LoraParams p{*a, 1};
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return a->dtype == QLIN_DT_BF16 ? pick_lora<__nv_bfloat16>(p, s) : pick_lora<__half>(p, s);
}
