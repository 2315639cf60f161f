// qlin_prompt_attention: attention of packed prompts under a causal mask, a sliding window and first tokens that stay visible.
//
//   o_i = sum_j w_j v_j / sum_j w_j,   w_j = 2^(x_j - r),   x_j = q_i.k_j scale log2(e),   j over the keys that i sees
//
// for any r; r follows the running maximum.  A persistent block has two tiles of 128 rows of one kv head and goes over tiles of 128
// keys.  A tile's rows are 128 / G queries times the G query heads that share the kv head, so grouped heads share each load and a
// tile spans few positions, which keeps what the mask throws away small.  S = Q K^T on tcgen05 with both operands in shared memory, one
// thread for each row of 128 logits in tensor memory, the weights back to tensor memory over their logits in 16 bits, O += P V
// with the weights as the operand from there.  At head_dim 128 tensor memory is full: two S of 128 columns, two O of head_dim.  The tiles take turns, one in the softmax
// while the other is in the tensor core.
//
// What bounds it: that chain.  A turn (two tiles against 128 keys) is 2048 cycles of tensor core and 2048 of exponentials (two
// tiles x 128 a thread x 8 cycles), and takes about 4100: the exponentials of a tile and its products follow one another, and the
// third pair of buffers that would let a tile's next logits be made meanwhile does not fit (at 64 it would).  The operands that the products
// read from shared memory and the tiles that arrive there are some 256 KB a turn, about 2048 cycles more beside them.  Measured (device time): 8 x 2048, 32 + 8 heads
// of 128 in bf16 280 us, 980 TFLOP/s = 0.60 of the measured rate; 1 x 8191 under a window of 2048 with four first keys 242 us,
// 995; 5 x up to 333 after 77, 12 heads of 64 in fp16 13 us, four turns behind a cold start.  With exponentials, maxima and masks left
// out the first two would take 252 and 204: what else is in a turn is loads and stores of tensor memory, conversions and hand-overs.
// Tried and slower, 8 x 2048 in us at the time: a warp for each tile's products 340 against 290 (both tiles fall into step and wait
// together), the same with the tensor core handed from one to the other 299, all of a tile's weights in one hand-over 307, logits read
// twice instead of held in registers 317, half of a tile's weights ahead of its maximum instead of a quarter 304.
#include <type_traits>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qlin_internal.h"
#include "qlin_ptx.cuh"

namespace qlin {

constexpr int kMostTokens = 1 << 30;

struct PromptParams {
  qlin_prompt_attention_args a;
  int32_t group;  // query heads per kv head
  int32_t tq;     // queries of a tile: its rows are tq queries times the group's heads
  int32_t units;  // pairs of tiles of the longest sequence
  float cl2;      // scale * log2(e)
};

// A sequence's rows of q and k; bad: the offsets do not fit the tensors or each other.
struct Sequence {
  int q0, n, k0, m;
  bool bad;
};
__device__ __forceinline__ Sequence sequence_of(const PromptParams& p, int b) {
  const int q0 = p.a.cu_q[b], q1 = p.a.cu_q[b + 1], k0 = p.a.cu_k[b], k1 = p.a.cu_k[b + 1];
  Sequence s{q0, q1 - q0, k0, k1 - k0, false};
  s.bad = q0 < 0 || q1 < q0 || q1 > p.a.tokens_q || k0 < 0 || k1 < k0 || k1 > p.a.tokens_k || q1 - q0 > p.a.max_q;
  if (b == 0) s.bad |= q0 != 0 || k0 != 0;
  if (b == p.a.batch - 1) s.bad |= q1 != p.a.tokens_q || k1 != p.a.tokens_k;
  return s;
}

template <typename T>
__device__ __forceinline__ float2 pair16(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

__device__ __forceinline__ uint32_t nans_of(float a, float b, float c, float d) {
  return (a != a ? 1u : 0u) | (b != b ? 2u : 0u) | (c != c ? 4u : 0u) | (d != d ? 8u : 0u);
}

// The visible keys of the query at a position: those under `first`, then `start` to the position itself.
struct Seen {
  int start, first, count;
};
__device__ __forceinline__ Seen seen_from(const PromptParams& p, int pos) {
  Seen s;
  s.start = p.a.window > 0 ? max(0, pos - p.a.window + 1) : 0;
  s.first = min(max(p.a.sinks, 0), s.start);
  s.count = pos < 0 ? 0 : s.first + pos + 1 - s.start;
  return s;
}

// ------------------------------------------------------------------------------------------------ tensor cores
constexpr int kRows = 128;        // rows of a tile of queries
constexpr int kKeys = 128;        // keys of a tile
constexpr int kSoftmaxWarps = 8;  // four a tile of queries, a thread a row
constexpr int kLoadWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1;
constexpr int kPromptThreads = (kSoftmaxWarps + 4) * 32;  // whole warpgroups: registers are handed over between them
// A block starts with 168 registers a thread (64,512 in all); the softmax warps take 216 each once the others have gone down to 72
// (64,512): a row of 128 logits stays in registers.
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
constexpr int kChunkBytes = 128 * 128;  // 128 rows of 64 elements, 128-byte swizzle
// The reference may lie this far (in powers of two) below the maximum.  Weights up to 2^8 are as exact in 16 bits as those up to 1;
// fp16 ones carry a factor of 2^6 on top, so that they stay below 2^14 and lose bits only under 2^-20 of the largest.
constexpr float kSlack = 8.0f;
constexpr int kSplitTiles = 10;

struct PromptAux {
  uint64_t q_full[2], q_empty[2], kv_full[8], kv_empty[8], s_full[2], p_full[2][2], o_full[2], drain;
  uint32_t tmem_base;
  int abort_flag;
};

template <typename T, int DP>
struct PromptCfg {
  static constexpr int CHUNKS = DP / 64;
  static constexpr int TILE_BYTES = CHUNKS * kChunkBytes;  // a tile of queries, keys or values
  static constexpr int STAGES = DP == 128 ? 4 : 8;         // tiles of keys or values in flight
  static constexpr int KV_OFFSET = 2 * TILE_BYTES;
  static constexpr int OUT_OFFSET = KV_OFFSET + STAGES * TILE_BYTES;  // 32 rows of 64 outputs for each softmax warp
  static constexpr int AUX_OFFSET = OUT_OFFSET + kSoftmaxWarps * 4096;
  // with a unit split over a cluster: a block's accumulators and (maximum, sum), over the tiles that are no longer needed
  static constexpr int PART_ML = 2 * kRows * DP * 4;
  static_assert(PART_ML + 2 * kRows * 8 <= OUT_OFFSET, "the sums fit the tiles' place");
  static __device__ __forceinline__ uint32_t part_o(int row, int piece) { return static_cast<uint32_t>(row * DP * 4 + ((piece ^ (row & 7)) << 4)); }
  static constexpr int SMEM_BYTES = AUX_OFFSET + static_cast<int>(sizeof(PromptAux));
  static constexpr float SHIFT = std::is_same<T, __half>::value ? 6.0f : 0.0f;
  // A weight is 2^(x cl2 - r) with r rounded and the product not, so half a unit of r's last place and more is in its exponent, the same for all
  // keys of a row.  From these references on (logits of 2.9e6 in fp16, 3.7e8 in bf16) that could carry weights out of 16 bits: rows that meet one are
  // computed again, with the difference taken first.
  static constexpr float LARGE_REF = std::is_same<T, __half>::value ? 0x1p22f : 0x1p29f;
  static constexpr uint32_t FMT = std::is_same<T, __half>::value ? 0u : 1u;
  static constexpr uint32_t IDESC_S = make_idesc(1u, FMT, kRows, kKeys);
  static constexpr uint32_t IDESC_O = make_idesc(1u, FMT, kRows, DP) | (1u << 16);  // V is read with its head dimension contiguous
};

__device__ __forceinline__ void prompt_load(uint64_t* bar, void* dst, const void* tmap, int32_t x, int32_t y, int32_t z) {
  asm volatile(
      "{\n\t"
      ".reg .pred pe;\n\t"
      "elect.sync _|pe, 0xffffffff;\n\t"
      "@pe cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%3, %4, %5}], [%0];\n\t"
      "}" ::"r"(smem_u32(bar)),
      "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void prompt_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile(
      "{\n\t"
      ".reg .pred pe;\n\t"
      "elect.sync _|pe, 0xffffffff;\n\t"
      "@pe mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t"
      "}" ::"r"(smem_u32(bar)),
      "r"(bytes)
      : "memory");
}
// A value that is the same in every lane, in a form that the compiler knows to be: with it in the loops' bounds the products are issued
// from uniform registers (8 x 2048: 304 us; by a single lane from ordinary ones 377).
__device__ __forceinline__ int uniform(int v) { return __reduce_max_sync(0xffffffffu, v); }
// A bounded wait of a whole warp for one barrier, or two, whose loop and answer are uniform too.
__device__ __forceinline__ bool uniform_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t* other = nullptr, uint32_t other_parity = 0) {
  uint64_t began = 0;
#pragma unroll 1
  for (uint32_t n = 0;; ++n) {
    bool done = mbar_try_wait(bar, parity);
    if (other != nullptr) done &= mbar_try_wait(other, other_parity);
    if (__all_sync(0xffffffffu, done)) return true;
    if (n < kSpinFast) continue;
    const uint64_t now = global_timer_ns();
    if (began == 0) began = now;
    if (__any_sync(0xffffffffu, *abort_flag != 0 || now - began > kWaitBudgetNs)) return false;
    __nanosleep(64);
  }
}
// Descriptors are built from their low words: start address in units of 16 bytes and leading offset.  The high words: 1024 bytes
// between groups of eight rows, version, 128-byte swizzle.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// Low word of a tile of values, [128 keys][64 elements] pieces 16 KB apart, the head dimension contiguous.
constexpr uint32_t kValuesLow = static_cast<uint32_t>(kChunkBytes >> 4) << 16;
constexpr uint32_t kRowsLow = 1u << 16;
// Four K = 16 steps; A from shared memory (two units of 16 bytes a step) and B likewise.  One elected lane issues.
__device__ __forceinline__ void mma4_ss(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred pe, pa, pt;\n\t"
      ".reg .b32 l;\n\t"
      ".reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t"
      "elect.sync _|pe, 0xffffffff;\n\t"
      "setp.ne.b32 pa, %4, 0;\n\t"
      "setp.ne.b32 pt, %3, 0;\n\t"
      "mov.b64 a0, {%1, %5};\n\t"
      "mov.b64 b0, {%2, %5};\n\t"
      "add.u32 l, %1, 2;\n\t"
      "mov.b64 a1, {l, %5};\n\t"
      "add.u32 l, %2, 2;\n\t"
      "mov.b64 b1, {l, %5};\n\t"
      "add.u32 l, %1, 4;\n\t"
      "mov.b64 a2, {l, %5};\n\t"
      "add.u32 l, %2, 4;\n\t"
      "mov.b64 b2, {l, %5};\n\t"
      "add.u32 l, %1, 6;\n\t"
      "mov.b64 a3, {l, %5};\n\t"
      "add.u32 l, %2, 6;\n\t"
      "mov.b64 b3, {l, %5};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], a0, b0, %3, pa;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, pt;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, pt;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, pt;\n\t"
      "}" ::"r"(d_tmem),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
// Four K = 16 steps; A from tensor memory (8 columns a step), B a tile of values (128 units of 16 bytes a step).
__device__ __forceinline__ void mma4_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred pe, pa, pt;\n\t"
      ".reg .b32 l, a1, a2, a3;\n\t"
      ".reg .b64 b0, b1, b2, b3;\n\t"
      "elect.sync _|pe, 0xffffffff;\n\t"
      "setp.ne.b32 pa, %4, 0;\n\t"
      "setp.ne.b32 pt, %3, 0;\n\t"
      "mov.b64 b0, {%2, %5};\n\t"
      "add.u32 a1, %1, 8;\n\t"
      "add.u32 l, %2, 128;\n\t"
      "mov.b64 b1, {l, %5};\n\t"
      "add.u32 a2, %1, 16;\n\t"
      "add.u32 l, %2, 256;\n\t"
      "mov.b64 b2, {l, %5};\n\t"
      "add.u32 a3, %1, 24;\n\t"
      "add.u32 l, %2, 384;\n\t"
      "mov.b64 b3, {l, %5};\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b0, %3, pa;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, pt;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, pt;\n\t"
      "@pe tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, pt;\n\t"
      "}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two tiles of queries of one kv head and the tiles of keys that any of their rows sees.
struct Unit {
  Sequence seq;
  int b, kvh, t0;  // sequence, kv head, first query
  int shift;       // position of query 0
  int win_tile, win_tiles, tiles;
  int from, every; // of the unit's tiles, this block has every `every`-th one from `from` on
  bool second;     // the second tile has rows
  // Tiles of the window, then those of the first keys.  Under a window the tile at its edge comes last of the former: a row that sees few
  // keys of its first tile has a low reference, and the next tile would rewrite its accumulator (1 x 8191 under a window of 2048
  // with four first keys in front: a rewrite for every 13th tile of a warp, 277 us; 242 so).
  __device__ __forceinline__ int key0(int n) const {
    const int t = n * every + from;
    if (t >= win_tiles) return (t - win_tiles) * kKeys;
    if (win_tile == 0) return t * kKeys;
    return (win_tile + (t + 1 == win_tiles ? 0 : t + 1)) * kKeys;
  }
};
// The units of a block, every gridDim.x-th one of the list that begins with the last queries of the longest prompts, which see the
// most keys unless others have more in front of them.  `busy`: units without keys are passed over.  SPLIT: one unit for the two blocks of a cluster, which share out its keys.
template <bool SPLIT>
struct Units {
  uint32_t id, step, total;
  __device__ __forceinline__ explicit Units(const PromptParams& p)
      : id(SPLIT ? blockIdx.x / 2 : blockIdx.x), step(SPLIT ? 0x7fffffff : gridDim.x), total(static_cast<uint32_t>(p.units) * p.a.kv_heads * p.a.batch) {}
  __device__ __forceinline__ bool next(const PromptParams& p, bool busy, Unit& u) {
    const uint32_t lanes = p.a.kv_heads * p.a.batch;
#pragma unroll 1
    for (; id < total; id += step) {
      const int rest = static_cast<int>(id % lanes);
      u.b = rest / p.a.kv_heads;
      u.kvh = rest % p.a.kv_heads;
      u.t0 = (p.units - 1 - static_cast<int>(id / lanes)) * 2 * p.tq;
      u.seq = sequence_of(p, u.b);
      if (u.seq.bad || u.t0 >= u.seq.n) continue;
      u.shift = u.seq.m - u.seq.n;
      const int lo = u.t0 + u.shift, hi = min(u.t0 + 2 * p.tq, u.seq.n) - 1 + u.shift;
      const int end = hi < 0 ? 0 : hi / kKeys + 1;
      u.win_tile = p.a.window > 0 ? min(max(lo - p.a.window + 1, 0) / kKeys, end) : 0;
      u.win_tiles = end - u.win_tile;
      u.tiles = u.win_tiles + min((p.a.sinks + kKeys - 1) / kKeys, u.win_tile);
      u.from = SPLIT ? static_cast<int>(blockIdx.x % 2) : 0;
      u.every = SPLIT ? 2 : 1;
      if constexpr (SPLIT) u.tiles = (u.tiles - u.from + 1) / 2;
      u.second = u.t0 + p.tq < u.seq.n;
      if (busy && u.tiles == 0) continue;
      id += step;
      return true;
    }
    return false;
  }
};

__device__ __forceinline__ void tmem_issue32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// Waits for every load issued so far; the registers pass through so that no use of them can move above it.
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
// The larger of three, NaN if one is NaN.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint64_t pair64(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair64(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Rows of a warp's 32 (of one kv head, queries from t0 on, the group's heads innermost).
struct WarpRows {
  Sequence seq;
  int t0, kvh;
  __device__ __forceinline__ int query(const PromptParams& p, int lane) const { return t0 + (static_cast<int>(threadIdx.x & 96) + lane) / p.group; }
  __device__ __forceinline__ int head(const PromptParams& p, int lane) const { return kvh * p.group + (static_cast<int>(threadIdx.x & 96) + lane) % p.group; }
};

// Up to sixteen rows by one warp, from the definition and each over its visible keys alone, 16 keys at a time with m16n8k16 products:
// the queries are the rows of both, the keys the columns of the first.  The order of the head dimensions within a product is free, so each
// lane loads 16 bytes of a key, and 32 bytes of a value for the columns 16 g + j of the j-th product.  Weights go to 16 bits as in the tiles,
// but not to zero, so that an infinity that a row sees stays one; keys that only some of the rows see are added in fp32, row by row.
// Once each output that is NaN as the rows stand is NaN again they stay as they are, unless `rewrite`.
constexpr int kAgain = 16;
template <typename T>
__device__ __forceinline__ void attend_rows(const PromptParams& p, const WarpRows& rows, uint32_t which, bool rewrite) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr float kUp = kBf16 ? 0.0f : 12.0f, kLeast = kBf16 ? 0x1p-126f : 0x1p-24f;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, D = p.a.head_dim;
  const Sequence& s = rows.seq;
  const T* k = static_cast<const T*>(p.a.k) + s.k0 * p.a.k_token + rows.kvh * p.a.k_head;
  const T* v = static_cast<const T*>(p.a.v) + s.k0 * p.a.v_token + rows.kvh * p.a.v_head;
  const int n = __popc(which);
  const auto eight = [&](const T* row, int d) { return d < D ? *reinterpret_cast<const uint4*>(row + d) : make_uint4(0u, 0u, 0u, 0u); };
  const auto nans_of_eight = [](const uint4& w) {
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
    uint32_t r = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = pair16<T>(a[e]);
      r |= (f.x != f.x ? 1u : 0u) << (2 * e) | (f.y != f.y ? 2u : 0u) << (2 * e);
    }
    return r;
  };
  // The lane's rows g and g + 8 of the products and, of their outputs, the head dimensions 32 t to 32 t + 31.
  T* out[2];
  int pos[2];
  Seen seen[2];
  uint4 qw[2][4];
  uint32_t nans[2] = {0, 0};
  float top[2], sum[2], o[16][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t left = which;
    for (int j = 0; j < g + 8 * i && j < n - 1; ++j) left &= left - 1;  // rows that are not there repeat the last one
    const int row = __ffs(left) - 1, token = rows.query(p, row), head = rows.head(p, row);
    pos[i] = token + s.m - s.n;
    seen[i] = seen_from(p, pos[i]);
    out[i] = static_cast<T*>(p.a.out) + (static_cast<int64_t>(s.q0 + token) * p.a.q_heads + head) * D + 32 * t;
    const T* q = static_cast<const T*>(p.a.q) + (s.q0 + token) * p.a.q_token + head * p.a.q_head;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      qw[i][c] = eight(q, 32 * c + 8 * t);
      nans[i] |= (32 * t + 8 * c < D ? nans_of_eight(*reinterpret_cast<const uint4*>(out[i] + 8 * c)) : 0u) << (8 * c);
    }
    top[i] = -INFINITY;
    sum[i] = 0.0f;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  // the keys that any of the rows sees
  const int first = __reduce_max_sync(0xffffffffu, max(seen[0].first, seen[1].first));
  const int start = max(__reduce_min_sync(0xffffffffu, min(seen[0].start, seen[1].start)), first);
  const int count = first + max(0, __reduce_max_sync(0xffffffffu, max(pos[0], pos[1])) + 1 - start);
  const auto key_of = [&](int u) { return u < first ? u : start + (u - first); };
#pragma unroll 1
  for (int u0 = 0; u0 < count; u0 += 16) {
    uint4 kw[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 4; ++c) kw[h][c] = eight(k + key_of(min(u0 + 8 * h + g, count - 1)) * p.a.k_token, 32 * c + 8 * t);
    float x[2][4] = {};  // rows g, g, g + 8, g + 8; keys 8 h + 2 t, 8 h + 2 t + 1
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mma16816<kBf16>(x[h], qw[0][c].x, qw[1][c].x, qw[0][c].y, qw[1][c].y, kw[h][c].x, kw[h][c].y);
        mma16816<kBf16>(x[h], qw[0][c].z, qw[1][c].z, qw[0][c].w, qw[1][c].w, kw[h][c].z, kw[h][c].w);
      }
    uint4 vw[4][2];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < 2; ++c) vw[e][c] = eight(v + key_of(min(u0 + 2 * t + (e & 1) + 8 * (e >> 1), count - 1)) * p.a.v_token, 16 * g + 8 * c);
    bool all_see = true;
    uint32_t sees = 0;  // bit 4 h + e of x[h][e]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float most = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int u = u0 + 8 * h + 2 * t + e, key = key_of(u);
          const bool in = u < count && key <= pos[i] && (key >= seen[i].start || key < seen[i].first);
          float& y = x[h][2 * i + e];
          y = in ? y * p.cl2 : -INFINITY;
          most = fmaxf(most, y);
          all_see &= in;
          sees |= in ? 1u << (4 * h + 2 * i + e) : 0u;
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2)), top[i]);
      const float keep = most == top[i] ? 1.0f : exp2f(top[i] - most), ref = most == -INFINITY ? 0.0f : most;
      top[i] = most;
      sum[i] *= keep;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& y = x[h][2 * i + e];
          const float w = exp2f((y - ref) + kUp);  // the difference first: exact near the maximum, however large that is
          sum[i] += w;
          y = y > -INFINITY ? fmaxf(w, kLeast) : w;
        }
      if (__any_sync(0xffffffffu, keep != 1.0f)) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          o[j][2 * i] *= keep;
          o[j][2 * i + 1] *= keep;
        }
      }
    }
    if (__all_sync(0xffffffffu, all_see)) {
      const uint32_t a[4] = {pack2<T>(x[0][0], x[0][1]), pack2<T>(x[0][2], x[0][3]), pack2<T>(x[1][0], x[1][1]), pack2<T>(x[1][2], x[1][3])};
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const auto word = [&](int e) {
          const uint4& w = vw[e][j / 8];
          return j % 8 < 4 ? (j % 8 < 2 ? w.x : w.y) : (j % 8 < 6 ? w.z : w.w);
        };
        const uint32_t half = j & 1 ? 0x7632u : 0x5410u;
        mma16816<kBf16>(o[j], a[0], a[1], a[2], a[3], __byte_perm(word(0), word(1), half), __byte_perm(word(2), word(3), half));
      }
    } else {
#pragma unroll 1
      for (int l = 0; l < min(16, count - u0); ++l) {
        const T* row = v + key_of(u0 + l) * p.a.v_token;
        const int from = (lane & 28) | ((l & 7) >> 1), bit = 4 * (l >> 3) + (l & 1);
        float w[2];
        bool in[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float mine = l < 8 ? (l & 1 ? x[0][2 * i + 1] : x[0][2 * i]) : (l & 1 ? x[1][2 * i + 1] : x[1][2 * i]);
          w[i] = __shfl_sync(0xffffffffu, mine, from);
          in[i] = (__shfl_sync(0xffffffffu, sees, from) >> (bit + 2 * i)) & 1u;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 four = eight(row, 32 * t + 8 * c);
          const uint32_t a[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 f = pair16<T>(a[e / 2]);
            const float value = e & 1 ? f.y : f.x;
            const int d = 8 * c + e;  // of the lane's 32
            if (in[0]) o[d % 16][d / 16] += w[0] * value;
            if (in[1]) o[d % 16][2 + d / 16] += w[1] * value;
          }
        }
      }
    }
    if (u0 % 128 == 0 && !rewrite) {
      uint32_t now[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) now[e >> 1] |= o[j][e] != o[j][e] ? 1u << (j + 16 * (e & 1)) : 0u;
#pragma unroll
      for (int i = 0; i < 2; ++i) now[i] |= sum[i] != sum[i] ? 0xffffffffu : 0u;  // of the row's four lanes one has it
      if (!__any_sync(0xffffffffu, ((nans[0] & ~now[0]) | (nans[1] & ~now[1])) != 0)) return;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
    sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    const bool none = sum[i] == 0.0f;  // zeros, whatever the values hold
    const float f = none ? 0.0f : 1.0f / sum[i];
    const auto output = [&](int d) { return none ? 0.0f : o[d % 16][2 * i + d / 16] * f; };
    if (g + 8 * i >= n) continue;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (32 * t + 8 * c < D)
        *reinterpret_cast<uint4*>(out[i] + 8 * c) = make_uint4(pack2<T>(output(8 * c), output(8 * c + 1)), pack2<T>(output(8 * c + 2), output(8 * c + 3)),
                                                               pack2<T>(output(8 * c + 4), output(8 * c + 5)), pack2<T>(output(8 * c + 6), output(8 * c + 7)));
  }
}

// The warp's rows of a unit that came out with NaN.  A weight of zero times NaN or infinity is NaN, so this may come from values
// that a row does not see (its tile has them), or sees with a weight that is zero in 16 bits: such a row is computed again from what it
// sees.  But mostly it sees the NaN, and is right.  The keys that all rows see are gone through once, four columns a lane, from both
// ends: a NaN or two opposite infinities among the values settle that column of every row, a NaN in a key settles whole rows.
// `large`: all rows are computed again (see LARGE_REF).
template <typename T>
__device__ __forceinline__ void look_again(const PromptParams& p, const WarpRows& rows, bool large) {
  const int lane = threadIdx.x & 31, D = p.a.head_dim;
  const Sequence& s = rows.seq;
  const bool holds = lane * 4 < D;
  const uint32_t all = holds ? 15u : 0u;  // this lane's columns
  const auto nans_of_four = [&](const void* at) {
    const uint2 w = *static_cast<const uint2*>(at);
    const float2 a = pair16<T>(w.x), b = pair16<T>(w.y);
    return nans_of(a.x, a.y, b.x, b.y);
  };
  uint32_t odd = 0, whole = 0, open = 0, found = 0;  // rows with a NaN, rows of nothing else; columns with one, columns whose NaN is seen by all rows
  const auto attend = [&](uint32_t left) {
#pragma unroll 1
    while (left != 0) {
      uint32_t which = 0;
      for (int n = 0; n < kAgain && left != 0; ++n) {
        which |= left & -left;
        left &= left - 1;
      }
      attend_rows<T>(p, rows, which, large);
    }
  };
  const int most = min(32, (min(kRows / p.group, s.n - rows.t0)) * p.group - static_cast<int>(threadIdx.x & 96));  // rows that are a query's
  if (large) odd = most <= 0 ? 0u : 0xffffffffu >> (32 - most);
  uint32_t of_rows[4];  // the lane's four columns of each row, eight rows a word
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    of_rows[e] = 0;
    uint2 w[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int row = 8 * e + r;
      const T* at = static_cast<const T*>(p.a.out) + (static_cast<int64_t>(s.q0 + rows.query(p, row)) * p.a.q_heads + rows.head(p, row)) * D + lane * 4;
      w[r] = holds && row < most ? *reinterpret_cast<const uint2*>(at) : make_uint2(0u, 0u);
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const uint32_t nans = nans_of_four(&w[r]);
      of_rows[e] |= nans << (4 * r);
      open |= nans;
      odd |= __any_sync(0xffffffffu, nans != 0) ? 1u << (8 * e + r) : 0u;
      whole |= __all_sync(0xffffffffu, nans == all) ? 1u << (8 * e + r) : 0u;
    }
  }
  const auto nans_of_row = [&](int r) { return ((r < 16 ? (r < 8 ? of_rows[0] : of_rows[1]) : (r < 24 ? of_rows[2] : of_rows[3])) >> (4 * (r & 7))) & 15u; };
  if (odd == 0) return;
  const int shift = s.m - s.n, lo = rows.query(p, __ffs(odd) - 1) + shift, hi = rows.query(p, 31 - __clz(odd)) + shift;
  // seen by all: the first keys, and from where the last row's window starts to the first row's position
  const Seen last = seen_from(p, hi);
  const int first = min(last.first, lo + 1), count = first + max(0, lo + 1 - last.start);
  constexpr int kStep = 16;
  const int steps = count > 0 && !large ? (count + kStep - 1) / kStep : 0;
  const auto scan = [&](const void* base, int64_t stride, auto take) {  // until `take` says that it has seen enough
#pragma unroll 1
    for (int n = 0; n < steps; ++n) {
      const int u0 = (n & 1 ? steps - 1 - n / 2 : n / 2) * kStep;
      uint2 w[kStep];
#pragma unroll
      for (int e = 0; e < kStep; ++e) {
        const int u = min(u0 + e, count - 1), key = u < first ? u : last.start + (u - first);
        w[e] = holds ? *reinterpret_cast<const uint2*>(static_cast<const T*>(base) + key * stride + lane * 4) : make_uint2(0u, 0u);
      }
      if (take(w)) return;
    }
  };
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  scan(static_cast<const T*>(p.a.v) + s.k0 * p.a.v_token + rows.kvh * p.a.v_head, p.a.v_token, [&](const uint2(&w)[kStep]) {
#pragma unroll
    for (int e = 0; e < kStep; ++e) {
      const float2 a = pair16<T>(w[e].x), b = pair16<T>(w[e].y);
      constexpr float kDown = 0x1p-40f;  // finite values of 2^30 keys stay finite together
      sum[0] += a.x * kDown;
      sum[1] += a.y * kDown;
      sum[2] += b.x * kDown;
      sum[3] += b.y * kDown;
    }
    found = nans_of(sum[0], sum[1], sum[2], sum[3]);
    return !__any_sync(0xffffffffu, (open & ~found) != 0);
  });
  const auto unsettled = [&](int r) { return __any_sync(0xffffffffu, (nans_of_row(r) & ~found) != 0); };
  uint32_t left = large ? odd : 0u;
#pragma unroll 1
  for (uint32_t rest = large ? 0u : odd; rest != 0; rest &= rest - 1) left |= unsettled(__ffs(rest) - 1) ? rest & -rest : 0u;
  if (!large && (left & whole) != 0) {
    bool key_nan = false;
    scan(static_cast<const T*>(p.a.k) + s.k0 * p.a.k_token + rows.kvh * p.a.k_head, p.a.k_token, [&](const uint2(&w)[kStep]) {
#pragma unroll
      for (int e = 0; e < kStep; ++e) key_nan |= nans_of_four(&w[e]) != 0;
      key_nan = __any_sync(0xffffffffu, key_nan);
      return key_nan;
    });
    if (key_nan) left &= ~whole;
  }
  attend(left);
}

// All units of a block once more, for a warp that met such rows.  Behind everything else: nothing in the block waits for it, however
// many keys there are, and it takes no registers from the loop over the units (as functions that are called, spills and 3 %).  8 x 2048 with a
// NaN in the first, the 700th, the 2040th value of each sequence: 0.43, 1.1, 1.0 ms, 0.31 without (events around a call); with every
// such row computed again by itself, in the loop, 101, 92, 17.
template <typename T, bool SPLIT>
__device__ __forceinline__ void look_again_at_all(const PromptParams& p, bool large) {
  const int i = threadIdx.x >> 7;  // the warp's tile of queries
  Unit u;
#pragma unroll 1
  for (Units<SPLIT> walk(p); walk.next(p, false, u);)
    if ((i == 0 || u.second) && u.from == 0) look_again<T>(p, WarpRows{u.seq, u.t0 + i * p.tq, u.kvh}, large);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2_in_order(float a, float b) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  } else {
    asm volatile("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  }
  return r;
}

// The largest of a row's 128 logits, in pieces that fit between other work.  NaN if one is NaN.
struct Largest {
  float top[4];
  __device__ __forceinline__ explicit Largest(const uint32_t (&x)[4][32]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) top[c] = max3_nan(__uint_as_float(x[c][0]), __uint_as_float(x[c][1]), __uint_as_float(x[c][31]));
  }
  __device__ __forceinline__ explicit Largest(const float (&t)[4]) : top{t[0], t[1], t[2], t[3]} {}
  // one of 15 steps
  __device__ __forceinline__ void step(const uint32_t (&x)[4][32], int n) {
    if (n < 0 || n > 14) return;
    const int j = n == 14 ? 30 : 2 + 2 * n;
#pragma unroll
    for (int c = 0; c < 4; ++c) top[c] = max3_nan(top[c], __uint_as_float(x[c][j]), __uint_as_float(x[c][n == 14 ? 30 : j + 1]));
  }
  __device__ __forceinline__ float result() const { return max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[3]); }
};

// Weights 2^(x cl2 + ref) of the pairs of columns FIRST to LAST.  The exponentials keep their unit (8 cycles a warp's instruction)
// busy only if the work around them is done between them, so the multiplications run two pairs ahead of them, the sums and the
// roundings two pairs behind; `beside(i)` is more work to be done in between, `done(k, words)` takes 16 words of two weights each.
template <typename T, int FIRST, int LAST, typename Beside, typename Done>
__device__ __forceinline__ void weigh(const uint32_t (&x)[4][32], uint64_t cl2, uint64_t ref, uint64_t (&sum)[2], Beside beside, Done done) {
  uint64_t y[LAST - FIRST];
  float a[LAST - FIRST], b[LAST - FIRST];
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < LAST - FIRST + 4; ++i) {
    if (i < LAST - FIRST) {
      const int c = (FIRST + i) / 16, j = 2 * (FIRST + i) % 32;
      y[i] = fma2(pair64(__uint_as_float(x[c][j]), __uint_as_float(x[c][j + 1])), cl2, ref);
    }
    if (i >= 2 && i - 2 < LAST - FIRST) {
      unpair64(y[i - 2], a[i - 2], b[i - 2]);
      a[i - 2] = exp2_fast(a[i - 2]);
      b[i - 2] = exp2_fast(b[i - 2]);
    }
    beside(i);
    if (i >= 4) {
      const int k = i - 4;
      sum[k & 1] = add2(sum[k & 1], pair64(a[k], b[k]));
      w[k % 16] = pack2_in_order<T>(a[k], b[k]);
      if (k % 16 == 15) done((FIRST + k) / 16, w);
    }
  }
}
// Columns under n of the 32 that begin at `from`.
__device__ __forceinline__ uint32_t columns_under(int n, int from) { return n <= from ? 0u : (n >= from + 32 ? 0xffffffffu : (1u << (n - from)) - 1u); }

// One tile of logits to weights: the row's 128 logits come from tensor memory and the weights go there over them, half by half;
// each half is handed to the product when it is there.  The first quarter is made relative to the reference of the tiles before
// while the maximum is still being looked for, and made again where that has outgrown the reference.
template <typename T, int DP, bool MASKED>
__device__ __forceinline__ void softmax_tile(uint32_t s_addr, uint32_t o_addr, float cl2, int hi, int lo, int sinks, bool first, bool live, uint64_t* p_full, float& m, float& l,
                                             bool& far) {
  using C = PromptCfg<T, DP>;
  uint32_t x[4][32], w[16];
  // column j is seen when j <= hi and (j > lo or j < sinks)
  const auto mask = [&](int c) {
    if constexpr (MASKED) {
      const uint32_t seen = columns_under(hi + 1, 32 * c) & (~columns_under(lo + 1, 32 * c) | columns_under(sinks, 32 * c));
      if (__any_sync(0xffffffffu, seen != 0xffffffffu)) {  // most quarters of a tile at the edge are seen by all rows of a warp
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!((seen >> j) & 1u)) x[c][j] = 0xff800000u;
      }
    }
  };
  const uint64_t cl22 = pair64(cl2, cl2);
  const auto reference = [&]() {
    const float ref = C::SHIFT - (m == -INFINITY ? 0.0f : m);
    return pair64(ref, ref);
  };
  const auto rest = [&]() {
#pragma unroll
    for (int c = 1; c < 4; ++c) tmem_wait32(x[c]);
#pragma unroll
    for (int c = 1; c < 4; ++c) mask(c);
  };
  const auto nothing = [](int) {};
  const auto keep_words = [&](int, const uint32_t(&words)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j] = words[j];
  };
  uint64_t sum[2] = {0, 0};
  tmem_issue32(s_addr, x[0]);
  tmem_wait32(x[0]);
#pragma unroll
  for (int c = 1; c < 4; ++c) tmem_issue32(s_addr + 32 * c, x[c]);
  mask(0);
  float most;
  if (first) {
    rest();
    Largest top(x);
#pragma unroll
    for (int n = 0; n < 15; ++n) top.step(x, n);
    most = top.result() * cl2;
  } else {
    if constexpr (MASKED) rest();
    float top[4];
    weigh<T, 0, 16>(x, cl22, reference(), sum,
                    [&](int i) {
                      if (i == 4) {
                        if constexpr (!MASKED) rest();
                        const Largest l0(x);
#pragma unroll
                        for (int c = 0; c < 4; ++c) top[c] = l0.top[c];
                      }
                      if (i > 4) {
                        Largest li(top);
                        li.step(x, i - 5);
#pragma unroll
                        for (int c = 0; c < 4; ++c) top[c] = li.top[c];
                      }
                    },
                    keep_words);
    most = Largest(top).result() * cl2;
  }
  // The reference that the weights are relative to follows the maximum only when that has outgrown it by 2^kSlack: the sums are the
  // same up to rounding, and the accumulator is seldom rewritten.  A NaN or an infinity among the logits makes it NaN, and with it the row.
  // Rows that are no query's hold anything and are left alone.
  const bool grow = live && (!(most <= m + kSlack) || (m == -INFINITY && most > -INFINITY));
  if (first || __any_sync(0xffffffffu, grow)) {
    const float next = !grow ? m : (most == INFINITY ? __int_as_float(0x7fc00000) : most);
    if (!first) {
      const float keep = grow ? exp2f(m - next) : 1.0f;
      l *= keep;
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        uint32_t o[16];
        tmem_issue16(o_addr + 16 * c, o);
        tmem_wait16(o);
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
        tmem_st16(o_addr + 16 * c, o);
      }
    }
    m = next;
    far |= live && fabsf(m) >= C::LARGE_REF && m != -INFINITY;
    sum[0] = sum[1] = 0;
    weigh<T, 0, 16>(x, cl22, reference(), sum, nothing, keep_words);
  }
  tmem_st16(s_addr, w);
  weigh<T, 16, 64>(x, cl22, reference(), sum, nothing, [&](int c, const uint32_t(&words)[16]) {
    tmem_st16(s_addr + 16 * c, words);
    if (c & 1) {
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full + c / 2);
    }
  });
  float a, b;
  unpair64(add2(sum[0], sum[1]), a, b);
  l += a + b;
}

// SPLIT: where units are few, the two blocks of a cluster share one, every second tile of its keys each, and the first joins their
// sums over distributed shared memory.
template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(kPromptThreads, 1)
prompt_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
              const __grid_constant__ PromptParams p) {
  using C = PromptCfg<T, DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  PromptAux* aux = reinterpret_cast<PromptAux*>(smem + C::AUX_OFFSET);
  volatile int* abort_flag = &aux->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0 && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_ALIGN));
    return;
  }
  if (blockIdx.x == 0 && p.a.status != nullptr)
    for (int b = threadIdx.x; b < p.a.batch; b += kPromptThreads)
      if (sequence_of(p, b).bad) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&aux->kv_full[i], 1);
      mbar_init(&aux->kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&aux->q_full[i], 1);
      mbar_init(&aux->q_empty[i], 1);
      mbar_init(&aux->s_full[i], 1);
      mbar_init(&aux->p_full[i][0], 128);
      mbar_init(&aux->p_full[i][1], 128);
      mbar_init(&aux->o_full[i], 1);
    }
    mbar_init(&aux->drain, 1);
    aux->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&aux->tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == kLoadWarp && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = aux->tmem_base;  // S 0, S 1 (128 columns each), O 0, O 1 (DP columns each)
  bool ok = true, timed_out = false;

  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == kLoadWarp) {
      // ------------------------------------------------------------------ loads: per unit Q 0, K 0, Q 1, V 0, K 1, V 1, K 2, ...
      uint32_t s = 0, ph = 1, uses[2] = {0, 0};
      int issued = 0;
      Unit u;
      for (Units<SPLIT> walk(p); ok && walk.next(p, true, u);) {
        const auto load_q = [&](int i) {
          ok = uniform_wait(&aux->q_empty[i], (uses[i] & 1) ^ 1, abort_flag);
          if (!ok) return;
          ++uses[i];
          prompt_expect(&aux->q_full[i], static_cast<uint32_t>(C::CHUNKS * p.tq * p.group * 128));
          for (int c = 0; c < C::CHUNKS; ++c)
            prompt_load(&aux->q_full[i], smem + i * C::TILE_BYTES + c * kChunkBytes, &tmap_q, c * 64, u.kvh * p.group, u.seq.q0 + u.t0 + i * p.tq);
        };
        load_q(0);
        for (int t = 0; t < u.tiles && ok; ++t) {
          const int row = u.seq.k0 + u.key0(t);
          for (int kv = 0; kv < 2 && ok; ++kv) {
            ok = uniform_wait(&aux->kv_empty[s], ph, abort_flag);
            if (!ok) break;
            ++issued;
            prompt_expect(&aux->kv_full[s], C::TILE_BYTES);
            for (int c = 0; c < C::CHUNKS; ++c)
              prompt_load(&aux->kv_full[s], smem + C::KV_OFFSET + s * C::TILE_BYTES + c * kChunkBytes, kv ? &tmap_v : &tmap_k, c * 64, u.kvh, row);
            if (++s == C::STAGES) {
              s = 0;
              ph ^= 1u;
            }
            if (t == 0 && kv == 0 && u.second) load_q(1);
          }
        }
      }
      if (!ok) {  // copies in flight land before the block retires
        if (lane == 0) {
          timed_out = !*abort_flag;
          *abort_flag = 1;
        }
        for (int i = 0; i < 2; ++i)
          if (uses[i] > 0) mbar_wait_drain(&aux->q_full[i], (uses[i] - 1) & 1);
        for (int n = max(0, issued - C::STAGES); n < issued; ++n) mbar_wait_drain(&aux->kv_full[n % C::STAGES], (n / C::STAGES) & 1);
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      // ------------------------------------------------------------------ products
      // The tiles of queries take turns, so that one is in the softmax while the other is in the tensor core.
      // in a cluster the address also names the block, which is no part of a descriptor
      const uint32_t base = (smem_u32(smem) & 0x3FFFFu) >> 4, d0 = uniform(tmem);
      uint32_t s = 0, ph = 0, q_ph = 0, p_ph = 0;  // bit i of the last two: tile i
      const auto step = [&]() {
        if (++s == C::STAGES) {
          s = 0;
          ph ^= 1u;
        }
      };
      const auto logits = [&](int i, uint32_t stage) {
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c)
          mma4_ss(d0 + i * kKeys, (base + ((i * C::TILE_BYTES + c * kChunkBytes) >> 4)) | kRowsLow,
                  (base + ((C::KV_OFFSET + c * kChunkBytes) >> 4) + stage * (C::TILE_BYTES >> 4)) | kRowsLow, C::IDESC_S, c > 0);
        tc_commit_elect(&aux->s_full[i]);
      };
      const auto first_logits = [&](int i, uint32_t stage, bool only) {
        ok = uniform_wait(&aux->q_full[i], (q_ph >> i) & 1, abort_flag);
        if (!ok) return;
        q_ph ^= 1u << i;
        tc_fence_after();
        logits(i, stage);
        if (only) tc_commit_elect(&aux->q_empty[i]);
      };
      // The weights' product waits for either half of them, then takes its half of the values.
      const auto outputs = [&](int i, uint32_t stage, bool first) {
        const uint32_t values = (base + (C::KV_OFFSET >> 4) + stage * (C::TILE_BYTES >> 4)) | kValuesLow;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          ok = uniform_wait(&aux->p_full[i][half], (p_ph >> i) & 1, abort_flag);
          if (!ok) return;
          tc_fence_after();
          mma4_ts(d0 + 2 * kKeys + i * DP, d0 + i * kKeys + 32 * half, values + 512 * half, C::IDESC_O, !first || half);
        }
        p_ph ^= 1u << i;
      };
      Unit unit;
      Units<SPLIT> walk(p);
      const auto advance = [&](int& tiles, bool& second) {
        const bool have = uniform(walk.next(p, true, unit)) != 0;
        tiles = uniform(have ? unit.tiles : 0);
        second = uniform(have && unit.second) != 0;
        return have;
      };
      int tiles, next_tiles;
      bool second, next_second;
      bool have = advance(tiles, second);
      if (have) {
        const uint32_t sk = s;
        ok = uniform_wait(&aux->kv_full[sk], ph, abort_flag);
        step();
        if (ok) first_logits(0, sk, tiles == 1);
        if (ok && second) first_logits(1, sk, tiles == 1);
        if (ok) tc_commit_elect(&aux->kv_empty[sk]);
      }
      while (have && ok) {
        const bool next = advance(next_tiles, next_second);
        for (int t = 0; t < tiles && ok; ++t) {
          const bool more = t + 1 < tiles;
          // the values of this tile and the keys of the next one, in one wait
          const uint32_t sv = s, v_ph = ph;
          step();
          const uint32_t sk = s, k_ph = ph;
          if (more || next) step();
          ok = uniform_wait(&aux->kv_full[sv], v_ph, abort_flag, more || next ? &aux->kv_full[sk] : nullptr, k_ph);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const bool mine = i == 0 || second;
            if (mine && ok) {
              outputs(i, sv, t == 0);
              if (ok && !more) tc_commit_elect(&aux->o_full[i]);
            }
            if (ok && i == (second ? 1 : 0)) tc_commit_elect(&aux->kv_empty[sv]);
            if (ok && more && mine) {
              logits(i, sk);
              if (t + 2 == tiles) tc_commit_elect(&aux->q_empty[i]);
            } else if (ok && !more && next && (i == 0 || next_second)) {
              first_logits(i, sk, next_tiles == 1);  // right behind the last outputs of the unit before
            }
          }
          if (ok && (more || next)) tc_commit_elect(&aux->kv_empty[sk]);
        }
        tiles = next_tiles;
        second = next_second;
        have = next;
      }
      if (!ok && lane == 0) {
        timed_out = !*abort_flag;
        *abort_flag = 1;
      }
      __syncwarp();
      // nothing may still be reading shared memory or writing tensor memory when the block retires
      tc_commit_elect(&aux->drain);
      mbar_wait_drain(&aux->drain, 0);
    }
  } else {
    // ------------------------------------------------------------------ softmax: a thread a row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int i = warp >> 2, r = (warp & 3) * 32 + lane;
    const int row_token = r / p.group, row_head = r % p.group;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + i * kKeys, o_addr = tmem + lanes + 2 * kKeys + i * DP;
    uint32_t s_uses = 0, o_uses = 0;
    bool odd = false, large = false;  // an output is NaN where it may not be; a reference was too large
    // The outputs of a tile of queries, from its accumulator and sum (with SPLIT, and those of the cluster's other block).
    const auto finish = [&](const Unit& u, float m, float l, bool far) {
      const int token = u.t0 + i * p.tq + row_token, head = u.kvh * p.group + row_head;
      const bool row_ok = row_token < p.tq && token < u.seq.n;
      float own = 1.0f, other = 0.0f;  // factors of the two blocks' sums
      if constexpr (SPLIT) {
        const float2 ml = ld_cluster_f2(smem_u32(smem) + C::PART_ML + (i * kRows + r) * 8, 1);
        const float top = max3_nan(m, ml.x, ml.x);
        far |= ml.x == INFINITY;
        own = m == top ? 1.0f : exp2f(m - top);
        other = ml.x == top ? 1.0f : exp2f(ml.x - top);
        l = l * own + ml.y * other;
      }
      const bool none = l == 0.0f;  // no weight anywhere: zeros, whatever the values hold
      const float scale = none ? 0.0f : 1.0f / l;
      // Rows go through shared memory, 64 outputs at a time, so that eight lanes write the 128 bytes of a row together (a lane for
      // each row touches 32 lines with every store: 8 x 2048 290 us, 282 so).
      T* out = static_cast<T*>(p.a.out) + (static_cast<int64_t>(u.seq.q0 + token) * p.a.q_heads + head) * p.a.head_dim;
      const uint64_t out_row = row_ok ? reinterpret_cast<uint64_t>(out) : 0;
      uint8_t* stage = smem + C::OUT_OFFSET + warp * 4096;
      bool again = false;
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        uint32_t o[32];
        if (u.tiles > 0) {
          tmem_ld32(o_addr + 32 * c, o);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0u;
        }
        if constexpr (SPLIT) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 v = ld_cluster_f4(smem_u32(smem) + C::part_o(i * kRows + r, 8 * c + j / 4), 1);
            o[j] = __float_as_uint(__uint_as_float(o[j]) * own + v.x * other);
            o[j + 1] = __float_as_uint(__uint_as_float(o[j + 1]) * own + v.y * other);
            o[j + 2] = __float_as_uint(__uint_as_float(o[j + 2]) * own + v.z * other);
            o[j + 3] = __float_as_uint(__uint_as_float(o[j + 3]) * own + v.w * other);
          }
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = none ? 0u : o[j];
#pragma unroll
        for (int j = 0; j < 32; ++j) again |= __uint_as_float(o[j]) != __uint_as_float(o[j]);
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = pack2<T>(__uint_as_float(o[j + 2 * e]) * scale, __uint_as_float(o[j + 2 * e + 1]) * scale);
          *reinterpret_cast<uint4*>(stage + lane * 128 + (((c & 1) * 4 + j / 8) ^ (lane & 7)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (c & 1) {
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int rr = 4 * k + (lane >> 3), piece = lane & 7;
            const uint64_t dst = __shfl_sync(0xffffffffu, out_row, rr);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((piece ^ (rr & 7)) * 16));
            if (dst != 0 && 32 * (c - 1) + piece * 8 < p.a.head_dim) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(dst) + 32 * (c - 1) + piece * 8) = v;
          }
          __syncwarp();
        }
      }
      tc_fence_before();  // the next unit's weights are announced behind these reads of the accumulator
      // NaN among the logits that a row sees makes its sum NaN, and with that every output, rightly.  With any other sum:
      odd |= row_ok && again && l == l;
      large |= far;
    };
    Unit u;
    bool mine = false;
    float m, l;
    bool far = false;  // a reference of this row was too large, if only at first
    for (Units<SPLIT> walk(p); ok && walk.next(p, false, u);) {
      if (i == 1 && !u.second) continue;
      mine = true;
      const int token = u.t0 + i * p.tq + row_token;
      const bool row_ok = row_token < p.tq && token < u.seq.n;
      const int pos = token + u.shift;
      const int tile_lo = u.t0 + i * p.tq + u.shift, tile_hi = tile_lo + p.tq - 1;  // positions of this tile of queries
      m = -INFINITY;
      l = 0.0f;
      far = false;
      for (int t = 0; t < u.tiles && ok; ++t) {
        ok = uniform_wait(&aux->s_full[i], s_uses & 1, abort_flag);
        if (!ok) break;
        ++s_uses;
        tc_fence_after();
        const int k0 = u.key0(t);
        const bool full = k0 + kKeys - 1 <= tile_lo && (p.a.window <= 0 || k0 > tile_hi - p.a.window || k0 + kKeys <= p.a.sinks);
        if (full) {
          softmax_tile<T, DP, false>(s_addr, o_addr, p.cl2, 0, 0, 0, t == 0, row_ok, aux->p_full[i], m, l, far);
        } else {
          softmax_tile<T, DP, true>(s_addr, o_addr, p.cl2, pos - k0, p.a.window > 0 ? pos - p.a.window - k0 : -1, p.a.sinks - k0, t == 0, row_ok, aux->p_full[i], m, l, far);
        }
      }
      if (ok && u.tiles > 0) {
        ok = uniform_wait(&aux->o_full[i], o_uses & 1, abort_flag);
        ++o_uses;
      }
      if (!ok) break;
      tc_fence_after();
      if constexpr (!SPLIT) {
        finish(u, m, l, far);
      } else {
        // the other tile's products may still read what the sums go over
        if (u.second && u.tiles > 0) ok = uniform_wait(&aux->o_full[1 - i], 0, abort_flag);
        if (!ok) break;
        if (u.from > 0) {
#pragma unroll 1
          for (int c = 0; c < DP / 16; ++c) {
            uint32_t o[16] = {};
            if (u.tiles > 0) {
              tmem_issue16(o_addr + 16 * c, o);
              tmem_wait16(o);
            }
#pragma unroll
            for (int j = 0; j < 16; j += 4) *reinterpret_cast<uint4*>(smem + C::part_o(i * kRows + r, 4 * c + j / 4)) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
          *reinterpret_cast<float2*>(smem + C::PART_ML + (i * kRows + r) * 8) = make_float2(far ? INFINITY : m, l);
        }
      }
    }
    if (!ok && lane == 0) {
      timed_out = !*abort_flag;
      *abort_flag = 1;
    }
    __syncwarp();
    if constexpr (SPLIT) {
      cluster_arrive_wait();
      if (mine && ok && u.from == 0) finish(u, m, l, far);
      __syncwarp();
    }
    large = __any_sync(0xffffffffu, large);
    if (ok && __any_sync(0xffffffffu, odd || large)) look_again_at_all<T, SPLIT>(p, large);
  }
  if constexpr (SPLIT) {
    __syncwarp();  // the barriers of a cluster are taken by whole warps
    if (warp >= kSoftmaxWarps) cluster_arrive_wait();
    cluster_arrive_wait();  // nobody leaves while its sums are read
  }
  if (timed_out && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_TIMEOUT));
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// [tokens, heads, head_dim] read in boxes of box_tokens x box_heads x 64 elements; head dimensions past the end are zeros.
static int head_map(CUtensorMap* tm, const void* base, int dtype, int64_t tokens, int64_t heads, int64_t dim, int64_t token_stride, int64_t head_stride, int box_tokens,
                    int box_heads) {
  using Fn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                          CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  const Fn enc = reinterpret_cast<Fn>(tensor_map_encoder());
  if (enc == nullptr) return fail(QLIN_ERR_DEVICE, "cuTensorMapEncodeTiled is not available from this driver");
  const int64_t row = (dim * 2 + 15) / 16 * 16;  // stands in for the stride of a dimension with one entry
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(heads > 1 ? head_stride * 2 : row), static_cast<cuuint64_t>(tokens > 1 ? token_stride * 2 : row)};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(tm, dtype == QLIN_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(QLIN_ERR_BAD_ALIGN, "qlin_prompt_attention: cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
  return QLIN_OK;
}

template <typename T, int DP, bool SPLIT>
static int launch_prompt_as(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PromptParams& p, unsigned grid, cudaStream_t stream) {
  using C = PromptCfg<T, DP>;
  const auto kernel = prompt_kernel<T, DP, SPLIT>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(QLIN_ERR_DEVICE, "device ordinal %d out of range", dev);
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    if (e != cudaSuccess) return fail(QLIN_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    cudaFuncAttributes attr;
    const cudaError_t f = cudaFuncGetAttributes(&attr, kernel);
    if (f != cudaSuccess) return fail(QLIN_ERR_LAUNCH, "cudaFuncGetAttributes: %s", cudaGetErrorString(f));
    // what the softmax warps ask for must be there, or they would wait for it for good
    if (attr.numRegs * kPromptThreads < 32 * (kSoftmaxWarps * kSoftmaxRegs + 4 * kOtherRegs))
      return fail(QLIN_ERR_LAUNCH, "qlin_prompt_attention: built with %d registers a thread, too few for its split", attr.numRegs);
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(kPromptThreads, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SPLIT ? 2 : 1;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = SPLIT ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tq, tk, tv, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(QLIN_ERR_LAUNCH, "qlin_prompt_attention: %s", cudaGetErrorString(e));
  }
  return QLIN_OK;
}

template <typename T, int DP>
static int launch_prompt(const PromptParams& p, cudaStream_t stream) {
  CUtensorMap tq, tk, tv;
  int rc = head_map(&tq, p.a.q, p.a.dtype, p.a.tokens_q, p.a.q_heads, p.a.head_dim, p.a.q_token, p.a.q_head, p.tq, p.group);
  if (rc == QLIN_OK) rc = head_map(&tk, p.a.k, p.a.dtype, p.a.tokens_k, p.a.kv_heads, p.a.head_dim, p.a.k_token, p.a.k_head, kKeys, 1);
  if (rc == QLIN_OK) rc = head_map(&tv, p.a.v, p.a.dtype, p.a.tokens_k, p.a.kv_heads, p.a.head_dim, p.a.v_token, p.a.v_head, kKeys, 1);
  if (rc != QLIN_OK) return rc;
  const int64_t blocks = static_cast<int64_t>(p.units) * p.a.kv_heads * p.a.batch;
  if (blocks > 0x7fffffff) return fail(QLIN_ERR_TOO_LARGE, "qlin_prompt_attention: too many queries, heads and sequences");
  // Units that leave half of the SMs idle are split over two blocks where the longest has kSplitTiles tiles of keys (as far as the host
  // knows: the earlier keys are taken as evenly spread).  Device time without and with: 1200 queries of 12 heads of 64 (10 tiles) 24.4 and 19.8 us,
  // 2000 of 8 + 1 heads of 96 36.3 and 30.7, 16 after 2900 of 32 + 8 heads of 128 41.8 and 29.4; 40 after 900 (8 tiles) 21.6 and 22.4.
  // Four blocks lose more in the join, which one of them does alone, than they save (64 after 2900 of 8 + 2 heads 50 in one, 37 in two, 59 in four).
  int64_t keys = p.a.max_q + (p.a.tokens_k > p.a.tokens_q ? (p.a.tokens_k - p.a.tokens_q) / p.a.batch : 0);
  const int64_t seen = static_cast<int64_t>(p.a.window) + p.a.sinks + 2 * p.tq;
  if (p.a.window > 0 && keys > seen) keys = seen;
  if (2 * blocks <= sm_count() && (keys + kKeys - 1) / kKeys >= kSplitTiles) return launch_prompt_as<T, DP, true>(tq, tk, tv, p, static_cast<unsigned>(2 * blocks), stream);
  return launch_prompt_as<T, DP, false>(tq, tk, tv, p, static_cast<unsigned>(blocks < sm_count() ? blocks : sm_count()), stream);
}

// The check of the offsets alone, for calls that compute nothing: without sequences, queries of a sequence or keys.
__global__ void prompt_offsets_kernel(const __grid_constant__ PromptParams p) {
  bool bad = p.a.batch == 0 || p.a.max_q == 0;  // there are rows, so the offsets cannot cover them
  if (!bad)
    for (int b = threadIdx.x; b < p.a.batch; b += blockDim.x) bad |= sequence_of(p, b).bad;
  if (bad) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
}
static int check_offsets(const PromptParams& p, cudaStream_t stream) {
  if (p.a.status == nullptr) return QLIN_OK;
  prompt_offsets_kernel<<<1, 256, 0, stream>>>(p);
  QLIN_CHECK_LAUNCH("qlin_prompt_attention");
  return QLIN_OK;
}

}  // namespace qlin

extern "C" int qlin_prompt_attention(const qlin_prompt_attention_args* a, void* stream) {
  using namespace qlin;
  if (a == nullptr) return fail(QLIN_ERR_NULL, "qlin_prompt_attention: args is NULL");
  if (a->tokens_q < 0 || a->tokens_k < 0 || a->batch < 0 || a->max_q < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads != 0)
    return fail(QLIN_ERR_BAD_SHAPE, "qlin_prompt_attention: q_heads must be a multiple of kv_heads");
  if (a->q_heads / a->kv_heads > 128) return fail(QLIN_ERR_UNSUPPORTED, "qlin_prompt_attention: at most 128 query heads share a kv head");
  if (a->dtype != QLIN_DT_F16 && a->dtype != QLIN_DT_BF16) return fail(QLIN_ERR_BAD_DTYPE, "qlin_prompt_attention: q, k and v must be fp16 or bf16");
  if (a->head_dim < 8 || a->head_dim % 8 != 0 || a->head_dim > 128) return fail(QLIN_ERR_BAD_SHAPE, "qlin_prompt_attention: head_dim must be a multiple of 8 up to 128");
  if (a->tokens_q == 0) return QLIN_OK;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  PromptParams p;
  p.a = *a;
  if (a->batch == 0 || a->max_q == 0) return check_offsets(p, s);
  if (a->q == nullptr || a->out == nullptr || a->cu_q == nullptr || a->cu_k == nullptr) return fail(QLIN_ERR_NULL, "qlin_prompt_attention: q, out, cu_q or cu_k is NULL");
  if (a->tokens_k > 0 && (a->k == nullptr || a->v == nullptr)) return fail(QLIN_ERR_NULL, "qlin_prompt_attention: k or v is NULL");
  if (a->tokens_q > kMostTokens || a->tokens_k > kMostTokens) return fail(QLIN_ERR_TOO_LARGE, "qlin_prompt_attention: at most 2^30 tokens");
  if (static_cast<int64_t>(a->kv_heads) * a->batch > (1 << 24)) return fail(QLIN_ERR_TOO_LARGE, "qlin_prompt_attention: too many heads and sequences");
  if (!(a->scale > 0.0f) || a->scale > 3.0e38f) return fail(QLIN_ERR_UNSUPPORTED, "qlin_prompt_attention: scale must be positive and finite");
  const auto pitch = [](int64_t entries, int64_t stride) { return entries > 1 && (stride <= 0 || stride >= (int64_t{1} << 38)); };
  if (pitch(a->tokens_q, a->q_token) || pitch(a->q_heads, a->q_head) || pitch(a->tokens_k, a->k_token) || pitch(a->kv_heads, a->k_head) ||
      pitch(a->tokens_k, a->v_token) || pitch(a->kv_heads, a->v_head))
    return fail(QLIN_ERR_BAD_SHAPE, "qlin_prompt_attention: strides must be positive");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) || a->q_token % 8 != 0 || a->q_head % 8 != 0 || a->k_token % 8 != 0 ||
      a->k_head % 8 != 0 || a->v_token % 8 != 0 || a->v_head % 8 != 0)
    return fail(QLIN_ERR_BAD_ALIGN, "qlin_prompt_attention: every row must start on 16 bytes");
  p.group = a->q_heads / a->kv_heads;
  p.cl2 = a->scale * 1.4426950408889634f;
  if (p.a.window > kMostTokens) p.a.window = kMostTokens;  // as far as any sequence reaches, and sums with positions stay in 32 bits
  if (p.a.sinks > kMostTokens) p.a.sinks = kMostTokens;
  if (p.a.sinks < 0) p.a.sinks = 0;
  p.tq = kRows / p.group;
  p.units = static_cast<int32_t>((static_cast<int64_t>(a->max_q) + 2 * p.tq - 1) / (2 * p.tq));
  if (a->tokens_k == 0) {  // nothing to see: the tensor maps have no memory to describe
    const cudaError_t e = cudaMemsetAsync(a->out, 0, static_cast<size_t>(a->tokens_q) * a->q_heads * a->head_dim * 2, s);
    return e == cudaSuccess ? check_offsets(p, s) : fail(QLIN_ERR_LAUNCH, "qlin_prompt_attention: %s", cudaGetErrorString(e));
  }
  if (a->dtype == QLIN_DT_BF16) return a->head_dim <= 64 ? launch_prompt<__nv_bfloat16, 64>(p, s) : launch_prompt<__nv_bfloat16, 128>(p, s);
  return a->head_dim <= 64 ? launch_prompt<__half, 64>(p, s) : launch_prompt<__half, 128>(p, s);
}
