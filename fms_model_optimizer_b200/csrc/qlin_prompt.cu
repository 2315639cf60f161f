// qlin_prompt_attention: attention of packed prompts under a causal mask, a sliding window and first tokens that stay visible.
//
//   o_i = sum_j w_j v_j / sum_j w_j,   w_j = 2^(x_j - r),   x_j = q_i.k_j scale log2(e),   j over the keys that i sees
//
// for any r; r follows the running maximum.  A persistent block has two tiles of 128 rows of one kv head and goes over tiles of 128
// keys.  A tile's rows are 128 / G queries times the G query heads that share the kv head, so grouped heads share each load and a
// tile spans few positions, which keeps what the mask throws away small.  S = Q K^T on tcgen05 with both operands in shared memory, one
// thread for each row of 128 logits in tensor memory, the weights back to tensor memory over their logits in 16 bits, O += P V
// with the weights as the operand from there.  Tensor memory is full: two S of 128 columns, two O of head_dim.  The tiles take turns, one in the softmax
// while the other is in the tensor core.
//
// What bounds it: that chain.  A turn (two tiles against 128 keys) is 2048 cycles of tensor core and 2048 of exponentials (two
// tiles x 128 a thread x 8 cycles), and takes about 4200: the exponentials of a tile and its products follow one another, and the
// third pair of buffers that would let a tile's next logits be made meanwhile does not fit.  Measured (device time): 8 x 2048, 32 + 8 heads
// of 128 in bf16 280 us, 980 TFLOP/s = 0.60 of the measured rate; 1 x 8191 under a window of 2048 with four first keys 243 us,
// 990; 5 x up to 333 after 77, 12 heads of 64 in fp16 13 us, four turns behind a cold start.  With exponentials, maxima and masks left
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

// One query of one head by one warp, from the definition and over the visible keys alone: 32 keys at a time, a lane for each key's
// logit, then four neighbouring outputs for each lane.
template <typename T>
__device__ __noinline__ void attend_row(const PromptParams& p, const Sequence& s, int i, int head) {
  const int lane = threadIdx.x & 31, D = p.a.head_dim, pos = i + s.m - s.n;
  const T* q = static_cast<const T*>(p.a.q) + (s.q0 + i) * p.a.q_token + head * p.a.q_head;
  const T* k = static_cast<const T*>(p.a.k) + s.k0 * p.a.k_token + head / p.group * p.a.k_head;
  const T* v = static_cast<const T*>(p.a.v) + s.k0 * p.a.v_token + head / p.group * p.a.v_head;
  const int start = p.a.window > 0 ? max(0, pos - p.a.window + 1) : 0, first = min(max(p.a.sinks, 0), start);
  const int count = pos < 0 ? 0 : first + pos + 1 - start;
  const bool writes = lane * 4 < D;
  float top = -INFINITY, sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int u0 = 0; u0 < count; u0 += 32) {
    const int u = u0 + lane, key = u < first ? u : start + (u - first);
    float x = -INFINITY;
    if (u < count) {
      float dot = 0.0f;
      const uint4* kr = reinterpret_cast<const uint4*>(k + key * p.a.k_token);
      const uint4* qr = reinterpret_cast<const uint4*>(q);
      for (int c = 0; c < D / 8; ++c) {
        const uint4 kw = kr[c], qw = qr[c];
        const uint32_t ka[4] = {kw.x, kw.y, kw.z, kw.w}, qa[4] = {qw.x, qw.y, qw.z, qw.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 kp = pair16<T>(ka[e]), qp = pair16<T>(qa[e]);
          dot += kp.x * qp.x + kp.y * qp.y;
        }
      }
      x = dot * p.cl2;
    }
    float most = x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    most = fmaxf(most, top);
    const float keep = most == top ? 1.0f : exp2f(top - most), ref = most == -INFINITY ? 0.0f : most;
    top = most;
    const float w = u < count ? exp2f(x - ref) : 0.0f;
    float part = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    sum = sum * keep + part;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= keep;
    const int here = min(32, count - u0);
    for (int l = 0; l < here; ++l) {
      const float wl = __shfl_sync(0xffffffffu, w, l);
      const int kl = __shfl_sync(0xffffffffu, key, l);
      if (writes) {
        const uint2 r = *reinterpret_cast<const uint2*>(v + kl * p.a.v_token + lane * 4);
        const float2 a = pair16<T>(r.x), b = pair16<T>(r.y);
        acc[0] += wl * a.x;
        acc[1] += wl * a.y;
        acc[2] += wl * b.x;
        acc[3] += wl * b.y;
      }
    }
  }
  if (writes) {
    const bool none = sum == 0.0f;  // zeros, whatever the values hold
    const float r = none ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = none ? 0.0f : acc[e];
    T* out = static_cast<T*>(p.a.out) + (static_cast<int64_t>(s.q0 + i) * p.a.q_heads + head) * D + lane * 4;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(acc[0] * r, acc[1] * r), pack2<T>(acc[2] * r, acc[3] * r));
  }
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
  // with four first keys in front: a rewrite for every 13th tile of a warp, 277 us; 243 so).
  __device__ __forceinline__ int key0(int n) const {
    const int t = n * every + from;
    if (t >= win_tiles) return (t - win_tiles) * kKeys;
    if (win_tile == 0) return t * kKeys;
    return (win_tile + (t + 1 == win_tiles ? 0 : t + 1)) * kKeys;
  }
};
// The units of a block, every gridDim.x-th one of the list that begins with the last queries of every sequence and head, which see
// the most keys.  `busy`: units without keys are passed over.  SPLIT: one unit for the two blocks of a cluster, which share out its keys.
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
__device__ __forceinline__ void softmax_tile(uint32_t s_addr, uint32_t o_addr, float cl2, int hi, int lo, int sinks, bool first, bool live, uint64_t* p_full, float& m, float& l) {
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
    // The outputs of a tile of queries, from its accumulator and sum (with SPLIT, and those of the cluster's other block).
    const auto finish = [&](const Unit& u, float m, float l) {
      const int token = u.t0 + i * p.tq + row_token, head = u.kvh * p.group + row_head;
      const bool row_ok = row_token < p.tq && token < u.seq.n;
      float own = 1.0f, other = 0.0f;  // factors of the two blocks' sums
      if constexpr (SPLIT) {
        const float2 ml = ld_cluster_f2(smem_u32(smem) + C::PART_ML + (i * kRows + r) * 8, 1);
        const float top = max3_nan(m, ml.x, ml.x);
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
      // A weight of zero times NaN or infinity is NaN: a value that the row does not see may have got into its sums, so rows that
      // come out as NaN are computed again from what they do see.  (A NaN or an infinity among the logits that a row sees makes its sum
      // NaN, and with that every output, rightly.)
      uint32_t redo = __ballot_sync(0xffffffffu, row_ok && again && l == l);
      __syncwarp();  // the rows are written before they are written again
      while (redo != 0) {
        const int r2 = (warp & 3) * 32 + __ffs(redo) - 1;
        redo &= redo - 1;
        attend_row<T>(p, u.seq, u.t0 + i * p.tq + r2 / p.group, u.kvh * p.group + r2 % p.group);
      }
    };
    Unit u;
    bool mine = false;
    float m, l;
    for (Units<SPLIT> walk(p); ok && walk.next(p, false, u);) {
      if (i == 1 && !u.second) continue;
      mine = true;
      const int token = u.t0 + i * p.tq + row_token;
      const bool row_ok = row_token < p.tq && token < u.seq.n;
      const int pos = token + u.shift;
      const int tile_lo = u.t0 + i * p.tq + u.shift, tile_hi = tile_lo + p.tq - 1;  // positions of this tile of queries
      m = -INFINITY;
      l = 0.0f;
      for (int t = 0; t < u.tiles && ok; ++t) {
        ok = uniform_wait(&aux->s_full[i], s_uses & 1, abort_flag);
        if (!ok) break;
        ++s_uses;
        tc_fence_after();
        const int k0 = u.key0(t);
        const bool full = k0 + kKeys - 1 <= tile_lo && (p.a.window <= 0 || k0 > tile_hi - p.a.window || k0 + kKeys <= p.a.sinks);
        if (full) {
          softmax_tile<T, DP, false>(s_addr, o_addr, p.cl2, 0, 0, 0, t == 0, row_ok, aux->p_full[i], m, l);
        } else {
          softmax_tile<T, DP, true>(s_addr, o_addr, p.cl2, pos - k0, p.a.window > 0 ? pos - p.a.window - k0 : -1, p.a.sinks - k0, t == 0, row_ok, aux->p_full[i], m, l);
        }
      }
      if (ok && u.tiles > 0) {
        ok = uniform_wait(&aux->o_full[i], o_uses & 1, abort_flag);
        ++o_uses;
      }
      if (!ok) break;
      tc_fence_after();
      if constexpr (!SPLIT) {
        finish(u, m, l);
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
          *reinterpret_cast<float2*>(smem + C::PART_ML + (i * kRows + r) * 8) = make_float2(m, l);
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
      if (mine && ok && u.from == 0) finish(u, m, l);
      __syncwarp();
    }
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
  // knows: the earlier keys are taken as evenly spread).  Device time without and with: 1200 queries of 12 heads of 64 (10 tiles) 23.7 and 19.7 us,
  // 2000 of 8 + 1 heads of 96 35.7 and 30.4, 16 after 2900 of 32 + 8 heads of 128 41.0 and 26.3; 40 after 900 (8 tiles) 20.8 and 22.4.
  // Four blocks lose more in the join than they save (64 after 2900 of 8 + 2 heads 39 in two, 59 in four).
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
