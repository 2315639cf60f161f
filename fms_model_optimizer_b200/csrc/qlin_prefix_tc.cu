// The prefix's part of qlin_prefix_attention for groups of many rows: tiles of 128 rows against tiles of 128 keys on tcgen05.
//
//   m = max x,  l = sum 2^((x - m) c),  o = sum 2^((x - m) c) v      over the keys of a split, for a row of logits x,  c = scale log2(e)
//
// A row is a query of one of the group's sequences; all of them see all the keys here, so nothing is masked but the end of the last tile.  S = Q K^T with both
// operands in shared memory, a thread for each row of 128 logits in tensor memory, the weights back to tensor memory over their logits in 16 bits, O += P V with the
// weights as the operand from there.  Two streams of tiles take turns, one in the softmax while the other is in the tensor core: two tiles of rows that share each tile of keys and
// values, or, where a group has no more than 128 rows, one tile of rows against two splits of the keys.
//
// Keys and values come by TMA, a box of up to 32 keys of a page at a time, found through the page table; pages whose size has no factor of 8, and strides that no tensor map
// describes, are left to the kernel of the attention over pages.  The keys that are read here begin and end at multiples of the box, so that no box holds a key that
// somebody does not see; the few beside them are the sequences' own.  e4m3 codes land beside the tiles and two warps make fp16 of them on the way there; a bf16 query
// meets these as fp16 times a power of two that brings its largest element to 2^13..2^14.  (Through the threads' registers and 16-byte asynchronous copies, which take
// pages of any size, the loads were what the rest waited for: with them 2 x 64 sequences behind 32768 keys took the whole operator 127 us at best, the first boxes by TMA 101.)
//
// What bounds it: the chain of products and exponentials, 3450 cycles for two tiles of rows against a tile of keys where the tensor core needs 2048 and so do the exponentials (2 x 64 sequences
// behind 32768 keys 72 us, the tensor pipe busy for half of it); short prefixes by the start and the end of a block, some 12 us.
//
// Logits enter the exponent as their difference from the reference, so that it is exact near the maximum however large they are.
#include <cuda.h>

#include "qlin_attend.cuh"
#include "qlin_paged.cuh"

namespace qlin {

constexpr int kSharedSoftmaxWarps = 8, kSharedLoadWarp = kSharedSoftmaxWarps, kSharedWidenWarp = kSharedLoadWarp + 1, kSharedWidenWarps = 2;
constexpr int kSharedMmaWarp = kSharedWidenWarp + kSharedWidenWarps;
constexpr int kMostBox = 32;  // keys of a copy
constexpr int kSharedThreads = (kSharedMmaWarp + 1) * 32;
// As in the attention of prompts: 168 registers a thread at first (64,512 in all), 216 for the softmax once the others are down to 72.
constexpr int kSharedSoftmaxRegs = 216, kSharedOtherRegs = 72;

struct SharedAux {
  uint64_t q_full[2], kv_full[8], kv_empty[8], raw_full[8], raw_empty[8], s_full[2], p_full[2][2], o_full[2], drain;
  uint32_t tmem_base;
  int abort_flag;
};

template <typename QT, bool F8, int DP, bool PAIR>
struct SharedCfg {
  using T = typename std::conditional<F8, __half, QT>::type;  // type of the products
  static constexpr bool HALF = std::is_same<T, __half>::value;
  static constexpr int ES = F8 ? 1 : 2;
  static constexpr int CHUNKS = DP / 64;
  static constexpr int TILE_BYTES = CHUNKS * kChunkBytes;
  static constexpr int Q_TILES = PAIR ? 2 : 1;
  static constexpr int STAGES = F8 ? (DP == 128 ? 3 : 6) : DP == 128 ? 5 : 8;
  static constexpr int RAW_BYTES = kKeys * DP, RAW = F8 ? (DP == 128 ? 4 : 6) : 0;  // tiles of codes
  static constexpr int KV_OFFSET = Q_TILES * TILE_BYTES;
  static constexpr int RAW_OFFSET = KV_OFFSET + STAGES * TILE_BYTES;
  // 32 rows of 32 outputs for each softmax warp: over the queries of the warp's own tile, which are no longer needed, or where the streams share these, beside the tiles
  static constexpr int OUT_OFFSET = PAIR ? 0 : RAW_OFFSET + RAW * RAW_BYTES, OUT_BYTES = 4096;
  static constexpr int AUX_OFFSET = RAW_OFFSET + RAW * RAW_BYTES + (PAIR ? 0 : kSharedSoftmaxWarps * OUT_BYTES);
  static constexpr int SMEM_BYTES = AUX_OFFSET + static_cast<int>(sizeof(SharedAux));
  // The reference may lie SLACK (in powers of two) below the maximum, and fp16 weights carry a factor of 2^SHIFT: they stay below 2^16, lose bits under 2^-26 of the largest only, and the
  // least of them, which a weight is kept at for the sake of infinite values, is 2^-36 of it, as in the attention over pages.
  static constexpr float SHIFT = HALF ? 12.0f : 0.0f, SLACK = HALF ? 3.875f : kSlack;
  static constexpr uint32_t FMT = HALF ? 0u : 1u;
  static constexpr uint32_t IDESC_S = make_idesc(1u, FMT, kRows, kKeys);
  static constexpr uint32_t IDESC_O = make_idesc(1u, FMT, kRows, DP) | (1u << 16);  // V is read with its head dimension contiguous
  static_assert(SMEM_BYTES <= 232448, "fits a block's shared memory");
};

// 16-byte piece c of a row of a tile.
__device__ __forceinline__ uint32_t tile_piece(int row, int c) { return static_cast<uint32_t>((c >> 3) * kChunkBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4)); }

// One tile of logits to weights; `left` columns are keys.
template <typename C, int DP, bool MASKED, bool FLOOR>
__device__ __forceinline__ void shared_softmax(uint32_t s_addr, uint32_t o_addr, float cl2, float slack, int left, bool first, uint64_t* p_full, float& m, float& l) {
  using T = typename C::T;
  uint32_t x[4][32];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_issue32(s_addr + 32 * c, x[c]);
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_wait32(x[c]);
  if constexpr (MASKED) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (32 * c + j >= left) x[c][j] = 0xff800000u;
  }
  Largest top(x);
#pragma unroll
  for (int n = 0; n < 15; ++n) top.step(x, n);
  const float most = top.result();
  // The reference follows the maximum only when that has outgrown it by 2^SLACK.  NaN or an infinity among the logits makes it NaN, and with it the row.
  // The difference, which is exact for numbers this near each other, is compared: m + slack rounds to a whole place of a large m, up to twice the slack, and 2^(2 SLACK + SHIFT) is
  // no fp16 number.
  const bool grow = m == -INFINITY ? !(most <= m) : !(most - m <= slack);
  if (first || __any_sync(0xffffffffu, grow)) {
    const float next = !grow ? m : (most == INFINITY ? __int_as_float(0x7fc00000) : most);
    if (!first) {
      const float keep = m == next ? 1.0f : exp2f((m - next) * cl2);
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
  }
  const float ref = m == -INFINITY ? 0.0f : m;
  const uint64_t minus = pair64(-ref, -ref), times = pair64(cl2, cl2), shift = pair64(C::SHIFT, C::SHIFT);
  uint64_t sum[2] = {0, 0};
  weigh<T, 0, 64>(
      x, [&](uint64_t pair) { return fma2(add2(pair, minus), times, shift); }, sum, [](int) {},
      [&](int c, const uint32_t(&words)[16]) {
        if constexpr (FLOOR) {  // not to zero in fp16, so that an infinite value stays one; NaN is in the sum
          uint32_t w[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&words[j]), __half2half2(__ushort_as_half(1)));
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
          }
          tmem_st16(s_addr + 16 * c, w);
        } else {
          tmem_st16(s_addr + 16 * c, words);
        }
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

// A box of keys of one page, [keys][64 elements or a row of codes].
__device__ __forceinline__ void box_load(uint32_t bar, uint32_t dst, const void* tmap, int32_t x, int32_t slot, int32_t head, int32_t page) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, {%3, %4, %5, %6}], [%0];" ::"r"(bar), "r"(dst),
               "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(slot), "r"(head), "r"(page)
               : "memory");
}

template <typename QT, bool F8, int DP, bool PAIR>
__global__ void __launch_bounds__(kSharedThreads, 1) shared_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                                                                    const __grid_constant__ PagedParams p) {
  using C = SharedCfg<QT, F8, DP, PAIR>;
  using T = typename C::T;
  extern __shared__ __align__(1024) uint8_t shared_tiles[];
  uint8_t* const smem = shared_tiles;
  SharedAux* aux = reinterpret_cast<SharedAux*>(smem + C::AUX_OFFSET);
  volatile int* abort_flag = &aux->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_launch();
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0 && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_ALIGN));
    return;
  }
  if (blockIdx.x == 0) check_groups(p);
  const int splits = p.pre.splits, block_splits = PAIR ? splits : (splits + 1) / 2;
  const int part = blockIdx.x % block_splits;
  int kvh, g, unit;
  if (!shared_unit(p, blockIdx.x / block_splits, C::Q_TILES * kRows, kvh, g, unit)) return;
  const Common common = common_keys(p, g, p.pre.groups[g], p.pre.groups[g + 1], threadIdx.x == 0);
  const int keys = common.to - common.from, per = keys_per_split(keys, splits);
  const int rows = common.sequences * p.group - unit * C::Q_TILES * kRows;  // from the block's first one on
  // of each stream: its split, the first of its keys, their number; and the tiles of both
  const auto split_of = [&](int i) { return PAIR ? part : 2 * part + i; };
  const auto begin_of = [&](int i) { return common.from + split_of(i) * per; };
  const auto count_of = [&](int i) { return (PAIR ? rows > i * kRows : split_of(i) < splits) ? max(0, min(common.to, begin_of(i) + per) - begin_of(i)) : 0; };
  const int tiles0 = uniform((count_of(0) + kKeys - 1) / kKeys), tiles1 = uniform((count_of(1) + kKeys - 1) / kKeys);
  if (rows <= 0 || tiles0 == 0) return;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) {
      mbar_init(&aux->kv_full[i], 1);
      mbar_init(&aux->kv_empty[i], 1);
      mbar_init(&aux->raw_full[i], 1);
      mbar_init(&aux->raw_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&aux->q_full[i], kRows);
      mbar_init(&aux->s_full[i], 1);
      mbar_init(&aux->p_full[i][0], kRows);
      mbar_init(&aux->p_full[i][1], kRows);
      mbar_init(&aux->o_full[i], 1);
    }
    mbar_init(&aux->drain, 1);
    aux->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kSharedMmaWarp) {
    tmem_alloc(&aux->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = aux->tmem_base;  // S 0, S 1 (128 columns each), O 0, O 1 (DP columns each)
  bool ok = true, timed_out = false;

  if (warp >= kSharedSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSharedOtherRegs));
    // The tiles in the order in which the products take them: `tile(stream, values, t)` until it says no.
    const auto every_tile = [&](auto tile) {
      if constexpr (PAIR) {
        for (int t = 0; t < tiles0; ++t)
          if (!tile(0, false, t) || !tile(0, true, t)) return;
      } else {
        if (!tile(0, false, 0) || (tiles1 > 0 && !tile(1, false, 0))) return;
        for (int t = 0; t < tiles0; ++t)
          for (int i = 0; i < 2; ++i) {
            const int mine = i ? tiles1 : tiles0;
            if (t < mine && !tile(i, true, t)) return;
            if (t + 1 < mine && !tile(i, false, t + 1)) return;
          }
      }
    };
    if (warp == kSharedLoadWarp) {
      // ------------------------------------------------------------------ loads: lane i brings the i-th box of a tile
      constexpr int RING = F8 ? C::RAW : C::STAGES, BYTES = F8 ? C::RAW_BYTES : C::TILE_BYTES;
      constexpr int CHUNKS = F8 ? 1 : C::CHUNKS, ROW = F8 ? DP : 128;  // pieces of a row, bytes of one
      uint64_t* const full = F8 ? aux->raw_full : aux->kv_full;
      uint64_t* const empty = F8 ? aux->raw_empty : aux->kv_empty;
      const uint32_t ring = smem_u32(smem) + (F8 ? C::RAW_OFFSET : C::KV_OFFSET);
      const int32_t* table = p.pre.table + g * p.pre.table_stride;
      const int box = p.pre.align;
      bool bad_page = false;
      uint32_t s = 0, ph = 1;
      int issued = 0;
      every_tile([&](int i, bool values, int t) {
        const int key = begin_of(i) + t * kKeys + lane * box, left = min(count_of(i) - t * kKeys, kKeys);  // a multiple of the box
        const bool mine = lane * box < left;
        const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / p.a.page_size;
        int page = mine ? table[pg] : 0;
        ok = uniform_wait(&empty[s], ph, abort_flag);
        if (!ok) return false;
        if (page < 0 || page >= p.a.num_pages) {
          bad_page = true;
          page = 0;
        }
        const uint32_t dst = ring + s * BYTES;
        if (left < kKeys) {  // rows behind the last key are zeros: what lay there before meets weights of zero, but may be infinite
          for (int at = left * ROW / 16 + lane; at < kKeys * ROW / 16; at += 32)
            for (int c = 0; c < CHUNKS; ++c) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + c * kChunkBytes + at * 16), "r"(0u) : "memory");
          fence_proxy_async();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>(left * ROW * CHUNKS));
        __syncwarp();
        if (mine)
          for (int c = 0; c < CHUNKS; ++c)
            box_load(smem_u32(&full[s]), dst + c * kChunkBytes + lane * box * ROW, values ? &tmap_v : &tmap_k, c * 64, key - pg * p.a.page_size, kvh, page);
        __syncwarp();
        ++issued;
        if (++s == RING) {
          s = 0;
          ph ^= 1u;
        }
        return true;
      });
      if (!ok) {  // copies in flight land before the block retires
        if (lane == 0) {
          timed_out = !*abort_flag;
          *abort_flag = 1;
        }
        for (int n = max(0, issued - RING); n < issued; ++n) mbar_wait_drain(&full[n % RING], (n / RING) & 1);
      }
      if (bad_page && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
      __syncwarp();
    } else if (warp < kSharedMmaWarp) {
      // ------------------------------------------------------------------ codes to fp16, every other tile
      if constexpr (F8) {
        constexpr int CH = DP / 16, AT_ONCE = 32 / CH;  // 16-byte pieces of a row of codes, rows that a warp's instruction takes
        const int lrow = lane / CH, lc = lane % CH;
        // lanes of the second 64 dimensions write their halves in the other order: eight lanes meet all banks
        const bool swap = lc >= 4;
        int n = 0;
        every_tile([&](int, bool, int) {
          const int turn = n++;
          if (turn % kSharedWidenWarps != warp - kSharedWidenWarp) return true;
          const int r = turn % C::RAW, s = turn % C::STAGES;
          ok = uniform_wait(&aux->raw_full[r], (turn / C::RAW) & 1, abort_flag, &aux->kv_empty[s], ((turn / C::STAGES) & 1) ^ 1);
          if (!ok) return false;
          const uint32_t from = smem_u32(smem) + C::RAW_OFFSET + r * C::RAW_BYTES, dst = smem_u32(smem) + C::KV_OFFSET + s * C::TILE_BYTES;
#pragma unroll 4
          for (int k = 0; k < kKeys / AT_ONCE; ++k) {
            const int row = k * AT_ONCE + lrow;
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from + piece<DP>(row, lc)) : "memory");
            const uint32_t x = swap ? v.z : v.x, y = swap ? v.w : v.y, z = swap ? v.x : v.z, w = swap ? v.y : v.w;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + tile_piece(row, 2 * lc + (swap ? 1 : 0))), "r"(widen_lo(x)), "r"(widen_hi(x)), "r"(widen_lo(y)),
                         "r"(widen_hi(y))
                         : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + tile_piece(row, 2 * lc + (swap ? 0 : 1))), "r"(widen_lo(z)), "r"(widen_hi(z)), "r"(widen_lo(w)),
                         "r"(widen_hi(w))
                         : "memory");
          }
          fence_proxy_async();  // what all lanes wrote is there for the tensor core, and what they read may be written over
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&aux->kv_full[s]);
            mbar_arrive(&aux->raw_empty[r]);
          }
          return true;
        });
        if (!ok && lane == 0) {
          timed_out = !*abort_flag;
          *abort_flag = 1;
        }
        __syncwarp();
      }
    } else {
      // ------------------------------------------------------------------ products
      const uint32_t base = (smem_u32(smem) & 0x3FFFFu) >> 4, d0 = uniform(tmem);
      uint32_t s = 0, ph = 0, p_ph = 0;  // bit i of the last: stream i
      const auto step = [&]() {
        if (++s == C::STAGES) {
          s = 0;
          ph ^= 1u;
        }
      };
      const auto logits = [&](int i, uint32_t stage) {
        const uint32_t q = PAIR ? i * C::TILE_BYTES : 0;
#pragma unroll
        for (int c = 0; c < C::CHUNKS; ++c)
          mma4_ss(d0 + i * kKeys, (base + ((q + c * kChunkBytes) >> 4)) | kRowsLow, (base + ((C::KV_OFFSET + c * kChunkBytes) >> 4) + stage * (C::TILE_BYTES >> 4)) | kRowsLow,
                  C::IDESC_S, c > 0);
        tc_commit_elect(&aux->s_full[i]);
      };
      const auto first_logits = [&](int i, uint32_t stage) {
        if (PAIR || i == 0) ok = uniform_wait(&aux->q_full[i], 0, abort_flag);
        if (!ok) return;
        tc_fence_after();
        logits(i, stage);
      };
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
      if constexpr (PAIR) {
        const bool second = tiles1 > 0;
        ok = uniform_wait(&aux->kv_full[0], 0, abort_flag);
        step();
        if (ok) first_logits(0, 0);
        if (ok && second) first_logits(1, 0);
        if (ok) tc_commit_elect(&aux->kv_empty[0]);
        for (int t = 0; t < tiles0 && ok; ++t) {
          const bool more = t + 1 < tiles0;
          const uint32_t sv = s, v_ph = ph;
          step();
          const uint32_t sk = s, k_ph = ph;
          if (more) step();
          ok = uniform_wait(&aux->kv_full[sv], v_ph, abort_flag, more ? &aux->kv_full[sk] : nullptr, k_ph);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const bool mine = i == 0 || second;
            if (ok && mine) {
              outputs(i, sv, t == 0);
              if (ok && !more) tc_commit_elect(&aux->o_full[i]);
            }
            if (ok && i == (second ? 1 : 0)) tc_commit_elect(&aux->kv_empty[sv]);
            if (ok && mine && more) logits(i, sk);
          }
          if (ok && more) tc_commit_elect(&aux->kv_empty[sk]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!ok || (i ? tiles1 : tiles0) == 0) continue;
          const uint32_t sk = s;
          ok = uniform_wait(&aux->kv_full[sk], ph, abort_flag);
          step();
          if (ok) first_logits(i, sk);
          if (ok) tc_commit_elect(&aux->kv_empty[sk]);
        }
        for (int t = 0; t < tiles0 && ok; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int mine = i ? tiles1 : tiles0;
            if (!ok || t >= mine) continue;
            const bool more = t + 1 < mine;
            const uint32_t sv = s, v_ph = ph;
            step();
            const uint32_t sk = s, k_ph = ph;
            if (more) step();
            ok = uniform_wait(&aux->kv_full[sv], v_ph, abort_flag, more ? &aux->kv_full[sk] : nullptr, k_ph);
            if (ok) outputs(i, sv, t == 0);
            if (!ok) continue;
            tc_commit_elect(&aux->kv_empty[sv]);
            if (more) {
              logits(i, sk);
              tc_commit_elect(&aux->kv_empty[sk]);
            } else {
              tc_commit_elect(&aux->o_full[i]);
            }
          }
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSharedSoftmaxRegs));
    const int i = warp >> 2, r = (warp & 3) * 32 + lane, D = p.a.head_dim;
    const int mine = i ? tiles1 : tiles0, count = count_of(i);
    if (mine > 0) {
      const int at = (PAIR ? i * kRows : 0) + r;  // among the block's rows
      const bool live = at < rows;
      const int row = unit * C::Q_TILES * kRows + at, sequence = common.first + row / p.group, head = kvh * p.group + row % p.group;
      const int64_t out_row = (static_cast<int64_t>(sequence) * p.a.q_heads + head) * splits + split_of(i);
      float cl2 = p.a.scale * 1.4426950408889634f;
      {
        uint32_t q[DP / 2];
        const QT* from = static_cast<const QT*>(p.a.q) + sequence * p.a.q_batch + head * p.a.q_head;
#pragma unroll
        for (int c = 0; c < DP / 8; ++c) {
          const uint4 v = live && 8 * c < D ? __ldg(reinterpret_cast<const uint4*>(from + 8 * c)) : make_uint4(0u, 0u, 0u, 0u);
          q[4 * c] = v.x;
          q[4 * c + 1] = v.y;
          q[4 * c + 2] = v.z;
          q[4 * c + 3] = v.w;
        }
        if constexpr (F8) {
          cl2 *= p.a.k_scale[kvh];
          // the keys' scale may have any sign: the maximum is looked for before it is applied
          const bool minus = cl2 < 0.0f, none = cl2 == 0.0f;
          cl2 = none ? 1.0f : fabsf(cl2);
#pragma unroll
          for (int c = 0; c < DP / 2; ++c) q[c] = none ? 0u : minus ? q[c] ^ 0x80008000u : q[c];
          if constexpr (std::is_same<QT, __nv_bfloat16>::value) {
            float top = 0.0f;
#pragma unroll
            for (int c = 0; c < DP / 2; ++c) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(q[c] << 16)), fabsf(__uint_as_float(q[c] & 0xffff0000u))));
            // 2^(13 - exponent), where that and its inverse are normal numbers
            const int e = static_cast<int>(__float_as_uint(top) >> 23), up_e = min(max(127 + 13 - (e - 127), 1), 253);
            const float up = top > 0.0f && e < 255 ? __uint_as_float(static_cast<uint32_t>(up_e) << 23) : 1.0f;
#pragma unroll
            for (int c = 0; c < DP / 2; ++c) q[c] = pack16<false>(__uint_as_float(q[c] << 16) * up, __uint_as_float(q[c] & 0xffff0000u) * up);
            cl2 /= up;
          }
        }
        if (PAIR || i == 0) {
          uint8_t* to = smem + (PAIR ? i * C::TILE_BYTES : 0);
#pragma unroll
          for (int c = 0; c < DP / 8; ++c) *reinterpret_cast<uint4*>(to + tile_piece(r, c)) = make_uint4(q[4 * c], q[4 * c + 1], q[4 * c + 2], q[4 * c + 3]);
          fence_proxy_async();
          mbar_arrive(&aux->q_full[i]);
        }
      }
      const float slack = C::SLACK / cl2;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_addr = tmem + lanes + i * kKeys, o_addr = tmem + lanes + 2 * kKeys + i * DP;
      float m = -INFINITY, l = 0.0f;
      constexpr bool FLOOR = C::HALF && !F8;
      for (int t = 0; t < mine && ok; ++t) {
        ok = uniform_wait(&aux->s_full[i], t & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const int left = count - t * kKeys;
        if (left >= kKeys) shared_softmax<C, DP, false, FLOOR>(s_addr, o_addr, cl2, slack, 0, t == 0, aux->p_full[i], m, l);
        else shared_softmax<C, DP, true, FLOOR>(s_addr, o_addr, cl2, slack, left, t == 0, aux->p_full[i], m, l);
      }
      if (ok) ok = uniform_wait(&aux->o_full[i], 0, abort_flag);
      if (ok) {
        tc_fence_after();
        constexpr float down = C::HALF ? 1.0f / 4096.0f : 1.0f;  // without the factor that fp16 weights carry
        if (live) p.pre.part_ml[out_row] = make_float2(m * cl2, l * down);
        // Rows go through shared memory, 32 outputs at a time, so that eight lanes write 128 bytes of a row together.
        const uint64_t to = live ? reinterpret_cast<uint64_t>(p.pre.part_o + out_row * D) : 0;
        uint8_t* stage = smem + C::OUT_OFFSET + (PAIR ? i * C::TILE_BYTES + (warp & 3) * C::OUT_BYTES : warp * C::OUT_BYTES);
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * c, o);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(__uint_as_float(o[4 * j]) * down, __uint_as_float(o[4 * j + 1]) * down,
                                                                                                  __uint_as_float(o[4 * j + 2]) * down, __uint_as_float(o[4 * j + 3]) * down);
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int from = 4 * k + (lane >> 3), j = lane & 7;
            const uint64_t row_to = __shfl_sync(0xffffffffu, to, from);
            const float4 v = *reinterpret_cast<const float4*>(stage + from * 128 + ((j ^ (from & 7)) << 4));
            if (row_to != 0 && 32 * c + 4 * j < D) *reinterpret_cast<float4*>(reinterpret_cast<float*>(row_to) + 32 * c + 4 * j) = v;
          }
          __syncwarp();
        }
      }
      if (!ok && lane == 0) {
        timed_out = !*abort_flag;
        *abort_flag = 1;
      }
      __syncwarp();
    }
  }
  if (timed_out && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_TIMEOUT));
  tc_fence_before();
  __syncthreads();
  if (warp == kSharedMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The keys of a page that one copy takes: a power of two that divides the page, so that a box lies in one page; 0 where there is none of 8 or the strides are no tensor map's.
int prefix_box(const qlin_paged_attention_args& a) {
  int box = a.page_size & -a.page_size;
  if (box > kMostBox) box = kMostBox;
  const int64_t size = a.cache_dtype == QLIN_DT_F8E4M3 ? 1 : 2, most = int64_t{1} << 38;
  const auto fits = [&](int64_t stride, int64_t n) { return n <= 1 || (stride > 0 && stride * size < most); };
  return box >= 8 && fits(a.slot_stride, a.page_size) && fits(a.head_stride, a.kv_heads) && fits(a.page_stride, a.num_pages) && tensor_map_encoder() != nullptr ? box : 0;
}
// [pages, kv heads, slots, head_dim] read in boxes of `box` keys of one head; head dimensions past the end are zeros.
static int page_map(CUtensorMap* tm, const void* base, const qlin_paged_attention_args& a, int box) {
  using Fn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                          CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  const Fn enc = reinterpret_cast<Fn>(tensor_map_encoder());
  const bool f8 = a.cache_dtype == QLIN_DT_F8E4M3;
  const int64_t size = f8 ? 1 : 2, row = (a.head_dim * size + 15) / 16 * 16;  // stands in for the stride of a dimension with one entry
  const int width = f8 ? (a.head_dim <= 64 ? 64 : 128) : 64;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.page_size), static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.num_pages)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(a.page_size > 1 ? a.slot_stride * size : row), static_cast<cuuint64_t>(a.kv_heads > 1 ? a.head_stride * size : row),
                           static_cast<cuuint64_t>(a.num_pages > 1 ? a.page_stride * size : row)};
  cuuint32_t boxes[4] = {static_cast<cuuint32_t>(width), static_cast<cuuint32_t>(box), 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(tm, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : a.dtype == QLIN_DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                         const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         width * size == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(QLIN_ERR_BAD_ALIGN, "qlin_prefix_attention: cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
  return QLIN_OK;
}

template <typename QT, bool F8, int DP, bool PAIR>
static int launch_shared(const PagedParams& p, cudaStream_t stream) {
  using C = SharedCfg<QT, F8, DP, PAIR>;
  const auto kernel = shared_kernel<QT, F8, DP, PAIR>;
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
    if (attr.numRegs * kSharedThreads < 32 * (kSharedSoftmaxWarps * kSharedSoftmaxRegs + 4 * kSharedOtherRegs))
      return fail(QLIN_ERR_LAUNCH, "qlin_prefix_attention: built with %d registers a thread, too few for its split", attr.numRegs);
    configured[dev] = true;
  }
  CUtensorMap tk, tv;
  int rc = page_map(&tk, p.a.k_pages, p.a, p.pre.align);
  if (rc == QLIN_OK) rc = page_map(&tv, p.a.v_pages, p.a, p.pre.align);
  if (rc != QLIN_OK) return rc;
  shared_kernel<QT, F8, DP, PAIR><<<static_cast<unsigned>(p.pre.blocks), kSharedThreads, C::SMEM_BYTES, stream>>>(tk, tv, p);
  QLIN_CHECK_LAUNCH("qlin_prefix_attention");
  return QLIN_OK;
}
template <typename QT, bool F8>
static int pick_shared(const PagedParams& p, bool pair, cudaStream_t s) {
  if (p.a.head_dim <= 64) return pair ? launch_shared<QT, F8, 64, true>(p, s) : launch_shared<QT, F8, 64, false>(p, s);
  return pair ? launch_shared<QT, F8, 128, true>(p, s) : launch_shared<QT, F8, 128, false>(p, s);
}

int launch_prefix_tc(const PagedParams& p, bool pair, cudaStream_t s) {
  const bool f8 = p.a.cache_dtype == QLIN_DT_F8E4M3;
  if (p.a.dtype == QLIN_DT_BF16) return f8 ? pick_shared<__nv_bfloat16, true>(p, pair, s) : pick_shared<__nv_bfloat16, false>(p, pair, s);
  return f8 ? pick_shared<__half, true>(p, pair, s) : pick_shared<__half, false>(p, pair, s);
}

}  // namespace qlin
