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
#include "qlin_paged.cuh"

namespace qlin {

template <typename QT, bool F8>
static int pick_paged(const PagedParams& p, cudaStream_t s) {
  const bool wide = heads_per_block(p.group) == 16;
  if (p.a.head_dim <= 64) return wide ? launch_paged<QT, F8, 64, 2, kSingle>(p, s) : launch_paged<QT, F8, 64, 1, kSingle>(p, s);
  return wide ? launch_paged<QT, F8, 128, 2, kSingle>(p, s) : launch_paged<QT, F8, 128, 1, kSingle>(p, s);
}

}  // namespace qlin

extern "C" int64_t qlin_paged_attention_workspace_bytes(const qlin_paged_attention_args* a) {
  using namespace qlin;
  const int rc = check_paged(a, "qlin_paged_attention");
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
  const int rc = check_paged(a, "qlin_paged_attention");
  if (rc != QLIN_OK) return rc;
  if (a->batch == 0) return QLIN_OK;
  const int given = check_paged_pointers(a, "qlin_paged_attention");
  if (given != QLIN_OK) return given;
  const bool f8 = a->cache_dtype == QLIN_DT_F8E4M3;
  PagedParams p = {};
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
