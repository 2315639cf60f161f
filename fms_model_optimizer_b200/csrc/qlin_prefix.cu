// qlin_prefix_attention: one new token of every sequence against its keys in a paged cache, where groups of sequences share the first of them.
//
// The softmax of a row splits into any parts of its keys, each with its own maximum and sums.  Here the keys of the prefix that all sequences of a group
// see are one part: the queries of all of them are the columns of the products (eight or sixteen a block, or a tile or two of 128), and each key is loaded once for these.
// What else a sequence sees, its own keys, and those of the prefix that its window or length sets apart from the others', is the part that
// qlin_paged_attention's kernel reads, whose blocks then take in the sums over the prefix.  No row of a product is masked that way: what a sequence does not see
// is not loaded beside its query, NaN and infinities included.
//
// What bounds it: HBM, each key of a prefix once for a block's columns and each own key once, while a group has few rows; then the products, which groups of 32 rows and more (48 with e4m3) have on tcgen05
// (qlin_prefix_tc.cu).  The launch for the own keys begins while the one for the prefixes ends, and waits for its sums only when it joins them.
//
// Measured (device time, 32 + 8 heads of 128): 2 x 64 sequences behind 32768 keys with up to 300 of their own in bf16 86 us, 774 TFLOP/s, 0.47 of the burst rate (72 for the prefixes, the
// own keys 15 behind them; 103 a call in a long run, whose clock falls); 61 behind 8200 with up to 515 in e4m3 39 us (40 a call); 4 behind 2048 with 128 in bf16 12.9 us, two launches of 8
// that overlap (14.4 a call).
// Beside the attention over pages, which reads the prefix for each sequence: 16 behind 8192 with 128 30 us, 64 there; 32 behind 2048 25.5 and 37.5, 16 22.7 and 24.7, 8 15.8 and 18.9, 4
// 13.2 and 13.8; but 4 behind 512 with 50 11.6 and 7.2, and 16 16.0 and 14.5: a prefix of a few hundred keys, which L2 holds, does not pay for its launch.
//
// The host knows neither the groups' sizes nor the prefixes' lengths, which lie on the device; the rules below go by averages and by the tables' widths.  So 64 sequences behind 32768 keys with
// 100 of their own take 55 us, with 8 single requests in the same call 161 and with 63 of them 455 (838 over pages): the average says few rows and few splits.  And 15 sequences behind
// 8192 keys with a 16th of 100 take 82 us (63 over pages), since what all of them see ends there and the rest is left to each, unsplit.
#include "qlin_paged.cuh"

namespace qlin {

// Rows of a group (its sequences times the query heads of a kv head) from which on the tensor cores' 128-row tiles take the prefix, and above which a
// block has two of them.
// Measured with 128 keys of their own, mma.sync and tcgen05 in us: 8 sequences (32 rows) behind 8192 in bf16 24.4 and 22.4, in e4m3 25.1 and 26.6; 16 (64 rows) 42 and 34, 42 and 37.
constexpr int kRowsTensor = 32, kRowsTensorE4m3 = 48, kRowsPair = 128;
constexpr int kLongOwn = 2048;  // keys of its own that a sequence may have for fewer warps than four

struct PrefixPlan {
  Splits own;
  int32_t units, splits, columns;  // of the launch for the prefixes: blocks of columns of all kv heads at most, splits of the keys, columns of a block
  int32_t blocks;                  // of that launch
  int32_t align;                   // see SharedPrefix
  int32_t warps;                   // of a sequence's kv head in the launch for its own keys
  int64_t own_floats, shared_floats;  // of the workspace
};
static PrefixPlan plan_prefix(const qlin_prefix_attention_args& a) {
  PrefixPlan plan = {};
  plan.align = 1;
  const int group = a.own.q_heads / a.own.kv_heads;
  // the tables' widths say how many keys of their own sequences may have
  qlin_paged_attention_args own = a.own;
  own.max_pages = a.own.max_pages > a.max_prefix_pages ? a.own.max_pages - a.max_prefix_pages + 1 : 1;
  const int head_blocks = (group + heads_per_block(group) - 1) / heads_per_block(group);
  plan.own = choose_splits(own, head_blocks);
  // Warps that are resident at once, or nearly, if the keys are few enough for that to count: a second wave of blocks costs the latency of the lookups, the keys and the join again.
  const bool f8 = a.own.cache_dtype == QLIN_DT_F8E4M3;
  const int64_t units = static_cast<int64_t>(a.own.batch) * a.own.kv_heads * head_blocks, slots = static_cast<int64_t>(group <= 8 ? 3 : 2) * kPagedWarps * sm_count(), nearly = slots + slots / 4;
  plan.warps = units * 4 <= nearly || static_cast<int64_t>(own.max_pages) * own.page_size > kLongOwn ? 4 : units * 2 <= nearly ? 2 : 1;
  if (plan.warps < 4 || (plan.own.cluster && units * 4 * plan.own.n > nearly)) plan.own = Splits{1, 0};
  const int64_t rows = static_cast<int64_t>(a.own.batch) * a.own.q_heads;
  if (plan.own.n > 1 && !plan.own.cluster) plan.own_floats = rows * plan.own.n * (a.own.head_dim + 2);
  const int64_t keys = static_cast<int64_t>(a.max_prefix_pages) * a.own.page_size;
  if (keys > 0 && a.own.num_pages > 0) {
    const int64_t per_head = rows / a.own.kv_heads, each = (per_head + a.num_groups - 1) / a.num_groups;  // rows of a kv head, and of a group on average
    const int box = prefix_box(a.own);
    plan.columns = box == 0 || each < (f8 ? kRowsTensorE4m3 : kRowsTensor) ? (each > 8 ? 16 : 8) : each > kRowsPair ? 256 : 128;
    if (plan.columns >= 128) plan.align = box;
    const int64_t blocks = per_head / plan.columns + a.num_groups;  // a group has one block that is not full at most
    if (blocks * a.own.kv_heads > (1 << 24)) return plan;
    plan.units = static_cast<int32_t>(blocks * a.own.kv_heads);
    const int64_t expected = a.num_groups * ((each + plan.columns - 1) / plan.columns) * a.own.kv_heads, most = (keys + kSharedStep - 1) / kSharedStep;
    if (plan.columns >= 128) {
      // one block an SM, none with fewer than two tiles of keys for each of its streams (16 sequences behind 2048 keys 24.2 us, with four 30.5); 128 rows take two splits at once
      const int streams = plan.columns == 128 ? 2 : 1;
      int64_t each_unit = sm_count() / expected;
      if (each_unit > most / (2 * streams)) each_unit = most / (2 * streams);
      if (each_unit < 1) each_unit = 1;
      plan.splits = static_cast<int32_t>(each_unit * streams);
      plan.blocks = plan.units * static_cast<int32_t>(each_unit);
    } else {
      const int64_t want = (2 * sm_count() + expected - 1) / expected;
      plan.splits = static_cast<int32_t>(want < most ? want : most);
      plan.blocks = plan.units * plan.splits;
    }
    plan.shared_floats = rows * plan.splits * (a.own.head_dim + 2);
  }
  return plan;
}

static int check_prefix(const qlin_prefix_attention_args* a) {
  if (a == nullptr) return fail(QLIN_ERR_NULL, "qlin_prefix_attention: args is NULL");
  const int rc = check_paged(&a->own, "qlin_prefix_attention");
  if (rc != QLIN_OK) return rc;
  if (a->num_groups < 0 || a->max_prefix_pages < 0 || (a->own.batch > 0 && a->num_groups < 1))
    return fail(QLIN_ERR_BAD_SHAPE, "qlin_prefix_attention: at least one group is wanted, and no negative width");
  if (a->num_groups > (1 << 20)) return fail(QLIN_ERR_TOO_LARGE, "qlin_prefix_attention: at most 2^20 groups");
  if (static_cast<int64_t>(a->max_prefix_pages) * a->own.page_size > (1 << 30)) return fail(QLIN_ERR_TOO_LARGE, "qlin_prefix_attention: at most 2^30 keys a prefix");
  return QLIN_OK;
}

template <typename QT, bool F8, int DP, int NT>
static int launch_own(const PagedParams& p, int warps, cudaStream_t s) {
  if (warps == 1) return launch_paged<QT, F8, DP, NT, kOwn, 1>(p, s);
  if (warps == 2) return launch_paged<QT, F8, DP, NT, kOwn, 2>(p, s);
  return launch_paged<QT, F8, DP, NT, kOwn>(p, s);
}
template <typename QT, bool F8, int DP>
static int launch_prefix(const PagedParams& p, const PrefixPlan& plan, cudaStream_t s) {
  if (p.pre.blocks > 0) {
    const int rc = plan.columns >= 128 ? launch_prefix_tc(p, plan.columns == 256, s) : plan.columns == 16 ? launch_paged<QT, F8, DP, 2, kShared>(p, s) : launch_paged<QT, F8, DP, 1, kShared>(p, s);
    if (rc != QLIN_OK) return rc;
  }
  return heads_per_block(p.group) == 16 ? launch_own<QT, F8, DP, 2>(p, plan.warps, s) : launch_own<QT, F8, DP, 1>(p, plan.warps, s);
}
template <typename QT, bool F8>
static int pick_prefix(const PagedParams& p, const PrefixPlan& plan, cudaStream_t s) {
  return p.a.head_dim <= 64 ? launch_prefix<QT, F8, 64>(p, plan, s) : launch_prefix<QT, F8, 128>(p, plan, s);
}

}  // namespace qlin

extern "C" int64_t qlin_prefix_attention_workspace_bytes(const qlin_prefix_attention_args* a) {
  using namespace qlin;
  const int rc = check_prefix(a);
  if (rc != QLIN_OK) return rc;
  if (a->own.batch == 0) return 0;
  const PrefixPlan plan = plan_prefix(*a);
  return (plan.own_floats + plan.shared_floats) * 4;
}

extern "C" int qlin_prefix_attention(const qlin_prefix_attention_args* a, void* stream) {
  using namespace qlin;
  int rc = check_prefix(a);
  if (rc != QLIN_OK) return rc;
  if (a->own.batch == 0) return QLIN_OK;
  rc = check_paged_pointers(&a->own, "qlin_prefix_attention");
  if (rc != QLIN_OK) return rc;
  if (a->groups == nullptr || a->prefix_lens == nullptr || (a->max_prefix_pages > 0 && (a->prefix_table == nullptr || (a->own.num_pages > 0 && (a->own.k_pages == nullptr || a->own.v_pages == nullptr)))))
    return fail(QLIN_ERR_NULL, "qlin_prefix_attention: groups, prefix_lens, prefix_table, k_pages or v_pages is NULL");
  const PrefixPlan plan = plan_prefix(*a);
  if (a->max_prefix_pages > 0 && a->own.num_pages > 0 && plan.blocks < 1) return fail(QLIN_ERR_TOO_LARGE, "qlin_prefix_attention: too many rows and groups");
  PagedParams p = {};
  p.a = a->own;
  p.group = a->own.q_heads / a->own.kv_heads;
  p.head_blocks = (p.group + heads_per_block(p.group) - 1) / heads_per_block(p.group);
  p.splits = plan.own.n;
  p.cluster = plan.own.cluster;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a->own.page_size == 1 << i) p.page_shift = i;
  const int64_t rows = static_cast<int64_t>(a->own.batch) * a->own.q_heads;
  if (plan.own_floats + plan.shared_floats > 0) {
    if (a->own.workspace == nullptr) return fail(QLIN_ERR_NULL, "qlin_prefix_attention: workspace is NULL");
    if (!aligned16(a->own.workspace)) return fail(QLIN_ERR_BAD_ALIGN, "qlin_prefix_attention: workspace must start on 16 bytes");
  }
  // outputs first, then maxima and sums: the former stay on 16 bytes
  float* at = static_cast<float*>(a->own.workspace);
  p.pre.part_o = at;
  p.part_o = at + rows * plan.splits * a->own.head_dim;
  const bool parts = plan.own_floats > 0;
  float* ml = p.part_o + (parts ? rows * plan.own.n * a->own.head_dim : 0);
  p.pre.part_ml = reinterpret_cast<float2*>(ml);
  p.part_ml = reinterpret_cast<float2*>(ml + rows * plan.splits * 2);
  p.pre.table = a->prefix_table;
  p.pre.lens = a->prefix_lens;
  p.pre.groups = a->groups;
  p.pre.table_stride = a->prefix_stride;
  p.pre.count = a->num_groups;
  p.pre.max_pages = a->max_prefix_pages;
  p.pre.splits = plan.splits > 0 ? plan.splits : 1;
  p.pre.blocks = plan.blocks;
  p.pre.align = plan.align;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool f8 = a->own.cache_dtype == QLIN_DT_F8E4M3;
  if (a->own.dtype == QLIN_DT_BF16) return f8 ? pick_prefix<__nv_bfloat16, true>(p, plan, s) : pick_prefix<__nv_bfloat16, false>(p, plan, s);
  return f8 ? pick_prefix<__half, true>(p, plan, s) : pick_prefix<__half, false>(p, plan, s);
}
