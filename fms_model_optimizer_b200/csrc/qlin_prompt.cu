// qlin_prompt_attention: attention of packed prompts under a causal mask, a sliding window and first tokens that stay visible.
//
//   o_i = sum_j w_j v_j / sum_j w_j,   w_j = 2^(x_j - max x),   x_j = q_i.k_j scale log2(e),   j over the keys that i sees
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qlin_internal.h"

namespace qlin {

struct PromptParams {
  qlin_prompt_attention_args a;
  int32_t group;  // query heads per kv head
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
    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
    T* out = static_cast<T*>(p.a.out) + (static_cast<int64_t>(s.q0 + i) * p.a.q_heads + head) * D + lane * 4;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(acc[0] * r, acc[1] * r), pack2<T>(acc[2] * r, acc[3] * r));
  }
}

template <typename T>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const __grid_constant__ PromptParams p) {
  const int b = blockIdx.z, head = blockIdx.y;
  const Sequence s = sequence_of(p, b);
  if (s.bad) {
    if (threadIdx.x == 0 && p.a.status != nullptr) atomicExch(p.a.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
    return;
  }
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (i < s.n) attend_row<T>(p, s, i, head);
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
  if (a->batch == 0 || a->tokens_q == 0 || a->max_q == 0) return QLIN_OK;
  if (a->q == nullptr || a->out == nullptr || a->cu_q == nullptr || a->cu_k == nullptr) return fail(QLIN_ERR_NULL, "qlin_prompt_attention: q, out, cu_q or cu_k is NULL");
  if (a->tokens_k > 0 && (a->k == nullptr || a->v == nullptr)) return fail(QLIN_ERR_NULL, "qlin_prompt_attention: k or v is NULL");
  if (a->q_heads > 65535 || a->batch > 65535) return fail(QLIN_ERR_TOO_LARGE, "qlin_prompt_attention: at most 65535 heads and sequences");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) || a->q_token % 8 != 0 || a->q_head % 8 != 0 || a->k_token % 8 != 0 ||
      a->k_head % 8 != 0 || a->v_token % 8 != 0 || a->v_head % 8 != 0)
    return fail(QLIN_ERR_BAD_ALIGN, "qlin_prompt_attention: every row must start on 16 bytes");
  PromptParams p;
  p.a = *a;
  p.group = a->q_heads / a->kv_heads;
  p.cl2 = a->scale * 1.4426950408889634f;
  const dim3 grid(static_cast<unsigned>((a->max_q + 3) / 4), static_cast<unsigned>(a->q_heads), static_cast<unsigned>(a->batch));
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == QLIN_DT_BF16) {
    prompt_rows_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
  } else {
    prompt_rows_kernel<__half><<<grid, 128, 0, s>>>(p);
  }
  QLIN_CHECK_LAUNCH("qlin_prompt_attention");
  return QLIN_OK;
}
