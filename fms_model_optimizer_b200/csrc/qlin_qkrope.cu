// qlin_qk_rope: per-head RMS norm of queries and keys, rotary embedding and the write of k and v into the paged cache, one pass.
//
//   y = x * rsqrt(mean x^2 + eps) * w,   z[i] = y[i] c[i] - y[i + r/2] s[i],   z[i + r/2] = y[i + r/2] c[i] + y[i] s[i]
//
// What bounds it: HBM, with one read and one write per element of q and k, a read of v and a write of k and v in the cache's type
// on top.  A block owns a token, so that the token's rows of cos and sin come from L1 for all but the first head.  A head
// belongs to a group of G lanes, the smallest power of two (from four up) that covers head_dim / 16; a lane holds the two 8-element
// chunks that the rotation pairs (or two neighbouring ones behind the rotated part), so the rotation stays inside the lane and
// only the sum of squares crosses lanes.  Everything is fp32 between the load and the one rounding of each output; the e4m3 code
// is made from the unrounded value.  Measured (device time): 16384 tokens of 32 + 8 heads of 128 in bf16 with cache 87 us, 5.1 TB/s =
// 0.78 of the copy rate; 1 token 3.5 us, a position, a row of cos and sin and a launch behind one another.
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "qlin_internal.h"

namespace qlin {

struct QkRopeParams {
  qlin_qk_rope_args a;
};

template <typename T>
struct Raw8 {  // eight elements as they lie in memory
  uint4 v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
__device__ __forceinline__ float2 pair_of(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 pair_of(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <typename T>
__device__ __forceinline__ void widen(const Raw8<T>& r, float (&f)[8]) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[4 * i] = __uint_as_float(r.v[i].x);
      f[4 * i + 1] = __uint_as_float(r.v[i].y);
      f[4 * i + 2] = __uint_as_float(r.v[i].z);
      f[4 * i + 3] = __uint_as_float(r.v[i].w);
    }
  } else {
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = pair_of(w[i], T());
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  if constexpr (std::is_same<T, float>::value) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_pair(f[0], f[1], T()), pack_pair(f[2], f[3], T()), pack_pair(f[4], f[5], T()), pack_pair(f[6], f[7], T()));
  }
}
// Codes of x * rs, clamped to +-448 (NaN stays NaN), eight bytes.
__device__ __forceinline__ void store8_codes(uint8_t* p, const float (&f)[8], float rs) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i] * rs, f[4 * i + 1] * rs), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2] * rs, f[4 * i + 3] * rs), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

enum class Cache { kNone, kSame, kF8 };

// THREADS of a block, which has one token.  U: heads whose loads a group has in flight together.
template <typename T, typename W, Cache C, int G, int U, int THREADS>
__global__ void __launch_bounds__(THREADS, 640 / THREADS) qk_rope_kernel(const __grid_constant__ QkRopeParams pp) {
  const qlin_qk_rope_args& p = pp.a;
  const int64_t token = blockIdx.x;
  const int j = threadIdx.x % G, sub = threadIdx.x / G;
  constexpr int kSubs = THREADS / G;
  const bool live = j < p.head_dim / 16;
  const bool rot = j < p.rotary / 16;
  const int c0 = rot ? 8 * j : p.rotary + 16 * (j - p.rotary / 16), c1 = rot ? c0 + p.rotary / 2 : c0 + 8;
  const int pos = p.positions[token];
  const bool pos_ok = pos >= 0 && pos < p.table_rows;
  int64_t cache_row = -1;  // offset of the token's slot without the head's
  if constexpr (C != Cache::kNone) {
    const int64_t slot = p.slots[token];
    if (slot >= p.num_slots) {
      if (threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
    } else if (slot >= 0 && pos_ok) {
      cache_row = slot / p.page_size * p.page_stride + slot % p.page_size * p.slot_stride;
    }
  }
  if (!pos_ok && threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, static_cast<int32_t>(QLIN_ERR_BAD_SHAPE));
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = 1.0f;
    sn[i] = 0.0f;
  }
  if (rot && pos_ok) {
    const int64_t row = static_cast<int64_t>(pos) * (p.rotary / 2) + c0;
    widen(load8(p.cos + row), cs);
    widen(load8(p.sin + row), sn);
  }
  const int heads = p.q_heads + p.kv_heads, items = heads + (C != Cache::kNone ? p.kv_heads : 0);
  for (int base = 0; base < items; base += kSubs * U) {
    Raw8<T> ra[U], rb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int it = base + u * kSubs + sub;
      if (it < items && live) {
        const T* src = it < p.q_heads ? static_cast<const T*>(p.q) + token * p.q_token + it * p.q_head
                       : it < heads   ? static_cast<const T*>(p.k) + token * p.k_token + (it - p.q_heads) * p.k_head
                                      : static_cast<const T*>(p.v) + token * p.v_token + (it - heads) * p.v_head;
        ra[u] = load8(src + c0);
        rb[u] = load8(src + c1);
      } else {
        ra[u] = Raw8<T>{};
        rb[u] = Raw8<T>{};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int it = base + u * kSubs + sub;
      float a[8], b[8];
      widen(ra[u], a);
      widen(rb[u], b);
      const W* weight = static_cast<const W*>(it < p.q_heads ? p.q_weight : p.k_weight);
      if (p.q_weight != nullptr || p.k_weight != nullptr) {  // the same for every lane: the sum below is taken by whole warps
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += a[i] * a[i] + b[i] * b[i];
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (it < heads && weight != nullptr && live) {
          const float r = rsqrtf(sum / static_cast<float>(p.head_dim) + p.eps);
          float wa[8], wb[8];
          widen(load8(weight + c0), wa);
          widen(load8(weight + c1), wb);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            a[i] = a[i] * r * wa[i];
            b[i] = b[i] * r * wb[i];
          }
        }
      }
      if (it >= items || !live) continue;
      if (it < heads) {
        float za[8], zb[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          za[i] = a[i] * cs[i] - b[i] * sn[i];
          zb[i] = b[i] * cs[i] + a[i] * sn[i];
        }
        if (!pos_ok) {
#pragma unroll
          for (int i = 0; i < 8; ++i) za[i] = zb[i] = __int_as_float(0x7fc00000);
        }
        if (!rot) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            za[i] = pos_ok ? a[i] : za[i];
            zb[i] = pos_ok ? b[i] : zb[i];
          }
        }
        T* dst = it < p.q_heads ? static_cast<T*>(p.q_out) + (token * p.q_heads + it) * p.head_dim
                                : (p.k_out != nullptr ? static_cast<T*>(p.k_out) + (token * p.kv_heads + (it - p.q_heads)) * p.head_dim : nullptr);
        if (dst != nullptr) {
          store8(dst + c0, za);
          store8(dst + c1, zb);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a[i] = za[i];
          b[i] = zb[i];
        }
      }
      if constexpr (C != Cache::kNone) {
        if (it >= p.q_heads && cache_row >= 0) {
          const bool is_k = it < heads;
          const int h = it - (is_k ? p.q_heads : heads);
          const int64_t at = cache_row + h * p.head_stride;
          void* pages = is_k ? p.k_pages : p.v_pages;
          if constexpr (C == Cache::kF8) {
            const float rs = __fdiv_rn(1.0f, (is_k ? p.k_scale : p.v_scale)[h]);
            store8_codes(static_cast<uint8_t*>(pages) + at + c0, a, rs);
            store8_codes(static_cast<uint8_t*>(pages) + at + c1, b, rs);
          } else {
            store8(static_cast<T*>(pages) + at + c0, a);
            store8(static_cast<T*>(pages) + at + c1, b);
          }
        }
      }
    }
  }
}

// With many tokens a warp for each: what a block waits for (its position, then its rows of cos and sin) is spread over four times
// the data, and more blocks are in flight.  With few a block of four warps, so that no lane has many heads to go through.  Device time,
// one warp against four: 32 + 8 heads of 128 in bf16 with cache, 64 tokens 8.3 / 3.5 us, 1200 tokens 10.6 / 8.9, 2400 tokens 15.9 /
// 18.2, 16384 tokens 87 / 103; 12 + 12 heads of 64 with e4m3 cache, 1200 tokens 6.5 / 6.5, 2400 tokens 7.7 / 10.6.
template <typename T, typename W, Cache C, int G>
static int launch_qk_rope(const QkRopeParams& p, cudaStream_t s) {
  constexpr int U = std::is_same<T, float>::value ? 2 : 3;
  if (p.a.tokens >= 9 * sm_count()) {
    qk_rope_kernel<T, W, C, G, U, 32><<<p.a.tokens, 32, 0, s>>>(p);
  } else {
    qk_rope_kernel<T, W, C, G, U, 128><<<p.a.tokens, 128, 0, s>>>(p);
  }
  QLIN_CHECK_LAUNCH("qlin_qk_rope");
  return QLIN_OK;
}
template <typename T, typename W, Cache C>
static int pick_group(const QkRopeParams& p, cudaStream_t s) {
  const int lanes = p.a.head_dim / 16;
  if (lanes <= 4) return launch_qk_rope<T, W, C, 4>(p, s);
  if (lanes <= 8) return launch_qk_rope<T, W, C, 8>(p, s);
  if (lanes <= 16) return launch_qk_rope<T, W, C, 16>(p, s);
  return launch_qk_rope<T, W, C, 32>(p, s);
}
template <typename T, typename W>
static int pick_cache(const QkRopeParams& p, cudaStream_t s) {
  if (p.a.k_pages == nullptr) return pick_group<T, W, Cache::kNone>(p, s);
  if (p.a.cache_dtype == QLIN_DT_F8E4M3) return pick_group<T, W, Cache::kF8>(p, s);
  return pick_group<T, W, Cache::kSame>(p, s);
}
template <typename T>
static int pick_weight(const QkRopeParams& p, cudaStream_t s) {
  return p.a.weight_dtype == QLIN_DT_F32 ? pick_cache<T, float>(p, s) : pick_cache<T, T>(p, s);
}

}  // namespace qlin

extern "C" int qlin_qk_rope(const qlin_qk_rope_args* a, void* stream) {
  using namespace qlin;
  if (a == nullptr) return fail(QLIN_ERR_NULL, "qlin_qk_rope: args is NULL");
  if (a->tokens < 0 || a->q_heads < 1 || a->kv_heads < 1 || a->table_rows < 1) return fail(QLIN_ERR_BAD_SHAPE, "qlin_qk_rope: bad dimensions");
  if (a->head_dim < 16 || a->head_dim % 16 != 0 || a->head_dim > 512) return fail(QLIN_ERR_BAD_SHAPE, "qlin_qk_rope: head_dim must be a multiple of 16 up to 512");
  if (a->rotary < 16 || a->rotary % 16 != 0 || a->rotary > a->head_dim) return fail(QLIN_ERR_BAD_SHAPE, "qlin_qk_rope: rotary must be a multiple of 16 up to head_dim");
  if (a->q_heads > (1 << 20) || a->kv_heads > (1 << 20)) return fail(QLIN_ERR_TOO_LARGE, "qlin_qk_rope: too many heads");
  if (a->dtype != QLIN_DT_F32 && a->dtype != QLIN_DT_F16 && a->dtype != QLIN_DT_BF16) return fail(QLIN_ERR_BAD_DTYPE, "qlin_qk_rope: q and k must be fp32, fp16 or bf16");
  if ((a->q_weight != nullptr || a->k_weight != nullptr) && a->weight_dtype != a->dtype && a->weight_dtype != QLIN_DT_F32)
    return fail(QLIN_ERR_BAD_DTYPE, "qlin_qk_rope: the norm's weights must have the type of q and k, or be fp32");
  if (a->tokens == 0) return QLIN_OK;
  if (a->q == nullptr || a->k == nullptr || a->q_out == nullptr || a->cos == nullptr || a->sin == nullptr || a->positions == nullptr)
    return fail(QLIN_ERR_NULL, "qlin_qk_rope: q, k, q_out, cos, sin or positions is NULL");
  const int es = dtype_size(a->dtype);
  const auto off16 = [&](int64_t stride, int size) { return stride * size % 16 != 0; };
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->q_out) || !aligned16(a->k_out) || !aligned16(a->cos) || !aligned16(a->sin) || !aligned16(a->q_weight) ||
      !aligned16(a->k_weight) || off16(a->q_token, es) || off16(a->q_head, es) || off16(a->k_token, es) || off16(a->k_head, es))
    return fail(QLIN_ERR_BAD_ALIGN, "qlin_qk_rope: every row must start on 16 bytes");
  if (a->k_pages != nullptr) {
    if (a->v_pages == nullptr || a->v == nullptr || a->slots == nullptr) return fail(QLIN_ERR_NULL, "qlin_qk_rope: v_pages, v or slots is NULL");
    if (a->cache_dtype != a->dtype && a->cache_dtype != QLIN_DT_F8E4M3) return fail(QLIN_ERR_BAD_DTYPE, "qlin_qk_rope: the cache must have the type of k, or e4m3");
    const bool f8 = a->cache_dtype == QLIN_DT_F8E4M3;
    if (f8 && (a->k_scale == nullptr || a->v_scale == nullptr)) return fail(QLIN_ERR_NULL, "qlin_qk_rope: an e4m3 cache needs k_scale and v_scale");
    if (a->page_size < 1 || a->num_slots < 0) return fail(QLIN_ERR_BAD_SHAPE, "qlin_qk_rope: bad page size or number of slots");
    const int cs = f8 ? 1 : es;
    if (!aligned16(a->v) || !aligned16(a->k_pages) || !aligned16(a->v_pages) || off16(a->v_token, es) || off16(a->v_head, es) || off16(a->page_stride, cs) ||
        off16(a->head_stride, cs) || off16(a->slot_stride, cs))
      return fail(QLIN_ERR_BAD_ALIGN, "qlin_qk_rope: every row of v and of the cache must start on 16 bytes");
  }
  const QkRopeParams p{*a};
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == QLIN_DT_F32) return pick_cache<float, float>(p, s);
  return a->dtype == QLIN_DT_F16 ? pick_weight<__half>(p, s) : pick_weight<__nv_bfloat16>(p, s);
}
