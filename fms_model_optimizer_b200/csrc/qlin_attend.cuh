// Tiles of 128 queries against 128 keys on tcgen05, with a thread for each row of logits: what the attention of prompts (qlin_prompt.cu) and that
// behind a shared prefix (qlin_prefix.cu) have in common.
#pragma once
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qlin_ptx.cuh"

namespace qlin {

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

constexpr int kRows = 128;              // rows of a tile of queries
constexpr int kKeys = 128;              // keys of a tile
constexpr int kChunkBytes = 128 * 128;  // 128 rows of 64 elements, 128-byte swizzle
// The reference may lie this far (in powers of two) below the maximum.  Weights up to 2^8 are as exact in 16 bits as those up to 1;
// fp16 ones carry a factor of 2^6 on top, so that they stay below 2^14 and lose bits only under 2^-20 of the largest.
constexpr float kSlack = 8.0f;

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

// Weights 2^arg(x) of the pairs of columns FIRST to LAST.  The exponentials keep their unit (8 cycles a warp's instruction)
// busy only if the work around them is done between them, so the multiplications run two pairs ahead of them, the sums and the
// roundings two pairs behind; `beside(i)` is more work to be done in between, `done(k, words)` takes 16 words of two weights each.
template <typename T, int FIRST, int LAST, typename Arg, typename Beside, typename Done>
__device__ __forceinline__ void weigh(const uint32_t (&x)[4][32], Arg arg, uint64_t (&sum)[2], Beside beside, Done done) {
  uint64_t y[LAST - FIRST];
  float a[LAST - FIRST], b[LAST - FIRST];
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < LAST - FIRST + 4; ++i) {
    if (i < LAST - FIRST) {
      const int c = (FIRST + i) / 16, j = 2 * (FIRST + i) % 32;
      y[i] = arg(pair64(__uint_as_float(x[c][j]), __uint_as_float(x[c][j + 1])));
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

}  // namespace qlin
