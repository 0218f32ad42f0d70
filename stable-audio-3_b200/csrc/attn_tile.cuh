// Pieces shared by the attention kernels on tcgen05: packed fp32 pairs, the exponentials of a chunk of scores and
// the MMA / commit issue of a converged warp.
#pragma once
#include "common.cuh"

namespace sa3 {

__device__ __forceinline__ uint32_t pack_2(float lo, float hi, bool f16) {
  if (f16) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  return pack_bf16x2(lo, hi);
}

// Packed pairs of fp32 (sm_100 f32x2 arithmetic: one instruction per two lanes of data).
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 f2_split(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t ffma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t fmul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fadd2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

constexpr uint32_t NEG_INF_BITS = 0xff800000u;

// Edge tile: scores of columns outside [lo, hi) (chunk-relative) become -inf.
__device__ __forceinline__ void mask_chunk(uint32_t (&s)[32], int lo, int hi) {
  const int a = min(max(lo, 0), 32), b = min(max(hi, 0), 32);
  const uint32_t below_b = b >= 32 ? 0xffffffffu : ((1u << b) - 1u);
  const uint32_t below_a = a >= 32 ? 0xffffffffu : ((1u << a) - 1u);
  const uint32_t m = below_b & ~below_a;
#pragma unroll
  for (int e = 0; e < 32; ++e) s[e] = (m >> e) & 1u ? s[e] : NEG_INF_BITS;
}

// Running maxima over one chunk, eight independent chains.
__device__ __forceinline__ void max_chunk(const uint32_t (&s)[32], float (&m)[8]) {
#pragma unroll
  for (int t = 0; t < 8; ++t)
    m[t] = fmax3(fmax3(m[t], __uint_as_float(s[4 * t]), __uint_as_float(s[4 * t + 1])),
                 __uint_as_float(s[4 * t + 2]), __uint_as_float(s[4 * t + 3]));
}

// P = exp2(s * scale - m) for one chunk as packed 16-bit pairs, row sums into four f32x2 chains.
__device__ __forceinline__ void exp_chunk(const uint32_t (&s)[32], uint64_t scale2, uint64_t negm2,
                                          uint64_t (&acc)[4], uint32_t (&w)[16], bool f16) {
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const float2 x = f2_split(ffma2(f2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale2, negm2));
    const float p0 = fast_exp2(x.x), p1 = fast_exp2(x.y);
    acc[(e >> 1) & 3] = fadd2(acc[(e >> 1) & 3], f2(p0, p1));
    w[e >> 1] = pack_2(p0, p1, f16);
  }
}

// tcgen05.mma / commit issued by one elected lane of a converged warp, descriptors given as (low
// word, shared high word): the issue loop only adds constants to the low word (the start-address
// field). Running the issue loop on the whole warp keeps its operands warp-uniform, which lets the
// MMAs go out back to back (from a single lane in a divergent branch the 64-wide P V steps issue at
// about 60% of the tensor rate).
__device__ __forceinline__ void mma_ss_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts_lo(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 r;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit_elect(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
      : "memory");
}
// mbar_wait whose tries suspend the thread for up to a millisecond each: a waiting warp then leaves the issue slots and
// the shared-memory pipe to the others instead of trying again every few dozen cycles.
__device__ __forceinline__ bool mbar_try_wait_1ms(uint32_t addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(addr), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int site) {
  const uint32_t addr = smem_u32(bar);
  if (mbar_try_wait_1ms(addr, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (mbar_try_wait_1ms(addr, parity)) return true;
    if (*abort) return false;
    if (clock64() - t0 > SA3_WAIT_BUDGET_CYCLES) {
      record_error(SA3_DEVERR_TIMEOUT, site);
      *abort = 1;
      return false;
    }
  }
}
__device__ __forceinline__ bool warp_bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int site) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, abort, site));
}
// Bring one box of a tensor map into L2 (rows and columns outside the tensor are skipped).
__device__ __forceinline__ void tma_prefetch_l2_2d(const CUtensorMap* m, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(m)),
               "r"(x), "r"(y)
               : "memory");
}
// 16 columns of this thread's TMEM lane, complete on return
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  tmem_wait_ld();
}

// Four K = 16 steps under one election: SS operands K-major in 128-byte rows (+32 bytes a step on both sides), TS with
// A in TMEM (+8 columns a step) and an MN-major B (+16 rows of 128 bytes a step).
__device__ __forceinline__ void mma4_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 r, x, y;\n\t.reg .b64 da, db;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t"
      "setp.eq.b32 p, %4, %4;\n\t"
      "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 da, {x, %3};\n\tmov.b64 db, {y, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t"
      "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 da, {x, %3};\n\tmov.b64 db, {y, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t"
      "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 da, {x, %3};\n\tmov.b64 db, {y, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma4_ts(uint32_t d_tmem, uint32_t a0, uint32_t a1, uint32_t b_lo, uint32_t b_hi,
                                        uint32_t idesc, uint32_t accumulate) {
  // a0: columns of steps 0 and 1, a1: of steps 2 and 3
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b32 r, x, y;\n\t.reg .b64 db;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %5, p;\n\t"
      "setp.eq.b32 p, %5, %5;\n\t"
      "add.u32 x, %1, 8;\n\tadd.u32 y, %3, 128;\n\tmov.b64 db, {y, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %5, p;\n\t"
      "add.u32 y, %3, 256;\n\tmov.b64 db, {y, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%2], db, %5, p;\n\t"
      "add.u32 x, %2, 8;\n\tadd.u32 y, %3, 384;\n\tmov.b64 db, {y, %4};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %5, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a0), "r"(a1), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit2_elect(uint64_t* a, uint64_t* b) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t.reg .b32 r;\n\t"
      "elect.sync r|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}\n" ::"r"(smem_u32(a)),
      "r"(smem_u32(b))
      : "memory");
}
// A value that all lanes of a converged warp share, in a uniform register. What an issue loop computes from such values
// stays there; operands of an MMA that the compiler cannot see to be uniform are moved there one by one before each
// instruction, which made an issue loop several times as slow as the products it sent.
__device__ __forceinline__ int uniform_int(int x) { return __reduce_max_sync(0xffffffffu, x); }
// mbar_wait on every lane of a converged warp; the warp agrees on the outcome.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int site) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, site));
}

}  // namespace sa3
