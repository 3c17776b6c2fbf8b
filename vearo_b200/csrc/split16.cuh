// f32 matrices as pairs of half-precision planes for the tensor cores, and the tcgen05.mma kind::f16 pieces that read them.
//
// A value x of a 128 x 128 block is held as (hi + lo) * 2^-e with hi = half(x 2^e), lo = half(x 2^e - hi) and one exponent e per
// block, chosen so that the block's largest finite magnitude lies in [2^14, 2^15).  hi + lo carries 22 significant bits for
// magnitudes down to 2^-17 of the block's largest and an absolute error of 2^-40 of that largest below (where lo, then hi, is
// subnormal).  A product of two such matrices is hi hi' + hi lo' + lo hi'; the dropped lo lo' is at most 2^-24 of |x x'|.  The
// half-precision instruction does 16 steps of k where TF32 does 8 for the same 22 bits, which is why these kernels do
// not use the TF32 split of gemm_tc.cu.
//
// The tensor core adds to its f32 accumulator by truncation (measured: a relative bias of -1e-7 for every 1.2 instructions of equal
// sign, -4e-6 after 48), so no accumulator is fed for long: the kernels add it to registers, rounding to nearest, after at
// most 128 steps of k, and within such a run the small cross products go first where all of them are at hand.
#pragma once
#include <cuda_fp16.h>
#include "common.h"
#include "gemm16.h"
#include "tc_util.cuh"

namespace vb {

// scale 2^e of a block with largest finite magnitude amax (0: an empty block), and its inverse.  e stays within +-100 so that both are
// normal numbers; blocks below 2^-86 keep fewer bits.
__device__ __forceinline__ float block_scale(float amax, float* inverse) {
  int e = 0;
  if (amax > 0.0f) {
    e = 14 - (((int)(__float_as_uint(amax) >> 23) & 255) - 127);
    e = e > 100 ? 100 : e;
  }
  *inverse = __uint_as_float((uint32_t)(127 - e) << 23);
  return __uint_as_float((uint32_t)(127 + e) << 23);
}
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e38f; }
__device__ __forceinline__ float finite_abs(float x) { const float a = fabsf(x); return a <= 3.402823466e38f ? a : 0.0f; }

// hi and lo of a scaled pair, packed (a value that is not finite has lo = 0, so that hi alone carries it)
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  float la = a - f.x, lb = b - f.y;
  if (!(fabsf(la) <= 65504.0f)) la = 0.0f;
  if (!(fabsf(lb) <= 65504.0f)) lb = 0.0f;
  const __half2 l = __floats2half2_rn(la, lb);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  *lo = *reinterpret_cast<const uint32_t*>(&l);
}
// the same for values known to be finite and below 2^15
__device__ __forceinline__ void split2_finite(float a, float b, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 d = fma2(__half22float2(h), make_float2(-1.0f, -1.0f), make_float2(a, b));
  const __half2 l = __floats2half2_rn(d.x, d.y);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  *lo = *reinterpret_cast<const uint32_t*>(&l);
}

namespace tc {

// Shared-memory descriptors of half-precision tiles in the 128-byte swizzle.  K-major: rows of 64 k values (128 bytes), groups of 8
// rows 1024 bytes apart; 16 k values further are 32 bytes further.  MN-major: blocks of 64 mn values (128 bytes), one 128-byte row per
// k; groups of 8 k rows are 1024 bytes apart, blocks `block_bytes`; 16 k values further are 2048 bytes further.
__device__ __forceinline__ uint64_t desc16(uint32_t smem_addr, uint32_t block_bytes) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFF) | (uint64_t)((block_bytes >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// D = f32, A = B = f16
__device__ __forceinline__ uint32_t idesc16(int m, int n, int a_mn, int b_mn) {
  return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// The issuing warp runs converged and one lane of it, the leader, executes the instruction.  (Issued by one lane of a diverged warp, MMAs came 65-75
// cycles apart by the clock, more than a 128 x 128 x 16 product takes: attention of 16384 tokens, 8 + 2 heads of 128, 1359 us instead of 1063.)
__device__ __forceinline__ uint32_t elect_leader() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
__device__ __forceinline__ void mma_f16(uint32_t leader, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %9, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(leader) : "memory");
}
// A read from tensor memory: row i of A on lane i, 16 k values in 8 consecutive columns
__device__ __forceinline__ void mma_f16_ta(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %9, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u), "r"(0u), "r"(0u), "r"(0u), "r"(leader) : "memory");
}
__device__ __forceinline__ void commit_by(uint32_t leader, uint64_t* bar) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
               ::"r"(smem_u32(bar)), "r"(leader) : "memory");
}
// The wait for a load from tensor memory, with the registers that it fills: they may not be used before it, and without the dependence the
// compiler is free to move arithmetic on them ahead of it.
template <int W>
__device__ __forceinline__ void wait_for_cols(uint32_t* r) {
  if constexpr (W == 32)
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 ::"memory");
  else
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 ::"memory");
}
// a wait of the whole warp, the same answer for all of it
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

}  // namespace tc

// A target column as an integer.  A row whose target is `ignore` is left out (kNoTarget); a negative or too large one is reported and left out.
__device__ __forceinline__ int read_target(float v, i64 ignore, i64 vocab, int* err) {
  if (v == (float)ignore || (fabsf(v) < 1e9f && (i64)roundf(v) == ignore)) return kNoTarget;
  if (!(v > -0.5f)) { atomicOr(err, ERRBIT_NEG_ID); return kNoTarget; }
  if (!(roundf(v) < (float)vocab)) { atomicOr(err, ERRBIT_OOB_ID); return kNoTarget; }
  return (int)roundf(v);
}
// of a kernel launched by launch_early: nothing that the kernel ahead of it in the stream writes is touched before this
__device__ __forceinline__ void wait_for_last_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// A launch that is made ready while the kernel ahead of it in the stream still runs.  No kernel here lets its successor go before its own end, so what is
// saved is the launch's latency, not time of the kernel ahead.
template <class... P, class... A>
int launch_early(void (*kernel)(P...), dim3 ctas, dim3 threads, int smem, A... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = ctas; c.blockDim = threads; c.dynamicSmemBytes = (size_t)smem; c.stream = ctx().stream; c.attrs = &at; c.numAttrs = 1;
  VB_CUDA(cudaLaunchKernelEx(&c, kernel, args...));
  VB_LAUNCH_CHECK();
  return VB_OK;
}
}  // namespace vb
