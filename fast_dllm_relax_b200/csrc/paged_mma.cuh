// What the items of paged attention on the 5th-generation tensor cores share: the CTA's shape and its registers,
// the 8-bit MMA, small conversions.
#pragma once

#include "paged.h"

namespace fdllm {

constexpr int kThreads = 384;
constexpr int kRegsLaunch = 80;  // two CTAs of 384 threads on an SM; setmaxnreg moves them between the roles

// D[tmem] (+)= A[smem] * B[smem]^T, e4m3 operands, fp32 accumulate, one CTA.
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int kRegs, bool kGrow>
__device__ __forceinline__ void set_registers() {
  if constexpr (kGrow) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

}  // namespace fdllm
