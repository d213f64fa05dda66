// Pairs of fp32 values in one 64-bit register: the packed arithmetic of sm_100 (fma.rn.f32x2 and
// its kin), two results an instruction, each rounded as the scalar form rounds it.
#pragma once

#include "hoa_common.cuh"

namespace hoa {

using F2 = unsigned long long;
HOA_DEVICE F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
HOA_DEVICE F2 f2(float x) { return f2(x, x); }
HOA_DEVICE float2 f2_get(F2 x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
HOA_DEVICE F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
HOA_DEVICE F2 f2_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
HOA_DEVICE F2 f2_add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

}  // namespace hoa
