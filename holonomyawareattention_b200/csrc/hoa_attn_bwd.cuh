// Arguments of the attention's backward pass, shared by its two forms (bf16, fp32).
#pragma once

#include "hoa_common.cuh"

namespace hoa {

struct AttnBwdArgs {
  const void* q; const void* k; const void* v;      // (BH, Tq, d), (BH, Tk, d) in dtype
  const float* o; const float* lse;                 // (BH, Tq, d), (BH, Tq): what the forward left
  const void* dout;                                 // (BH, Tq, d) in dtype
  float* delta;                                     // (BH, Tq): D, scratch
  void* dq; void* dk; void* dv; int dtype;
  float scale;
  int Tq, Tk, q_offset, d;
  int* status;
  long long max_wait;                               // bound of a wait, SM cycles (wait_bound_cycles())
};

// The tcgen05 form (hoa_attn_bwd_tc.cu) for bf16; delta is there.  copies: attn_bwd_tc_bytes of scratch where d % 8 != 0
// or a tensor does not start at a 16-byte boundary, else null.
size_t attn_bwd_tc_bytes(int BH, int Tq, int Tk, int d);
int attn_bwd_tc(const AttnBwdArgs& a, int BH, void* copies, cudaStream_t s);

}  // namespace hoa
