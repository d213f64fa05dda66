// Arguments of the attention's backward pass, shared by its two forms.
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

// the tcgen05 form (hoa_attn_bwd_tc.cu): bf16, d % 8 == 0, every tensor from a 16-byte boundary; delta is there
int attn_bwd_tc(const AttnBwdArgs& a, int BH, cudaStream_t s);

}  // namespace hoa
