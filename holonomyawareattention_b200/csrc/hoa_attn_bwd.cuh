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

}  // namespace hoa
