// fp32-accurate products of the f16 tensor cores: factors split into two f16 parts, and the skew
// matrix of a row of generators as such a factor.
#pragma once

#include <cuda_fp16.h>

#include "hoa_f32x2.cuh"
#include "hoa_sm100.cuh"

namespace hoa {

// x = hi + lo to 2^-22, two f16 each
HOA_DEVICE void st_split2(F2 x, uint32_t& hi, uint32_t& lo) {
  const float2 v = f2_get(x);
  const __half2 h = __floats2half2_rn(v.x, v.y);
  const float2 f = __half22float2(h);
  const float2 r = f2_get(f2_fma(f2(f.x, f.y), f2(-1.f), x));
  const __half2 l = __floats2half2_rn(r.x, r.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

HOA_DEVICE F2 st_join2(uint32_t hi, uint32_t lo) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  return f2_add(f2(h.x, h.y), f2(l.x, l.y));
}

// Row `row` of the skew matrix of a head's generators (in shared memory), times sr, 16 columns from
// c0 on: entry (r, c) is +gen{r, c} right of the diagonal, -gen{c, r} left of it, 0 past column d and
// in rows past the last one.  The warp's 32 rows are consecutive from a multiple of 32, lane lid has
// row `row`; a chunk that the diagonal misses in all of them has one rule for the whole warp.
HOA_DEVICE void gen_row16(const float* gen, bool banked, int stride, int d, int row, int lid, int c0, float sr_in, F2 (&y)[8]) {
  const int w0 = row & ~31, rr = min(row, d - 1);        // (rows past the matrix read its last row and get 0)
  const float sr = row < d ? sr_in : 0.f;
  const int base_r = rr * (2 * d - rr - 1) / 2 - rr - 1; // packed: {r, c}, r < c, lies at base_r + c
  float v[16];
  float sg = sr;
  if (banked) {                                          // gen_banked_slot, 32 x 32 block by block
    const int nb = d >> 5, ba = w0 >> 5, bb = c0 >> 5, v0 = c0 & 31, lo = min(ba, bb), hi = max(ba, bb);
    const float* blk = gen + (lo * nb - lo * (lo + 1) / 2 + hi - lo - 1) * 1024;
    if (ba < bb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = blk[lid * 32 + ((v0 + e) ^ (4 * (lid & 7)))];
    } else if (ba > bb) {
      sg = -sr;
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = blk[(v0 + e) * 32 + (lid ^ (4 * ((v0 + e) & 7)))];
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int cc = c0 + e;
        const float g = gen[cc != rr ? gen_banked_slot(rr, cc, d) : 0];
        v[e] = cc > rr ? g : (cc < rr ? -g : 0.f);
      }
    }
  } else if (c0 > w0 + 31) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = gen[base_r + c0 + e];
  } else {
    int base_c = c0 * (2 * d - c0 - 1) / 2 - c0 - 1;
    if (c0 + 15 < w0) {
      sg = -sr;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        v[e] = gen[base_c + rr];
        base_c += d - c0 - e - 2;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int cc = c0 + e;
        const float g = gen[max(0, min(cc > rr ? base_r + cc : base_c + rr, stride - 1))];
        v[e] = cc > rr ? g : (cc < rr ? -g : 0.f);
        base_c += d - cc - 2;
      }
    }
  }
  if (c0 + 16 > d)                                       // pad columns
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = c0 + e < d ? v[e] : 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = f2_mul(f2(v[2 * e], v[2 * e + 1]), f2(sg));
}

}  // namespace hoa
