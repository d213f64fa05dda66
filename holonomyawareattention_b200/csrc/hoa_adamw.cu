// One AdamW step over many tensors (a module's parameters) in one launch.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  r = sqrt(v)
//   x = x (1 - lr wd) - lr / (1 - b1^t)  m / (r / sqrt(1 - b2^t) + eps)
//
// x is the parameter, or its fp32 master copy (then the parameter is x, rounded).  The
// moments are fp32 (m and v), or 8 bits: blocks of 256 elements, each with a scale that
// puts its largest magnitude at 448, the largest e4m3 value; m and the root r are held as
// e4m3 (r, not v: its range in a block is the square root of v's, and e4m3 has 2^17.8 of
// it).  A root that is not zero is held as at least e4m3's smallest value, so that an
// element with a small gradient is never divided by eps alone.  A moment that is not finite is
// held as e4m3's NaN and takes no part in its block's scale: as in fp32 it loses its own element
// and no other.  The step itself uses the new moments before they are rounded to 8 bits.
//
// Rounding.  To the nearest, but for m below 2^-5, where all steps are the smallest one (2^-9), if the
// gradient adds less than half of it (of the scale before): towards 0.  To the nearest, 4 of these steps
// times 0.9 are 4 again, so a weight whose gradient has ended would be moved for good (by 0.13 lr a
// step, betas 0.9 and 0.95: its root stays too, at 20 steps).
//
// With beta1 above 15/16 or beta2 above 0.95, up or down by chance, so that the mean is exact.  To the nearest, a moment
// that a step changes by less than half of its last place (3 to 6% of it) stays where it is: m falls by 1 - beta1 of itself at
// most, a root by (1 - beta2) / 2.  Held over true roots (their median) 60, 100 and 200 steps after gradients have fallen
// tenfold: beta2 0.95 to the nearest 1.6, 1.7 and 1.1, 0.97 to the nearest 2.4, 3.9 and 5.7, 0.999 to the nearest for good 6;
// by chance all 0.95 to 1.03, 1% to 99% of them within a factor of 1.4 at 0.97 and 2 at 0.999.  The chance is a hash of the
// element's number and the step's: the same state and gradients give the same bits.
//
// HBM bounds it: every byte is read and written once, a thread's loads come before all else.  Measured: 477 M elements,
// bf16 with masters and 8-bit moments (16 bytes an element), to the nearest 1.60 to 1.68 ms, 4.5 to 4.8 TB/s (conversions,
// roots and the block's maxima beside the loads), by chance 2.0 ms (the hash and the second rounding: 30 operations an
// element), with half of the gradients ended 1.96; 3.9 M fp32 in six tensors (28 bytes an element) 20 to 23 us, 4.8 to 5.4 TB/s.
#include <cuda_fp8.h>

#include <cmath>

#include "hoa_common.cuh"

namespace hoa {

constexpr int kAwThreads = 256, kAwBlock = 256, kAwPer = 8;       // a CTA: 8 elements a thread
constexpr int kAwSpan = kAwThreads * kAwPer;                      // elements of a CTA, a multiple of kAwBlock
constexpr int kAwCtas = 4;                                        // CTAs of an SM: 3 leave loads too little room, 5 and 6 spill
constexpr int kAwMost = 256;                                      // tensors of one launch
constexpr float kAwLeast = 0.001953125f;                          // 2^-9, the smallest e4m3 value: the least a root is held as
constexpr float kAwHalf = 0.5f * kAwLeast;

struct AwTensor {
  void* p; float* master; const void* g; void* m; void* v; float* scales;
  long long n;
  int vec;                        // every pointer is a multiple of 16 bytes (8 of the 8-bit moments)
};
struct AwArgs {
  AwTensor t[kAwMost];
  unsigned first[kAwMost];        // the first CTA of each tensor
  unsigned ctas;                  // parts of kAwSpan elements, all tensors together
  int count, p_dtype, g_dtype;
  const int* step;
  float b1, nb1, b2, nb2, eps, keep;
  float lr;
  double ln1, ln2;                // of the betas
};
static_assert(sizeof(AwArgs) <= 32000, "kernel parameters");

// two e4m3 bytes <-> values
HOA_DEVICE float2 aw_values(unsigned pair) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3);
  return __half22float2(__half2(h));
}
HOA_DEVICE unsigned aw_e4m3(float x, float y) { return __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3); }

// a / b rounded to nearest, b the same for many a: with y = 1 / b rounded to nearest and q = a y, q + (a - q b) y is the
// correctly rounded quotient (Markstein, IBM J. Res. Dev. 34, 1990, theorem 8), as long as nothing leaves the normal range.
// (Here |a| <= 448 b and 1e-12 < b < 1e12; what underflows is far below half the smallest e4m3 value and rounds to 0 anyway.)
HOA_DEVICE float aw_div(float a, float b, float y) {
  const float q = __fmul_rn(a, y);
  return fmaf(fmaf(-q, b, a), y, q);
}
HOA_DEVICE bool aw_div_by(float b) { return b > 1e-12f && b < 1e12f; }

// the largest of a warp's values, none below 0
HOA_DEVICE float aw_warp_max(float x) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x))); }
// a block's scale, of its finite values alone
HOA_DEVICE float aw_scale(const float (&x)[8], float scale) {
  if (scale < INFINITY) return scale;
  float t = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) t = fabsf(x[e]) < INFINITY ? fmaxf(t, fabsf(x[e])) : t;
  return __fmul_rn(aw_warp_max(t), 1.f / 448.f);
}
// x in units of a scale of any size (0 where that is 0; infinity and NaN: NaN)
HOA_DEVICE float aw_quotient(float x, float scale) {
  return !(fabsf(x) < INFINITY) ? __uint_as_float(0x7fffffffu) : scale > 0.f ? __fdiv_rn(x, scale) : 0.f;
}

HOA_DEVICE float aw_sqrt(float x) {                     // to an ulp or two: for the update, not for what is kept
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// N consecutive elements from i on, in 16-byte pieces (kVec: the address is a multiple of what a piece takes), those past
// n as 0
template <bool kVec, int N>
HOA_DEVICE void aw_load(const void* x, int dtype, long long i, long long n, float (&v)[N]) {
  if (kVec && i + N <= n) {
    if (dtype == HOA_F32) {
#pragma unroll
      for (int q = 0; q < N / 4; ++q) {
        const float4 t = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + i)[q];
        v[4 * q] = t.x; v[4 * q + 1] = t.y; v[4 * q + 2] = t.z; v[4 * q + 3] = t.w;
      }
    } else {
#pragma unroll
      for (int q = 0; q < N / 8; ++q) {
        const uint4 t = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(x) + i)[q];
        const uint32_t u[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[8 * q + 2 * e] = __uint_as_float(u[e] << 16);
          v[8 * q + 2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = i + e < n ? load_elem(x, i + e, dtype) : 0.f;
  }
}

template <bool kVec, int N>
HOA_DEVICE void aw_store(void* x, int dtype, long long i, long long n, const float (&v)[N]) {
  if (kVec && i + N <= n) {
    if (dtype == HOA_F32) {
#pragma unroll
      for (int q = 0; q < N / 4; ++q)
        reinterpret_cast<float4*>(reinterpret_cast<float*>(x) + i)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    } else {
#pragma unroll
      for (int q = 0; q < N / 8; ++q) {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
          u[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(x) + i)[q] = make_uint4(u[0], u[1], u[2], u[3]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (i + e < n) store_elem(x, i + e, dtype, v[e]);
  }
}

// 8 bytes from i on, as words
template <bool kVec>
HOA_DEVICE uint2 aw_load8(const void* x, long long i, long long n) {
  const unsigned char* b = reinterpret_cast<const unsigned char*>(x) + i;
  if (kVec && i + 8 <= n) return *reinterpret_cast<const uint2*>(b);
  unsigned u[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (i + e < n) u[e / 4] |= (unsigned)b[e] << (8 * (e & 3));
  return make_uint2(u[0], u[1]);
}
template <bool kVec>
HOA_DEVICE void aw_store8(void* x, long long i, long long n, uint2 v) {
  unsigned char* b = reinterpret_cast<unsigned char*>(x) + i;
  if (kVec && i + 8 <= n) {
    *reinterpret_cast<uint2*>(b) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (i + e < n) b[e] = (unsigned char)((e < 4 ? v.x : v.y) >> (8 * (e & 3)));
}
// e4m3 bytes of x[0..8), each times what f says
template <class Fn>
HOA_DEVICE uint2 aw_pack8(const float (&x)[8], Fn f) {
  unsigned u[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    u[h] = aw_e4m3(f(x[4 * h]), f(x[4 * h + 1])) | aw_e4m3(f(x[4 * h + 2]), f(x[4 * h + 3])) << 16;
  return make_uint2(u[0], u[1]);
}

// 32 bits that are as good as random, of an element's number and a step's (multiplications by odd numbers and shifts; any
// would do that spread one bit's change over all)
HOA_DEVICE uint32_t aw_noise(long long i, uint32_t step) {
  uint32_t x = (uint32_t)i * 0x9e3779b1u ^ (uint32_t)((unsigned long long)i >> 32) * 0xb5297a4du;
  x += step * 0x68e31da5u;
  x = (x ^ (x >> 16)) * 0x7a3f5c2bu;
  x = (x ^ (x >> 15)) * 0xc4d1e6b7u;
  return x ^ (x >> 16);
}
// q -> one of the two e4m3 values around it, by 16 random bits: those added below the last place (2^-9 up to 2^-6), the rest
// cut off.  (The half behind them keeps a value of e4m3 that is a few ulps off where it is.)
HOA_DEVICE float aw_chance(float q, uint32_t u) {
  const float a = fabsf(q);
  const float big = __uint_as_float((__float_as_uint(a) + (u << 4 | 8u)) & 0xfff00000u);
  const float small = floorf(fmaf(a, 512.f, fmaf((float)u, 1.f / 65536.f, 0.5f / 65536.f))) * (1.f / 512.f);
  return copysignf(a >= 0.015625f ? big : small, q);
}

// The moments of a block that is not as most are, from shared memory (m, then r, kAwThreads apart), out of line and at the
// block's end: its registers are not the others'.  old: m's scale before.
template <bool kVec, bool kChance>
__device__ __noinline__ void aw_rare(const AwTensor& t, long long blk, int g_dtype, float nb1, float old, float ms, float vs, uint32_t step,
                                     const float* at) {
  const int lid = threadIdx.x & 31;
  const long long i = blk * kAwBlock + 8 * lid, blocks = (t.n + kAwBlock - 1) / kAwBlock;
  float x[8], g[8];
  auto load = [&](int from) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = at[(from + e) * kAwThreads];
  };
  load(0);
  ms = aw_scale(x, ms);
  if (!kChance) aw_load<kVec>(t.g, g_dtype, i, t.n, g);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = aw_quotient(x[e], ms);
    if (kChance) x[e] = aw_chance(x[e], aw_noise(i + e, step) >> 16);
    else if (__fmul_rn(fabsf(g[e]), nb1) < kAwHalf * old && fabsf(x[e]) < 0.03125f) x[e] = truncf(x[e] * 512.f) * (1.f / 512.f);
  }
  aw_store8<kVec>(t.m, i, t.n, aw_pack8(x, [](float q) { return q; }));
  load(8);
  vs = aw_scale(x, vs);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float q = aw_quotient(x[e], vs);
    if (kChance) q = aw_chance(q, aw_noise(i + e, step) & 0xffffu);
    x[e] = x[e] > 0.f && q < kAwLeast ? kAwLeast : q;
  }
  aw_store8<kVec>(t.v, i, t.n, aw_pack8(x, [](float q) { return q; }));
  if (lid == 0) {
    t.scales[blk] = ms;
    t.scales[blocks + blk] = vs;
  }
}

// A warp has one block of 256 elements, a lane 8 consecutive ones of it.
template <int kBits, bool kVec, bool kChance>
HOA_DEVICE void aw_block(const AwArgs& a, const AwTensor& t, long long blk, float lr, float y2, uint32_t step, float* rare) {
  const int lid = threadIdx.x & 31;
  const long long i = blk * kAwBlock + 8 * lid, n = t.n;
  const long long blocks = (n + kAwBlock - 1) / kAwBlock;
  float g[8], x[8], m[8], v[8];
  uint2 mb = make_uint2(0, 0), vb = mb;
  float ms = 0.f, vs = 0.f;
  bool ended = false;
  // all loads first
  aw_load<kVec>(t.g, a.g_dtype, i, n, g);
  if (t.master) aw_load<kVec>(t.master, HOA_F32, i, n, x);
  else aw_load<kVec>(t.p, a.p_dtype, i, n, x);
  if (kBits == 8) {
    mb = aw_load8<kVec>(t.m, i, n);
    vb = aw_load8<kVec>(t.v, i, n);
    ms = t.scales[blk];
    vs = t.scales[blocks + blk];
    float least = INFINITY;
#pragma unroll
    for (int e = 0; e < 8 && !kChance; e += 2) least = fminf(least, fminf(fabsf(g[e]), fabsf(g[e + 1])));
    ended = __fmul_rn(least, a.nb1) < kAwHalf * ms;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 mv = aw_values((e < 4 ? mb.x : mb.y) >> (8 * (e & 3)) & 0xffffu);
      const float2 rv = aw_values((e < 4 ? vb.x : vb.y) >> (8 * (e & 3)) & 0xffffu);
      m[e] = __fmul_rn(mv.x, ms);
      m[e + 1] = __fmul_rn(mv.y, ms);
      const float r0 = __fmul_rn(rv.x, vs), r1 = __fmul_rn(rv.y, vs);
      v[e] = __fmul_rn(r0, r0);
      v[e + 1] = __fmul_rn(r1, r1);
    }
  } else {
    aw_load<kVec>(t.m, HOA_F32, i, n, m);
    aw_load<kVec>(t.v, HOA_F32, i, n, v);
  }
  float r[8];
  const bool tail = kBits == 8 && i + 8 > n;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    m[e] = __fadd_rn(__fmul_rn(m[e], a.b1), __fmul_rn(g[e], a.nb1));
    v[e] = __fadd_rn(__fmul_rn(v[e], a.b2), __fmul_rn(__fmul_rn(g[e], g[e]), a.nb2));
    if (tail && i + e >= n) m[e] = v[e] = 0.f;                    // (a scale of NaN reaches the elements past the end too)
    r[e] = kBits == 8 ? __fsqrt_rn(v[e]) : aw_sqrt(v[e]);
    const float den = fmaf(r[e], y2, a.eps);
    x[e] = fmaf(x[e], a.keep, -lr * __fdividef(m[e], den));
  }
  if (t.master) aw_store<kVec>(t.master, HOA_F32, i, n, x);
  aw_store<kVec>(t.p, a.p_dtype, i, n, x);
  if (kBits != 8) {
    aw_store<kVec>(t.m, HOA_F32, i, n, m);
    aw_store<kVec>(t.v, HOA_F32, i, n, v);
    return;
  }
  // the largest of the block (a NaN is passed over)
  float mt = 0.f, rt = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    mt = fmaxf(mt, fmaxf(fabsf(m[e]), fabsf(m[e + 1])));
    rt = fmaxf(rt, fmaxf(r[e], r[e + 1]));
  }
  const float old = ms;
  ms = __fmul_rn(aw_warp_max(mt), 1.f / 448.f);
  vs = __fmul_rn(aw_warp_max(rt), 1.f / 448.f);
  if (__any_sync(0xffffffffu, ended) || !aw_div_by(ms) || !aw_div_by(vs)) {                // (uniform in the warp)
    float* at = rare + threadIdx.x;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      at[e * kAwThreads] = m[e];
      at[(8 + e) * kAwThreads] = r[e];
    }
    aw_rare<kVec, kChance>(t, blk, a.g_dtype, a.nb1, old, ms, vs, step, at);
    return;
  }
  const float ym = __frcp_rn(ms), yr = __frcp_rn(vs);
  if (kChance) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t u = aw_noise(i + e, step);
      m[e] = aw_chance(aw_div(m[e], ms, ym), u >> 16);
      r[e] = r[e] > 0.f ? fmaxf(aw_chance(aw_div(r[e], vs, yr), u & 0xffffu), kAwLeast) : r[e];
    }
    mb = aw_pack8(m, [](float q) { return q; });
    vb = aw_pack8(r, [](float q) { return q; });
  } else {
    mb = aw_pack8(m, [&](float q) { return aw_div(q, ms, ym); });
    vb = aw_pack8(r, [&](float q) { return q > 0.f ? fmaxf(aw_div(q, vs, yr), kAwLeast) : q; });
  }
  aw_store8<kVec>(t.m, i, n, mb);
  aw_store8<kVec>(t.v, i, n, vb);
  if (lid == 0) {
    t.scales[blk] = ms;
    t.scales[blocks + blk] = vs;
  }
}

template <int kBits, bool kChance>
__global__ void __launch_bounds__(kAwThreads, kAwCtas) adamw_kernel(const __grid_constant__ AwArgs a) {
  __shared__ float rare[kBits == 8 ? 16 * kAwThreads : 1];
  // 1 - b^t = -(e^{t ln b} - 1)
  const int step = *a.step;
  const double t = (double)step;
  const float lr = a.lr / -expm1f((float)(t * a.ln1)), y2 = rsqrtf(-expm1f((float)(t * a.ln2)));
  int lo = 0;
  for (unsigned c = blockIdx.x; c < a.ctas; c += gridDim.x) {
    int hi = a.count - 1;                              // the tensor of this part: the last one that starts at or before it
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (a.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    const AwTensor& x = a.t[lo];
    const long long blk = (long long)(c - a.first[lo]) * (kAwSpan / kAwBlock) + (threadIdx.x >> 5);
    if (blk * kAwBlock >= x.n) continue;
    if (x.vec) aw_block<kBits, true, kChance>(a, x, blk, lr, y2, (uint32_t)step, rare);
    else aw_block<kBits, false, kChance>(a, x, blk, lr, y2, (uint32_t)step, rare);
  }
}

}  // namespace hoa

using namespace hoa;

extern "C" int hoa_adamw_step(void* const* params, int p_dtype, float* const* masters, const void* const* grads, int g_dtype,
                              void* const* m, void* const* v, float* const* scales, int state_bits, const long long* sizes, int count,
                              const int* step, double lr, double beta1, double beta2, double eps, double weight_decay, void* stream) {
  if (!params || !grads || !m || !v || !sizes || !step || count < 0) return HOA_ERR_INVALID_ARG;
  if ((p_dtype != HOA_F32 && p_dtype != HOA_BF16) || (g_dtype != HOA_F32 && g_dtype != HOA_BF16) ||
      (state_bits != 32 && state_bits != 8))
    return HOA_ERR_UNSUPPORTED;
  if (state_bits == 8 && !scales) return HOA_ERR_INVALID_ARG;
  for (int i = 0; i < count; ++i) {
    if (sizes[i] < 0) return HOA_ERR_INVALID_ARG;
    if (sizes[i] == 0) continue;
    if (!params[i] || !grads[i] || !m[i] || !v[i] || (state_bits == 8 && !scales[i])) return HOA_ERR_INVALID_ARG;
    if (sizes[i] > (long long)kAwSpan * 0x3fffffff) return HOA_ERR_UNSUPPORTED;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  static const unsigned most = []() {                      // CTAs that run at once; of the device that calls first: every GPU here is the same
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      n = 148;
    return (unsigned)n * kAwCtas;
  }();
  for (int i = 0; i < count;) {
    AwArgs a{};
    unsigned ctas = 0;
    for (; i < count && a.count < kAwMost; ++i) {
      const long long n = (sizes[i] + kAwSpan - 1) / kAwSpan;
      if (n == 0) continue;
      if (ctas + n > 0x7fffffffll) break;
      uintptr_t at = reinterpret_cast<uintptr_t>(params[i]) | reinterpret_cast<uintptr_t>(grads[i]) |
                     reinterpret_cast<uintptr_t>(masters ? masters[i] : nullptr);
      const uintptr_t mv = reinterpret_cast<uintptr_t>(m[i]) | reinterpret_cast<uintptr_t>(v[i]);
      at |= state_bits == 8 ? (mv & 7) : mv;
      a.t[a.count] = AwTensor{params[i], masters ? masters[i] : nullptr, grads[i], m[i], v[i], scales ? scales[i] : nullptr, sizes[i],
                              (at & 15) == 0};
      a.first[a.count++] = ctas;
      ctas += (unsigned)n;
    }
    if (a.count == 0) break;
    a.p_dtype = p_dtype;
    a.g_dtype = g_dtype;
    a.ctas = ctas;
    a.step = step;
    a.b1 = (float)beta1; a.nb1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2; a.nb2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.keep = (float)(1.0 - lr * weight_decay);
    a.lr = (float)lr;
    a.ln1 = log(beta1); a.ln2 = log(beta2);
    const unsigned grid = ctas < most ? ctas : most;
    if (state_bits == 32) adamw_kernel<32, false><<<grid, kAwThreads, 0, s>>>(a);
    else if (beta1 > 0.9375 || beta2 > 0.95) adamw_kernel<8, true><<<grid, kAwThreads, 0, s>>>(a);
    else adamw_kernel<8, false><<<grid, kAwThreads, 0, s>>>(a);
    if (int st = launch_status()) return st;
  }
  return HOA_OK;
}
