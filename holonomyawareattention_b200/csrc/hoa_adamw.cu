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
// element with a small gradient is never divided by eps alone.  The step itself uses the
// new moments before they are rounded to 8 bits.
//
// Every operation is rounded by itself (no fused multiply-add): the new moments, and so
// the 8-bit values, are those of the same formula written in separate fp32 operations.
#include <cuda_fp8.h>

#include "hoa_common.cuh"

namespace hoa {

constexpr int kAwThreads = 256, kAwBlock = 256, kAwPer = 8;       // a CTA: 8 elements a thread
constexpr int kAwSpan = kAwThreads * kAwPer;                      // elements of a CTA, a multiple of kAwBlock
constexpr int kAwMost = 256;                                      // tensors of one launch

struct AwTensor {
  void* p; float* master; const void* g; void* m; void* v; float* scales;
  long long n;
};
struct AwArgs {
  AwTensor t[kAwMost];
  unsigned first[kAwMost];        // the first CTA of each tensor
  int count, p_dtype, g_dtype, bits;
  const int* step;
  float b1, nb1, b2, nb2, eps, keep;
  double lr, b1d, b2d;
};
static_assert(sizeof(AwArgs) <= 32000, "kernel parameters");

HOA_DEVICE unsigned char aw_e4m3(float x) { return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }
HOA_DEVICE float aw_value(unsigned char c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
  return __half2float(__half(h));
}

__global__ void __launch_bounds__(kAwThreads) adamw_kernel(const __grid_constant__ AwArgs a) {
  __shared__ float s_lr, s_c2;
  if (threadIdx.x == 0) {
    const double t = (double)*a.step;
    s_lr = (float)(a.lr / (1.0 - pow(a.b1d, t)));
    s_c2 = (float)sqrt(1.0 - pow(a.b2d, t));
  }
  int lo = 0, hi = a.count - 1;                      // the tensor of this CTA: the last one that starts at or before it
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const AwTensor& t = a.t[lo];
  __syncthreads();
  const float lr = s_lr, c2 = s_c2;
  const long long base = (long long)(blockIdx.x - a.first[lo]) * kAwSpan;
  const int warp = threadIdx.x >> 5, lid = threadIdx.x & 31;
  // a warp has one block of 256 elements, lane l its elements l, l + 32, ...
  const long long blk = base / kAwBlock + warp;
  const long long b0 = blk * kAwBlock;
  if (b0 >= t.n) return;
  const long long blocks = (t.n + kAwBlock - 1) / kAwBlock;
  float ms = 0.f, vs = 0.f;
  if (a.bits == 8) {
    ms = t.scales[blk];
    vs = t.scales[blocks + blk];
  }
  float m[kAwPer], r[kAwPer], mtop = 0.f, rtop = 0.f;
  bool nan_m = false, nan_r = false;
#pragma unroll
  for (int k = 0; k < kAwPer; ++k) {
    const long long i = b0 + lid + 32 * k;
    m[k] = r[k] = 0.f;
    if (i >= t.n) continue;
    const float g = load_elem(t.g, i, a.g_dtype);
    float mo, vo;
    if (a.bits == 8) {
      mo = __fmul_rn(aw_value(reinterpret_cast<const unsigned char*>(t.m)[i]), ms);
      const float ro = __fmul_rn(aw_value(reinterpret_cast<const unsigned char*>(t.v)[i]), vs);
      vo = __fmul_rn(ro, ro);
    } else {
      mo = reinterpret_cast<const float*>(t.m)[i];
      vo = reinterpret_cast<const float*>(t.v)[i];
    }
    m[k] = __fadd_rn(__fmul_rn(mo, a.b1), __fmul_rn(g, a.nb1));
    const float v = __fadd_rn(__fmul_rn(vo, a.b2), __fmul_rn(__fmul_rn(g, g), a.nb2));
    r[k] = __fsqrt_rn(v);
    const float x = t.master ? t.master[i] : load_elem(t.p, i, a.p_dtype);
    const float den = __fadd_rn(__fdiv_rn(r[k], c2), a.eps);
    const float y = __fsub_rn(__fmul_rn(x, a.keep), __fmul_rn(__fdiv_rn(m[k], den), lr));
    if (t.master) t.master[i] = y;
    store_elem(t.p, i, a.p_dtype, y);
    if (a.bits != 8) {
      reinterpret_cast<float*>(t.m)[i] = m[k];
      reinterpret_cast<float*>(t.v)[i] = v;
    }
    mtop = fmaxf(mtop, fabsf(m[k]));
    rtop = fmaxf(rtop, r[k]);
    nan_m |= m[k] != m[k];
    nan_r |= r[k] != r[k];
  }
  if (a.bits != 8) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mtop = fmaxf(mtop, __shfl_xor_sync(0xffffffffu, mtop, o));
    rtop = fmaxf(rtop, __shfl_xor_sync(0xffffffffu, rtop, o));
  }
  // (a NaN among the moments is the block's scale, as a maximum that propagates it would be)
  const float nan = __int_as_float(0x7fffffff);
  ms = __any_sync(0xffffffffu, nan_m) ? nan : __fmul_rn(mtop, 1.f / 448.f);
  vs = __any_sync(0xffffffffu, nan_r) ? nan : __fmul_rn(rtop, 1.f / 448.f);
#pragma unroll
  for (int k = 0; k < kAwPer; ++k) {
    const long long i = b0 + lid + 32 * k;
    if (i >= t.n) continue;
    const float qm = ms > 0.f ? __fdiv_rn(m[k], ms) : 0.f;
    float qr = vs > 0.f ? __fdiv_rn(r[k], vs) : 0.f;
    if (r[k] > 0.f) qr = fmaxf(qr, 0.001953125f);
    reinterpret_cast<unsigned char*>(t.m)[i] = aw_e4m3(qm);
    reinterpret_cast<unsigned char*>(t.v)[i] = aw_e4m3(qr);
  }
  if (lid == 0) {
    t.scales[blk] = ms;
    t.scales[blocks + blk] = vs;
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
  for (int i = 0; i < count;) {
    AwArgs a{};
    unsigned ctas = 0;
    for (; i < count && a.count < kAwMost; ++i) {
      const long long n = (sizes[i] + kAwSpan - 1) / kAwSpan;
      if (n == 0) continue;
      if (ctas + n > 0x7fffffffll) break;
      a.t[a.count] = AwTensor{params[i], masters ? masters[i] : nullptr, grads[i], m[i], v[i], scales ? scales[i] : nullptr, sizes[i]};
      a.first[a.count++] = ctas;
      ctas += (unsigned)n;
    }
    if (a.count == 0) break;
    a.p_dtype = p_dtype;
    a.g_dtype = g_dtype;
    a.bits = state_bits;
    a.step = step;
    a.b1 = (float)beta1; a.nb1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2; a.nb2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.keep = (float)(1.0 - lr * weight_decay);
    a.lr = lr; a.b1d = beta1; a.b2d = beta2;
    adamw_kernel<<<ctas, kAwThreads, 0, s>>>(a);
    if (int st = launch_status()) return st;
  }
  return HOA_OK;
}
