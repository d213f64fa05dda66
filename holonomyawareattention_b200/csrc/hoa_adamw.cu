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
  int vec;                        // every pointer is a multiple of 16 bytes (8 of the 8-bit moments)
};
struct AwArgs {
  AwTensor t[kAwMost];
  unsigned first[kAwMost];        // the first CTA of each tensor
  unsigned ctas;                  // parts of kAwSpan elements, all tensors together
  int count, p_dtype, g_dtype;
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

// a / b rounded to nearest, b the same for many a: with y = 1 / b rounded to nearest and q = a y, q + (a - q b) y is the
// correctly rounded quotient (Markstein, IBM J. Res. Dev. 34, 1990, theorem 8), as long as nothing leaves the normal range.
HOA_DEVICE float aw_div(float a, float b, float y) {
  const float m = fabsf(a);
  if (!(m == 0.f || (m > 1e-25f && m < 1e25f))) return __fdiv_rn(a, b);
  const float q = __fmul_rn(a, y);
  return fmaf(fmaf(-q, b, a), y, q);
}
// whether aw_div may be used with b
HOA_DEVICE bool aw_div_by(float b) { return b > 1e-12f && b < 1e12f; }

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

// N bytes from i on
template <bool kVec, int N>
HOA_DEVICE void aw_load8(const void* x, long long i, long long n, unsigned char (&v)[N]) {
  static_assert(N == 8, "one 8-byte piece");
  const unsigned char* b = reinterpret_cast<const unsigned char*>(x) + i;
  if (kVec && i + N <= n) {
    const uint2 t = *reinterpret_cast<const uint2*>(b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = (unsigned char)(t.x >> (8 * e));
      v[4 + e] = (unsigned char)(t.y >> (8 * e));
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = i + e < n ? b[e] : 0;
  }
}
template <bool kVec, int N>
HOA_DEVICE void aw_store8(void* x, long long i, long long n, const unsigned char (&v)[N]) {
  unsigned char* b = reinterpret_cast<unsigned char*>(x) + i;
  if (kVec && i + N <= n) {
    uint2 t = make_uint2(0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t.x |= (uint32_t)v[e] << (8 * e);
      t.y |= (uint32_t)v[4 + e] << (8 * e);
    }
    *reinterpret_cast<uint2*>(b) = t;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (i + e < n) b[e] = v[e];
  }
}

// A warp has one block of 256 elements, a lane 8 consecutive ones of it.
template <int kBits, bool kVec>
HOA_DEVICE void aw_block(const AwArgs& a, const AwTensor& t, long long blk, float lr, float c2, float y2) {
  const int lid = threadIdx.x & 31;
  const long long i = blk * kAwBlock + 8 * lid, n = t.n;
  const long long blocks = (n + kAwBlock - 1) / kAwBlock;
  float g[8], x[8], m[8], v[8];
  unsigned char mb[8], vb[8];
  float ms = 0.f, vs = 0.f;
  // all loads first
  aw_load<kVec>(t.g, a.g_dtype, i, n, g);
  if (t.master) aw_load<kVec>(t.master, HOA_F32, i, n, x);
  else aw_load<kVec>(t.p, a.p_dtype, i, n, x);
  if (kBits == 8) {
    aw_load8<kVec>(t.m, i, n, mb);
    aw_load8<kVec>(t.v, i, n, vb);
    ms = t.scales[blk];
    vs = t.scales[blocks + blk];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m[e] = __fmul_rn(aw_value(mb[e]), ms);
      const float r = __fmul_rn(aw_value(vb[e]), vs);
      v[e] = __fmul_rn(r, r);
    }
  } else {
    aw_load<kVec>(t.m, HOA_F32, i, n, m);
    aw_load<kVec>(t.v, HOA_F32, i, n, v);
  }
  float r[8], mtop = 0.f, rtop = 0.f;
  bool nan_m = false, nan_r = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    m[e] = __fadd_rn(__fmul_rn(m[e], a.b1), __fmul_rn(g[e], a.nb1));
    v[e] = __fadd_rn(__fmul_rn(v[e], a.b2), __fmul_rn(__fmul_rn(g[e], g[e]), a.nb2));
    if (kBits == 8 && i + e >= n) m[e] = v[e] = 0.f;              // (a scale of NaN reaches the elements past the end too)
    r[e] = __fsqrt_rn(v[e]);
    const float den = __fadd_rn(aw_div(r[e], c2, y2), a.eps);
    x[e] = __fsub_rn(__fmul_rn(x[e], a.keep), __fmul_rn(__fdiv_rn(m[e], den), lr));
    mtop = fmaxf(mtop, fabsf(m[e]));
    rtop = fmaxf(rtop, r[e]);
    nan_m |= m[e] != m[e];
    nan_r |= r[e] != r[e];
  }
  if (t.master) aw_store<kVec>(t.master, HOA_F32, i, n, x);
  aw_store<kVec>(t.p, a.p_dtype, i, n, x);
  if (kBits != 8) {
    aw_store<kVec>(t.m, HOA_F32, i, n, m);
    aw_store<kVec>(t.v, HOA_F32, i, n, v);
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mtop = fmaxf(mtop, __shfl_xor_sync(0xffffffffu, mtop, o));
    rtop = fmaxf(rtop, __shfl_xor_sync(0xffffffffu, rtop, o));
  }
  // (a NaN among the moments is the block's scale, as a maximum that propagates it would be)
  const float nan = __int_as_float(0x7fffffff);
  ms = __any_sync(0xffffffffu, nan_m) ? nan : __fmul_rn(mtop, 1.f / 448.f);
  vs = __any_sync(0xffffffffu, nan_r) ? nan : __fmul_rn(rtop, 1.f / 448.f);
  const float ym = aw_div_by(ms) ? __frcp_rn(ms) : 0.f, yr = aw_div_by(vs) ? __frcp_rn(vs) : 0.f;   // (uniform in the warp)
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float qm = ym > 0.f ? aw_div(m[e], ms, ym) : ms > 0.f ? __fdiv_rn(m[e], ms) : 0.f;
    float qr = yr > 0.f ? aw_div(r[e], vs, yr) : vs > 0.f ? __fdiv_rn(r[e], vs) : 0.f;
    if (r[e] > 0.f) qr = fmaxf(qr, 0.001953125f);
    mb[e] = aw_e4m3(qm);
    vb[e] = aw_e4m3(qr);
  }
  aw_store8<kVec>(t.m, i, n, mb);
  aw_store8<kVec>(t.v, i, n, vb);
  if (lid == 0) {
    t.scales[blk] = ms;
    t.scales[blocks + blk] = vs;
  }
}

template <int kBits>
__global__ void __launch_bounds__(kAwThreads) adamw_kernel(const __grid_constant__ AwArgs a) {
  __shared__ float s_lr, s_c2;
  if (threadIdx.x == 0) {
    const double t = (double)*a.step;
    s_lr = (float)(a.lr / (1.0 - pow(a.b1d, t)));
    s_c2 = (float)sqrt(1.0 - pow(a.b2d, t));
  }
  __syncthreads();
  const float lr = s_lr, c2 = s_c2, y2 = __frcp_rn(c2);
  int lo = 0;
  for (unsigned c = blockIdx.x; c < a.ctas; c += gridDim.x) {
    int hi = a.count - 1;                              // the tensor of this part: the last one that starts at or before it
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (a.first[mid] <= c) lo = mid; else hi = mid - 1;
    }
    const AwTensor& t = a.t[lo];
    const long long blk = (long long)(c - a.first[lo]) * (kAwSpan / kAwBlock) + (threadIdx.x >> 5);
    if (blk * kAwBlock >= t.n) continue;
    if (t.vec) aw_block<kBits, true>(a, t, blk, lr, c2, y2);
    else aw_block<kBits, false>(a, t, blk, lr, c2, y2);
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
    return (unsigned)n * 4;
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
    a.lr = lr; a.b1d = beta1; a.b2d = beta2;
    const unsigned grid = ctas < most ? ctas : most;
    if (state_bits == 8) adamw_kernel<8><<<grid, kAwThreads, 0, s>>>(a);
    else adamw_kernel<32><<<grid, kAwThreads, 0, s>>>(a);
    if (int st = launch_status()) return st;
  }
  return HOA_OK;
}
