// The path step: one generated token of every row (b, h).
//
//   P' = expm(skew(edge_scale a)) P          the edge from the row's last token to this one
//   q^ = P'^T q,  k^ = P'^T k,  v^ = P'^T v   k^ and v^ go to the row's page, slot lens[b] - 1
// (core/attention_fast_chunked.py:86-94 and :108-110 for one position.)  A row at
// its first token (lens 1) has no edge: P' = I.  A row without a token (lens 0)
// keeps P, gets q^ = 0 and writes nothing.
#include "hoa_sm100.cuh"

namespace hoa {

// degree-8 Taylor polynomial of exp in three products, see kT8 in hoa_link.cu
constexpr float kStX1 = 0.059249617736388274f, kStX2 = 0.014812404434097069f, kStX3 = 0.36450763864714936f,
                kStX5 = 0.29469080354241967f, kStX6 = 0.025771599210148963f, kStX7 = 0.11303901220301756f,
                kStY2 = 0.13549236135285064f;
constexpr float kStTheta = 0.6f;

struct StepArgs {
  const float* a; int banked, stride; const float* a_bias; float edge_scale;
  const float* P; float* P_out;
  const void* qkv; int qkv_dtype; long long qkv_stride;    // row stride, elements
  void* qh; void* kp; void* vp; int dtype;                 // q^ and the pages
  long long ps, hs, ts;
  const int* table; long long tstride; const int* lens;
  int B, H, d, page, W, n_pages;
  int* status;
};

HOA_DEVICE void st_fail(int* status) {
  if (status != nullptr) *reinterpret_cast<volatile int*>(status) = HOA_ERR_PAGES;
}

constexpr int kStThreads = 256;

// acc (thread (ty, tx) of 16 x 16: rows ty + 16 i, columns tx + 16 j) = X Y
HOA_DEVICE void st_mm(const float* X, const float* Y, int d, int ty, int tx, float (&acc)[8][8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
  for (int k = 0; k < d; ++k) {
    float x[8], y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ty + 16 * i < d ? X[(ty + 16 * i) * d + k] : 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = tx + 16 * j < d ? Y[k * d + tx + 16 * j] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
  }
}

template <class F>
HOA_DEVICE void st_each(int d, int ty, int tx, F f) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (ty + 16 * i < d && tx + 16 * j < d) f(i, j, ty + 16 * i, tx + 16 * j);
}

__global__ void __launch_bounds__(kStThreads) path_step_kernel(const __grid_constant__ StepArgs p) {
  extern __shared__ float sm[];
  const int d = p.d, dd = d * d;
  float *A = sm, *B1 = sm + dd, *B2 = sm + 2 * dd, *vec = sm + 3 * dd;   // vec: 3 d, and column sums d
  __shared__ int s_sq;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int u = blockIdx.x, b = u / p.H, h = u % p.H;
  const int len = p.lens[b];
  const float* P = p.P + (long long)u * dd;
  float* Po = p.P_out + (long long)u * dd;
  if (len <= 0) {
    for (int i = tid; i < dd; i += kStThreads) Po[i] = P[i];
    for (int i = tid; i < d; i += kStThreads) store_elem(p.qh, (long long)u * d + i, p.dtype, 0.f);
    return;
  }
  for (int i = tid; i < 3 * d; i += kStThreads)
    vec[i] = load_elem(p.qkv, b * p.qkv_stride + (long long)h * 3 * d + i, p.qkv_dtype);
  if (len == 1) {
    for (int i = tid; i < dd; i += kStThreads) B2[i] = (i / d == i % d) ? 1.f : 0.f;
  } else {
    const float* g = p.a + ((long long)b * p.H + h) * p.stride;
    const float* bias = p.a_bias ? p.a_bias + (long long)h * p.stride : nullptr;
    for (int i = tid; i < dd; i += kStThreads) {
      const int r = i / d, c = i % d;
      float v = 0.f;
      if (r != c) {
        const int lo = min(r, c), hi = max(r, c);
        const int at = p.banked ? gen_banked_slot(lo, hi, d) : lo * (2 * d - lo - 1) / 2 + hi - lo - 1;
        v = (g[at] + (bias ? bias[at] : 0.f)) * p.edge_scale;
        if (r > c) v = -v;
      }
      A[i] = v;
    }
    __syncthreads();
    float acc[8][8];
    st_mm(A, A, d, ty, tx, acc);                       // A^2
    st_each(d, ty, tx, [&](int i, int j, int r, int c) { B1[r * d + c] = acc[i][j]; });
    __syncthreads();
    // ||A^2||_1 bounds ||A||_2^2 (A is normal): scale by 2^-s to theta <= 0.6, square s times
    if (tid < d) {
      float s = 0.f;
      for (int r = 0; r < d; ++r) s += fabsf(B1[r * d + tid]);
      vec[3 * d + tid] = s;
    }
    __syncthreads();
    if (tid == 0) {
      float mx = 0.f;
      for (int c = 0; c < d; ++c) mx = fmaxf(mx, vec[3 * d + c]);
      float theta = sqrtf(mx);
      int s = 0;
      while (theta > kStTheta && s < 64) { theta *= 0.5f; ++s; }
      s_sq = s;
    }
    __syncthreads();
    const int nsq = s_sq;
    const float sa = ldexpf(1.f, -nsq), sa2 = ldexpf(1.f, -2 * nsq);
    for (int i = tid; i < dd; i += kStThreads) {
      A[i] *= sa;
      B1[i] *= sa2;
      B2[i] = kStX1 * A[i] + kStX2 * B1[i];
    }
    __syncthreads();
    st_mm(B1, B2, d, ty, tx, acc);                     // A4 = A2 (x1 A + x2 A2)
    __syncthreads();
    // left factor x3 A2 + A4 in B1, right factor in B2, E0 = A + y2 A2 in A
    st_each(d, ty, tx, [&](int i, int j, int r, int c) {
      const int o = r * d + c;
      const float a = A[o], a2 = B1[o], a4 = acc[i][j];
      B1[o] = kStX3 * a2 + a4;
      B2[o] = (r == c ? 1.f : 0.f) + kStX5 * a + kStX6 * a2 + kStX7 * a4;
      A[o] = a + kStY2 * a2;
    });
    __syncthreads();
    st_mm(B1, B2, d, ty, tx, acc);
    st_each(d, ty, tx, [&](int i, int j, int r, int c) { A[r * d + c] += acc[i][j]; });   // E = G - I
    __syncthreads();
    for (int s = 0; s < nsq; ++s) {                    // (I + E)^2 = I + (2 E + E E)
      st_mm(A, A, d, ty, tx, acc);
      __syncthreads();
      st_each(d, ty, tx, [&](int i, int j, int r, int c) { A[r * d + c] = fmaf(2.f, A[r * d + c], acc[i][j]); });
      __syncthreads();
    }
    for (int i = tid; i < dd; i += kStThreads) B2[i] = P[i];
    __syncthreads();
    st_mm(A, B2, d, ty, tx, acc);                      // P' = P + E P
    __syncthreads();
    st_each(d, ty, tx, [&](int i, int j, int r, int c) { B2[r * d + c] += acc[i][j]; });
  }
  __syncthreads();
  for (int i = tid; i < dd; i += kStThreads) Po[i] = B2[i];
  const int pos = len - 1, pg = pos / p.page;
  const int id = pg < p.W ? p.table[b * p.tstride + pg] : -1;
  const bool ok = id >= 0 && id < p.n_pages;
  if (!ok && tid == 0) st_fail(p.status);
  const long long slot = ok ? id * p.ps + h * p.hs + (long long)(pos % p.page) * p.ts : 0;
  for (int i = tid; i < 3 * d; i += kStThreads) {
    const int w = i / d, c = i % d;
    float y = 0.f;
    for (int r = 0; r < d; ++r) y = fmaf(B2[r * d + c], vec[w * d + r], y);
    if (w == 0) store_elem(p.qh, (long long)u * d + c, p.dtype, y);
    else if (ok) store_elem(w == 1 ? p.kp : p.vp, slot + c, p.dtype, y);
  }
}

}  // namespace hoa

using namespace hoa;

extern "C" int hoa_path_step(const float* a, int a_dtype, const float* a_bias, float edge_scale, const float* P, float* P_out,
                             const void* qkv, int qkv_dtype, long long qkv_stride, void* qh, void* k_pages, void* v_pages,
                             int dtype, const long long* page_strides, const int* table, long long table_stride, int W,
                             const int* lens, int B, int H, int d, int page, int n_pages, int* status, void* stream) {
  if (!a || !P || !P_out || !qkv || !qh || !k_pages || !v_pages || !page_strides || !table || !lens || B < 1 || H < 1 ||
      d < 2 || page < 1 || W < 1 || n_pages < 1)
    return HOA_ERR_INVALID_ARG;
  const int stride = gen_row_stride(a_dtype, d);
  if (d > 120 || stride == 0 || gen_elem_dtype(a_dtype) != HOA_F32 || (qkv_dtype != HOA_F32 && qkv_dtype != HOA_BF16) ||
      (dtype != HOA_F32 && dtype != HOA_BF16) || (long long)B * H > 0x7fffffffll)
    return HOA_ERR_UNSUPPORTED;
  StepArgs s{a, gen_is_banked(a_dtype) ? 1 : 0, stride, a_bias, edge_scale, P, P_out, qkv, qkv_dtype, qkv_stride, qh,
             k_pages, v_pages, dtype, page_strides[0], page_strides[1], page_strides[2], table, table_stride, lens,
             B, H, d, page, W, n_pages, status};
  const size_t smem = (3 * (size_t)d * d + 4 * d) * sizeof(float);
  if (cudaFuncSetAttribute(path_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return HOA_ERR_LAUNCH;
  path_step_kernel<<<(unsigned)(B * H), kStThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(s);
  return launch_status();
}
