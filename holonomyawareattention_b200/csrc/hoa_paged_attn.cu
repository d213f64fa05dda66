// Attention of a batch over a paged cache whose first pages all rows share.
//
//   o_i = sum_{j < n_i} softmax_j(q_i . k_j * scale) v_j,   n_i = lens[b] - Tq + t + 1
//   lse_i = log sum_{j < n_i} exp(q_i . k_j * scale)
// for query t of row b.  Keys 0 .. Ls-1 lie in the `shared` pages (Ls = n_shared *
// page), the rest in the row's own `table` pages.  A query that sees no key gives
// o = 0, lse = -inf.  With `paths` (one token a row) out = P o, the inverse
// transport of core/attention_fast_chunked.py:171.
//
// softmax over a union of key sets splits exactly: with m, l, O the maximum, sum
// and unnormalised output of each part, o = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.
// So the shared keys are read once for all rows (the rows of the whole batch are
// the rows of one product), each row's own keys once, either part cut into splits
// along the keys where rows alone would not fill the GPU, and a second kernel
// joins the parts.  Scores, maxima, sums and O are fp32; exponents are base 2.
#include "hoa_paged_attn.cuh"

namespace hoa {

// ---------------------------------------------------------------------------
// any head dim and alignment, fp32 products on the CUDA cores
// ---------------------------------------------------------------------------
constexpr int kPsRows = 16, kPsKeys = 64, kPsThreads = 128;

__global__ void __launch_bounds__(kPsThreads) paged_attn_simt_kernel(const __grid_constant__ PaArgs p, unsigned first) {
  extern __shared__ float sm[];
  const int d = p.d, ld = d | 1;                       // odd row stride: rows fall on different banks
  float* Qs = sm;                                      // [16][ld]
  float* Ks = Qs + kPsRows * ld;                       // [64][ld]
  float* Vs = Ks + kPsKeys * ld;                       // [64][ld]
  float* Ps = Vs + kPsKeys * ld;                       // [16][64]
  PaItem it = pa_item(p, first + blockIdx.x, kPsRows, kPsKeys);
  const int tid = threadIdx.x, row = tid >> 3, kg = tid & 7;
  const PaRow my = pa_row(p, it, it.row0 + row);
  for (int i = tid; i < kPsRows * d; i += kPsThreads) {
    const int r = i / d, c = i % d;
    const PaRow q = pa_row(p, it, it.row0 + r);
    Qs[r * ld + c] = q.ok ? load_elem(p.q, q.b * p.qsb + q.t * p.qst + q.h * p.qsh + c, p.dtype) : 0.f;
  }
  const int seen = my.ok ? min(my.seen - it.key_base, it.k1) : 0;   // keys of this part that the row sees
  __shared__ int s_top;                                // no key past the last one that a row sees is read
  if (tid == 0) s_top = 0;
  __syncthreads();
  if (kg == 0) atomicMax(&s_top, seen);
  __syncthreads();
  it.k1 = min(it.k1, s_top);
  float o[16], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.f;
  for (int k0 = it.k0; k0 < it.k1; k0 += kPsKeys) {
    __syncthreads();
    for (int i = tid; i < kPsKeys * d; i += kPsThreads) {
      const int j = i / d, c = i % d;
      const long long at = k0 + j < it.k1 ? pa_key(p, it, k0 + j) : -1;
      Ks[j * ld + c] = at >= 0 ? load_elem(p.kp, at + c, p.dtype) : 0.f;
      Vs[j * ld + c] = at >= 0 ? load_elem(p.vp, at + c, p.dtype) : 0.f;
    }
    __syncthreads();
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = 0.f;
    for (int c = 0; c < d; ++c) {
      const float qv = Qs[row * ld + c];
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = fmaf(qv, Ks[(kg + 8 * j) * ld + c], s[j]);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s[j] = k0 + kg + 8 * j < seen ? s[j] * p.scale_log2 : -INFINITY;
      mx = fmaxf(mx, s[j]);
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float mn = fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.f : mn;      // a row that has seen no key yet
    const float corr = exp2f(m - ref);
    float ps = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float e = exp2f(s[j] - ref);
      Ps[row * kPsKeys + kg + 8 * j] = e;
      ps += e;
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) ps += __shfl_xor_sync(0xffffffffu, ps, x);
    l = l * corr + ps;
    m = mn;
    __syncwarp();                                      // a row's weights come from its own warp
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] *= corr;
    for (int k = 0; k < kPsKeys; ++k) {
      const float e = Ps[row * kPsKeys + k];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (kg + 8 * i < d) o[i] = fmaf(e, Vs[k * ld + kg + 8 * i], o[i]);
    }
  }
  if (!my.ok) return;
  const long long part = (long long)it.slot * p.rows + my.grow;
  if (kg == 0) p.part_ml[part] = make_float2(m, l);
  if (l > 0.f) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (kg + 8 * i < d) p.part_o[part * d + kg + 8 * i] = o[i];
  }
}

// ---------------------------------------------------------------------------
// join the parts of each (row, query, head); optionally out = P o
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(128) paged_attn_join_kernel(const __grid_constant__ PaArgs p) {
  __shared__ float s_o[128];
  const int d = p.d, c = threadIdx.x, slots = p.ns1 + p.ns2;
  for (long long g = blockIdx.x; g < p.rows; g += gridDim.x) {
    float m = -INFINITY;
    for (int s = 0; s < slots; ++s) {
      const float2 ml = p.part_ml[s * p.rows + g];
      if (ml.y > 0.f) m = fmaxf(m, ml.x);
    }
    float l = 0.f, o = 0.f;
    for (int s = 0; s < slots; ++s) {
      const float2 ml = p.part_ml[s * p.rows + g];
      if (!(ml.y > 0.f)) continue;
      const float w = exp2f(ml.x - m);
      l = fmaf(w, ml.y, l);
      if (c < d) o = fmaf(w, p.part_o[(s * p.rows + g) * d + c], o);
    }
    o = l > 0.f ? o / l : 0.f;
    if (c == 0) p.lse[g] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
    if (p.paths == nullptr) {
      if (c < d) store_elem(p.out, g * d + c, p.out_dtype, o);
      continue;
    }
    __syncthreads();
    s_o[c] = c < d ? o : 0.f;
    __syncthreads();
    const float* P = p.paths + g * d * d;
    for (int i = c >> 5; i < d; i += 4) {
      float y = 0.f;
      for (int j = c & 31; j < d; j += 32) y = fmaf(P[i * d + j], s_o[j], y);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) y += __shfl_xor_sync(0xffffffffu, y, x);
      if ((c & 31) == 0) store_elem(p.out, g * d + i, p.out_dtype, y);
    }
  }
}

}  // namespace hoa

using namespace hoa;

static bool pa_shape_ok(int B, int Tq, int H, int Hk, int d, int page, int n_shared, int W, int num_sms) {
  return B >= 1 && Tq >= 1 && Hk >= 1 && H >= Hk && H % Hk == 0 && d >= 1 && page >= 1 && n_shared >= 0 && W >= 0 &&
         num_sms >= 1;
}

static size_t pa_bytes(const PaPlan& pl, int B, int Tq, int H, int d) {
  return ((size_t)pl.ns1 + pl.ns2) * B * Tq * H * (8 + 4 * (size_t)d) + 256;
}

extern "C" size_t hoa_paged_attn_workspace_bytes(int B, int Tq, int H, int Hk, int d, int page, int n_shared, int W,
                                                 int num_sms) {
  if (!pa_shape_ok(B, Tq, H, Hk, d, page, n_shared, W, num_sms)) return 0;
  size_t most = 0;                                 // enough for whichever kernels take the call
  for (int k = 0; k < 3; ++k) {
    const size_t n = pa_bytes(pa_plan(B, Tq, H, Hk, page, n_shared, W, num_sms, k > 0, k > 1), B, Tq, H, d);
    most = n > most ? n : most;
  }
  return most;
}

static int run_items(int kind, const PaArgs& a, long long first, long long items, cudaStream_t s) {
  if (items == 0) return HOA_OK;
  if (kind == kPaTc) return paged_attn_tc(a, (unsigned)first, (unsigned)items, s);
  if (kind == kPaMma) return paged_attn_mma(a, (unsigned)first, (unsigned)items, s);
  const size_t smem = ((kPsRows + 2 * kPsKeys) * (size_t)(a.d | 1) + kPsRows * kPsKeys) * sizeof(float);
  if (cudaFuncSetAttribute(paged_attn_simt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return HOA_ERR_LAUNCH;
  paged_attn_simt_kernel<<<(unsigned)items, kPsThreads, smem, s>>>(a, (unsigned)first);
  return launch_status();
}

extern "C" int hoa_paged_attn_fwd(const void* q, const long long* q_strides, const void* k_pages, const void* v_pages,
                                  const long long* page_strides, int dtype, const int* shared, int n_shared,
                                  const int* table, long long table_stride, int W, const int* lens, const float* paths,
                                  void* out, int out_dtype, float* lse, float softmax_scale, int B, int Tq, int H, int Hk,
                                  int d, int page, int n_pages, int num_sms, void* workspace, size_t workspace_bytes,
                                  int* status, void* stream) {
  if (!q || !q_strides || !k_pages || !v_pages || !page_strides || !lens || !out || !lse || !workspace ||
      !pa_shape_ok(B, Tq, H, Hk, d, page, n_shared, W, num_sms) || n_pages < 1 || (n_shared > 0 && !shared) ||
      (W > 0 && !table) || (paths && Tq != 1))
    return HOA_ERR_INVALID_ARG;
  if ((dtype != HOA_F32 && dtype != HOA_BF16) || (out_dtype != HOA_F32 && out_dtype != HOA_BF16) || d > 128)
    return HOA_ERR_UNSUPPORTED;
  // key positions and item numbers are ints
  if ((long long)(n_shared + (long long)W) * page > 0x7fff0000ll) return HOA_ERR_UNSUPPORTED;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                         (uintptr_t)(page_strides[0] * 2) | (uintptr_t)(page_strides[1] * 2) | (uintptr_t)(page_strides[2] * 2);
  const bool tensor = dtype == HOA_BF16 && d % 8 == 0 && (bits & 15) == 0;
  const PaPlan pl = pa_plan(B, Tq, H, Hk, page, n_shared, W, num_sms, tensor, tensor && softmax_scale > 0.f);
  if (workspace_bytes < pa_bytes(pl, B, Tq, H, d)) return HOA_ERR_WORKSPACE;
  const long long items1 = (long long)pl.tiles1 * Hk * pl.ns1, items2 = (long long)B * Hk * pl.tiles2 * pl.ns2;
  if (items1 + items2 > 0x7fffffffll) return HOA_ERR_UNSUPPORTED;
  PaArgs a{};
  a.q = q; a.qsb = q_strides[0]; a.qst = q_strides[1]; a.qsh = q_strides[2];
  a.kp = k_pages; a.vp = v_pages; a.ps = page_strides[0]; a.hs = page_strides[1]; a.ts = page_strides[2];
  a.shared = shared; a.n_shared = n_shared; a.table = table; a.tstride = table_stride; a.W = W; a.lens = lens;
  a.paths = paths; a.out = out; a.out_dtype = out_dtype; a.lse = lse; a.dtype = dtype;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.B = B; a.Tq = Tq; a.H = H; a.Hk = Hk; a.G = H / Hk; a.d = d; a.page = page; a.n_pages = n_pages;
  a.rows = (long long)B * Tq * H;
  a.ns1 = pl.ns1; a.ns2 = pl.ns2; a.tiles1 = pl.tiles1; a.tiles2 = pl.tiles2;
  a.status = status;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)(pl.ns1 + pl.ns2) * a.rows * d);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int st;
  if (pl.kind1 == pl.kind2) {                      // one launch for both parts
    st = run_items(pl.kind1, a, 0, items1 + items2, s);
  } else {
    st = run_items(pl.kind1, a, 0, items1, s);
    if (st == HOA_OK) st = run_items(pl.kind2, a, items1, items2, s);
  }
  if (st != HOA_OK) return st;
  paged_attn_join_kernel<<<(unsigned)(a.rows < 148 * 64 ? a.rows : 148 * 64), 128, 0, s>>>(a);
  return launch_status();
}
