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
  pa_let_next_start();
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
  pa_end_after_previous();
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
// kWpr warps share an output row: one where rows are many, eight (a CTA a row) where
// the parts or P are most of the bytes.  A lane holds four columns (V = 4, d % 4 == 0)
// or up to four that are 32 apart.  Launched while the items still run: P, which does
// not depend on them, is read before the wait (8 lanes a row of P, 32 rows a pass,
// all passes' loads at once), so that its bytes - most of a decode step's, 4 d^2 a
// head - are under way when the parts arrive.
constexpr int kPjThreads = 256;

template <int V, int kWpr, bool kPaths>
__global__ void __launch_bounds__(kPjThreads) paged_attn_join_kernel(const __grid_constant__ PaArgs p) {
  static_assert(!kPaths || kWpr == 8, "P takes the whole CTA");
  __shared__ float4 s_o[8][32];
  __shared__ float s_l[8];
  const int d = p.d, slots = p.ns1 + p.ns2, warp = threadIdx.x >> 5, lid = threadIdx.x & 31;
  const int w = warp % kWpr;
  const long long g = (long long)blockIdx.x * (8 / kWpr) + warp / kWpr;
  const bool ok = g < p.rows;                          // (uniform in the warps that share a row)
  float4 P[4][4];                                      // pass, chunk of 4 columns
  const int pr = threadIdx.x >> 3, pq = threadIdx.x & 7;
  if constexpr (kPaths) {
    const float* Pg = p.paths + g * d * d;
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int r = pr + 32 * x, c = 4 * (pq + 8 * y);
        P[x][y] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < d) {
          if (V == 4) {
            if (c < d) P[x][y] = *reinterpret_cast<const float4*>(Pg + r * d + c);
          } else {
            const float* at = Pg + r * d + c;
            if (c < d) P[x][y].x = at[0];
            if (c + 1 < d) P[x][y].y = at[1];
            if (c + 2 < d) P[x][y].z = at[2];
            if (c + 3 < d) P[x][y].w = at[3];
          }
        }
      }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float m = -INFINITY;
  if (ok)
    for (int s = lid; s < slots; s += 32) {
      const float2 ml = p.part_ml[s * p.rows + g];
      if (ml.y > 0.f) m = fmaxf(m, ml.x);
    }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  if (ok && m != -INFINITY) {
#pragma unroll 4
    for (int s = w; s < slots; s += kWpr) {
      const float2 ml = p.part_ml[s * p.rows + g];
      const float f = ml.y > 0.f ? exp2f(ml.x - m) : 0.f;
      l = fmaf(f, ml.y, l);
      const float* at = p.part_o + (s * p.rows + g) * d;
      if (V == 4) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (4 * lid < d && ml.y > 0.f) v = *reinterpret_cast<const float4*>(at + 4 * lid);   // (a part without a key wrote no O)
        o[0] = fmaf(f, v.x, o[0]); o[1] = fmaf(f, v.y, o[1]); o[2] = fmaf(f, v.z, o[2]); o[3] = fmaf(f, v.w, o[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (lid + 32 * e < d && ml.y > 0.f) o[e] = fmaf(f, at[lid + 32 * e], o[e]);
      }
    }
  }
  if constexpr (kWpr > 1) {
    s_o[w][lid] = make_float4(o[0], o[1], o[2], o[3]);
    if (lid == 0) s_l[w] = l;
    __syncthreads();
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    l = 0.f;
#pragma unroll
    for (int x = 0; x < kWpr; ++x) {
      const float4 v = s_o[x][lid];
      t[0] += v.x; t[1] += v.y; t[2] += v.z; t[3] += v.w;
      l += s_l[x];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = t[e];
  }
  if (!ok) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= inv;
  if (w == 0 && lid == 0) p.lse[g] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  if constexpr (kPaths) {
    float* so = reinterpret_cast<float*>(s_o);         // o in column order, zero past d
    __syncthreads();
    if (w == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = V == 4 ? 4 * lid + e : lid + 32 * e;
        so[c] = c < d ? o[e] : 0.f;
      }
    }
    __syncthreads();
    float4 q[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) q[y] = *reinterpret_cast<const float4*>(so + 4 * (pq + 8 * y));
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      float y = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        y = fmaf(P[x][k].x, q[k].x, fmaf(P[x][k].y, q[k].y, fmaf(P[x][k].z, q[k].z, fmaf(P[x][k].w, q[k].w, y))));
#pragma unroll
      for (int k = 1; k < 8; k <<= 1) y += __shfl_xor_sync(0xffffffffu, y, k);
      const int r = pr + 32 * x;
      if (pq == 0 && r < d) store_elem(p.out, g * d + r, p.out_dtype, y);
    }
  } else if (w == 0) {
    if (V == 4 && 4 * lid < d) {
      if (p.out_dtype == HOA_BF16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(o[0], o[1]), b = __floats2bfloat162_rn(o[2], o[3]);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + g * d + 4 * lid) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
      } else {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + g * d + 4 * lid) = make_float4(o[0], o[1], o[2], o[3]);
      }
    } else if (V == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lid + 32 * e < d) store_elem(p.out, g * d + lid + 32 * e, p.out_dtype, o[e]);
    }
  }
}

template <int V, int kWpr, bool kPaths>
static int launch_join(const PaArgs& a, bool early, cudaStream_t s) {
  const long long blocks = (a.rows + 8 / kWpr - 1) / (8 / kWpr);
  if (blocks > 0x7fffffffll) return HOA_ERR_UNSUPPORTED;
  return pa_launch(paged_attn_join_kernel<V, kWpr, kPaths>, (unsigned)blocks, kPjThreads, 0, s, early, a);
}

static int join(const PaArgs& a, bool early, cudaStream_t s) {
  // 16-byte accesses: four columns a lane of o, the parts and P
  const bool v4 = a.d % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.paths) |
                                    reinterpret_cast<uintptr_t>(a.part_o)) & 15) == 0;
  if (a.paths) return v4 ? launch_join<4, 8, true>(a, early, s) : launch_join<1, 8, true>(a, early, s);
  // eight warps a row where one a row would leave SMs without work and there are parts to share
  if (a.rows < 148 * 16 && a.ns1 + a.ns2 > 4) return v4 ? launch_join<4, 8, false>(a, early, s) : launch_join<1, 8, false>(a, early, s);
  return v4 ? launch_join<4, 1, false>(a, early, s) : launch_join<1, 1, false>(a, early, s);
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

// `early`: may start while the launch before it (the other part's items) still runs
static int run_items(int kind, const PaArgs& a, long long first, long long items, bool early, cudaStream_t s) {
  if (items == 0) return HOA_OK;
  if (kind == kPaTc) return paged_attn_tc(a, (unsigned)first, (unsigned)items, early, s);
  if (kind == kPaMma) return paged_attn_mma(a, (unsigned)first, (unsigned)items, early, s);
  const size_t smem = ((kPsRows + 2 * kPsKeys) * (size_t)(a.d | 1) + kPsRows * kPsKeys) * sizeof(float);
  if (cudaFuncSetAttribute(paged_attn_simt_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return HOA_ERR_LAUNCH;
  return pa_launch(paged_attn_simt_kernel, (unsigned)items, kPsThreads, smem, s, early, a, (unsigned)first);
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
  // with 2^s >= page > 2^(s-1): ceil(2^(31+s) / page) < 2^32, exact for j < 2^31
  int sh = 0;
  while ((1ll << sh) < page) ++sh;
  a.page_mul = page > 1 ? (unsigned)(((1ull << (31 + sh)) + page - 1) / page) : 0u;
  a.page_shift = sh - 1;
  a.ns1 = pl.ns1; a.ns2 = pl.ns2; a.tiles1 = pl.tiles1; a.tiles2 = pl.tiles2;
  a.status = status;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)(pl.ns1 + pl.ns2) * a.rows * d);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int st;
  if (pl.kind1 == pl.kind2) {                      // one launch for both parts
    st = run_items(pl.kind1, a, 0, items1 + items2, false, s);
  } else {
    st = run_items(pl.kind1, a, 0, items1, false, s);
    if (st == HOA_OK) st = run_items(pl.kind2, a, items1, items2, items1 > 0, s);
  }
  if (st != HOA_OK) return st;
  return join(a, items1 + items2 > 0, s);
}
