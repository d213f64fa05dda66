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
// Kernels: here for fp32 and odd shapes (CUDA cores) and the join; bf16 in
// hoa_paged_attn_mma.cu (few rows) and hoa_paged_attn_tc.cu (many), chosen in pa_plan.
#include "hoa_paged_attn.cuh"

namespace hoa {

// ---------------------------------------------------------------------------
// any head dim, type and alignment, fp32 products on the CUDA cores
// ---------------------------------------------------------------------------
// RT = 8 R query rows against 64 keys at a time; 128 threads as 8 x 16: thread (ty, tx) has rows
// ty R .. + R - 1 and keys tx + 16 j of the scores, columns 4 tx + 64 k of the output.  Rows of K and V
// are padded to an odd number of 16-byte chunks, so that the 16 keys of a warp's read fall on different
// banks.  Few rows (R = 2) are bound by the loads, 8 d bytes a key; many (R = 4) by the FMAs, 4 d a key
// and row: 32 rows halve the shared-memory reads an FMA needs.  Measured in fp32: 16 rows of 16 heads of 96 over 4096
// shared tokens and their own 85 us; 32 queries of 8 rows over 2048 tokens 88 us, 17 TFLOP/s.
constexpr int kPsKeys = 64, kPsThreads = 128;

HOA_DEVICE int ps_ld(int d) { return ((d + 3) / 4 | 1) * 4; }    // floats of a padded row

// V4: fp32 with d % 4 == 0 and 16-byte aligned rows
template <int R, bool V4>
__global__ void __launch_bounds__(kPsThreads) paged_attn_simt_kernel(const __grid_constant__ PaArgs p, unsigned first) {
  constexpr int RT = 8 * R;
  extern __shared__ float sm[];
  pa_begin(p.leads);
  const int d = p.d, ld = ps_ld(d), d4 = (d + 3) / 4;
  float* Qs = sm;                                      // [RT][ld]
  float* Ks = Qs + RT * ld;                            // [64][ld]
  float* Vs = Ks + kPsKeys * ld;                       // [64][ld]
  float* Ps = Vs + kPsKeys * ld;                       // [RT][68] weights
  __shared__ int s_top;
  __shared__ long long s_key[kPsKeys];
  PaItem it = pa_item(p, first + blockIdx.x, RT, kPsKeys);
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15, warp = tid >> 5, lid = tid & 31;
  PaRow my[R];
  int seen[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    my[i] = pa_row(p, it, it.row0 + ty * R + i);
    seen[i] = my[i].ok ? min(my[i].seen - it.key_base, it.k1) : 0;   // keys of this part that the row sees
  }
  if (tid == 0) s_top = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (tx == 0) atomicMax(&s_top, seen[i]);
#pragma unroll
  for (int i = 0; i < R; ++i)                          // the 16 threads of a row read it
    for (int c = tx; c < ld; c += 16)
      Qs[(ty * R + i) * ld + c] =
          my[i].ok && c < d ? load_elem(p.q, my[i].b * p.qsb + my[i].t * p.qst + my[i].h * p.qsh + c, p.dtype) : 0.f;
  __syncthreads();
  it.k1 = min(it.k1, s_top);                           // no key past the last one that a row sees is read
  float4 o[R][2];
  float m[R], l[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    o[i][0] = o[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  for (int k0 = it.k0; k0 < it.k1; k0 += kPsKeys) {
    __syncthreads();                                   // the last tile has been read
    if (tid < kPsKeys) s_key[tid] = k0 + tid < it.k1 ? pa_key(p, it, k0 + tid) : -1;
    __syncthreads();
    if (V4) {
#pragma unroll 8
      for (int j = warp; j < kPsKeys; j += 4) {        // a warp a key, a lane 16 bytes of it
        const long long at = s_key[j];
        float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
        if (lid < d4) {
          if (at >= 0) {
            k = *reinterpret_cast<const float4*>(static_cast<const float*>(p.kp) + at + 4 * lid);
            v = *reinterpret_cast<const float4*>(static_cast<const float*>(p.vp) + at + 4 * lid);
          }
          *reinterpret_cast<float4*>(Ks + j * ld + 4 * lid) = k;
          *reinterpret_cast<float4*>(Vs + j * ld + 4 * lid) = v;
        }
      }
    } else {
#pragma unroll 4
      for (int j = warp; j < kPsKeys; j += 4) {
        const long long at = s_key[j];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = lid + 32 * e;
          if (c < 4 * d4) {
            const bool in = at >= 0 && c < d;
            Ks[j * ld + c] = in ? load_elem(p.kp, at + c, p.dtype) : 0.f;
            Vs[j * ld + c] = in ? load_elem(p.vp, at + c, p.dtype) : 0.f;
          }
        }
      }
    }
    __syncthreads();
    float s[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 2
    for (int c = 0; c < d4; ++c) {
      float4 q[R], k[4];
#pragma unroll
      for (int i = 0; i < R; ++i) q[i] = *reinterpret_cast<const float4*>(Qs + (ty * R + i) * ld + 4 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * j) * ld + 4 * c);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = fmaf(q[i].x, k[j].x, fmaf(q[i].y, k[j].y, fmaf(q[i].z, k[j].z, fmaf(q[i].w, k[j].w, s[i][j]))));
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = k0 + tx + 16 * j < seen[i] ? s[i][j] * p.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[i], mx), ref = mn == -INFINITY ? 0.f : mn;   // (a row that has seen no key yet)
      const float corr = exp2f(m[i] - ref);
      m[i] = mn;
      float ps = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(s[i][j] - ref);
        Ps[(ty * R + i) * 68 + tx + 16 * j] = e;
        ps += e;
      }
      l[i] = l[i] * corr + ps;                         // this thread's keys only; joined at the end
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        o[i][k].x *= corr; o[i][k].y *= corr; o[i][k].z *= corr; o[i][k].w *= corr;
      }
    }
    __syncwarp();                                      // a row's weights come from its own warp
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (4 * tx + 64 * g >= d) break;
#pragma unroll 4
      for (int k = 0; k < kPsKeys; k += 4) {
        float4 w[R];
#pragma unroll
        for (int i = 0; i < R; ++i) w[i] = *reinterpret_cast<const float4*>(Ps + (ty * R + i) * 68 + k);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 v = *reinterpret_cast<const float4*>(Vs + (k + e) * ld + 4 * tx + 64 * g);
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const float f = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
            o[i][g].x = fmaf(f, v.x, o[i][g].x); o[i][g].y = fmaf(f, v.y, o[i][g].y);
            o[i][g].z = fmaf(f, v.z, o[i][g].z); o[i][g].w = fmaf(f, v.w, o[i][g].w);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
  wait_previous();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (!my[i].ok) continue;
    const long long part = (long long)it.slot * p.rows + my[i].grow;
    if (tx == 0) p.part_ml[part] = make_float2(m[i], l[i]);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int c = 4 * tx + 64 * g;
      float* at = p.part_o + part * d + c;
      const float v[4] = {o[i][g].x, o[i][g].y, o[i][g].z, o[i][g].w};
      if (V4) {
        if (c < d) *reinterpret_cast<float4*>(at) = o[i][g];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < d) at[e] = v[e];
      }
    }
  }
}

template <int R, bool V4>
static int launch_simt(const PaArgs& a, unsigned first, unsigned items, cudaStream_t s) {
  const int ld = ((a.d + 3) / 4 | 1) * 4;
  const size_t smem = ((8 * R + 2 * kPsKeys) * (size_t)ld + 8 * R * 68) * sizeof(float);
  static std::atomic<unsigned long long> done{0};
  const size_t most = ((8 * R + 2 * kPsKeys) * (size_t)132 + 8 * R * 68) * sizeof(float);   // at d = 128
  if (!allow_smem(paged_attn_simt_kernel<R, V4>, most, done)) return HOA_ERR_LAUNCH;
  return launch_early(paged_attn_simt_kernel<R, V4>, items, 1, kPsThreads, smem, s, a, first);
}

static int paged_attn_simt(const PaArgs& a, int tile_rows, unsigned first, unsigned items, cudaStream_t s) {
  const bool v4 = a.dtype == HOA_F32 && a.d % 4 == 0 &&
                  ((reinterpret_cast<uintptr_t>(a.kp) | reinterpret_cast<uintptr_t>(a.vp) | (uintptr_t)(a.ps * 4) |
                    (uintptr_t)(a.hs * 4) | (uintptr_t)(a.ts * 4)) & 15) == 0;
  if (tile_rows == 32) return v4 ? launch_simt<4, true>(a, first, items, s) : launch_simt<4, false>(a, first, items, s);
  return v4 ? launch_simt<2, true>(a, first, items, s) : launch_simt<2, false>(a, first, items, s);
}

// ---------------------------------------------------------------------------
// fp32, up to 4 query rows: bound by the loads alone
// ---------------------------------------------------------------------------
// Eight lanes share a key (CH chunks of 4 columns each), a warp has four keys at a time and takes two
// such steps an iteration, straight from global memory to registers.  Every group of eight lanes keeps
// its own (m, l, O): a step needs three shuffles a row and no barrier; groups and warps join at the end.
// Two rows of 4 heads of 48 over 190 tokens: 8 us with the join (14 on the tiles of 16 rows).
constexpr int kPvThreads = 128;

template <int CH, int NR>
__global__ void __launch_bounds__(kPvThreads) paged_attn_vec_kernel(const __grid_constant__ PaArgs p, unsigned first) {
  __shared__ float s_o[4][NR][32 * CH];
  __shared__ float2 s_ml[4][NR];
  pa_begin(p.leads);
  const PaItem it = pa_item(p, first + blockIdx.x, NR, 16);
  const int warp = threadIdx.x >> 5, lid = threadIdx.x & 31, gl = lid & 7, g = lid >> 3, d = p.d;
  const float* q = static_cast<const float*>(p.q);
  float4 qv[NR][CH], o[NR][CH];
  float m[NR], l[NR];
  int seen[NR], top = 0;
  long long grow[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const PaRow row = pa_row(p, it, it.row0 + r);
    const float* at = q + row.b * p.qsb + row.t * p.qst + row.h * p.qsh;
    seen[r] = row.ok ? min(row.seen - it.key_base, it.k1) : 0;
    top = max(top, seen[r]);
    grow[r] = row.ok ? row.grow : -1;
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = 4 * (gl + 8 * i);
      o[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      qv[r][i] = o[r][i];
      if (row.ok && c < d)
        qv[r][i] = make_float4(at[c] * p.scale_log2, at[c + 1] * p.scale_log2, at[c + 2] * p.scale_log2, at[c + 3] * p.scale_log2);
    }
  }
  const int k1 = min(it.k1, top);                      // no key past the last one that a row sees is read
  for (int k0 = it.k0 + warp * 8; k0 < k1; k0 += 32) {
    float4 k[2][CH], v[2][CH];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j = k0 + 4 * u + g;
      const long long at = j < k1 ? pa_key(p, it, j) : -1;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int c = 4 * (gl + 8 * i);
        k[u][i] = v[u][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (at >= 0 && c < d) {
          k[u][i] = *reinterpret_cast<const float4*>(static_cast<const float*>(p.kp) + at + c);
          v[u][i] = *reinterpret_cast<const float4*>(static_cast<const float*>(p.vp) + at + c);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
          s[u] = fmaf(qv[r][i].x, k[u][i].x, fmaf(qv[r][i].y, k[u][i].y, fmaf(qv[r][i].z, k[u][i].z, fmaf(qv[r][i].w, k[u][i].w, s[u]))));
      }
#pragma unroll
      for (int x = 1; x < 8; x <<= 1)
#pragma unroll
        for (int u = 0; u < 2; ++u) s[u] += __shfl_xor_sync(0xffffffffu, s[u], x);
#pragma unroll
      for (int u = 0; u < 2; ++u) s[u] = k0 + 4 * u + g < seen[r] ? s[u] : -INFINITY;
      const float mn = fmaxf(m[r], fmaxf(s[0], s[1])), ref = mn == -INFINITY ? 0.f : mn;   // (no key seen yet: weights 0)
      const float f = pa_ex2(m[r] - ref), p0 = pa_ex2(s[0] - ref), p1 = pa_ex2(s[1] - ref);
      m[r] = mn;
      l[r] = fmaf(l[r], f, p0 + p1);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        o[r][i].x = fmaf(p1, v[1][i].x, fmaf(p0, v[0][i].x, o[r][i].x * f));
        o[r][i].y = fmaf(p1, v[1][i].y, fmaf(p0, v[0][i].y, o[r][i].y * f));
        o[r][i].z = fmaf(p1, v[1][i].z, fmaf(p0, v[0][i].z, o[r][i].z * f));
        o[r][i].w = fmaf(p1, v[1][i].w, fmaf(p0, v[0][i].w, o[r][i].w * f));
      }
    }
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float mx = m[r];
#pragma unroll
    for (int x = 8; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float f = pa_ex2(m[r] - (mx == -INFINITY ? 0.f : mx));
    l[r] *= f;
#pragma unroll
    for (int x = 8; x < 32; x <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float4 y = make_float4(o[r][i].x * f, o[r][i].y * f, o[r][i].z * f, o[r][i].w * f);
#pragma unroll
      for (int x = 8; x < 32; x <<= 1) {
        y.x += __shfl_xor_sync(0xffffffffu, y.x, x); y.y += __shfl_xor_sync(0xffffffffu, y.y, x);
        y.z += __shfl_xor_sync(0xffffffffu, y.z, x); y.w += __shfl_xor_sync(0xffffffffu, y.w, x);
      }
      if (g == 0) *reinterpret_cast<float4*>(&s_o[warp][r][4 * (gl + 8 * i)]) = y;
    }
    if (lid == 0) s_ml[warp][r] = make_float2(mx, l[r]);
  }
  wait_previous();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (grow[r] < 0) continue;
    float mx = -INFINITY, sum = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, s_ml[w][r].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = pa_ex2(s_ml[w][r].x - (mx == -INFINITY ? 0.f : mx));
      sum = fmaf(f[w], s_ml[w][r].y, sum);
    }
    const long long part = (long long)it.slot * p.rows + grow[r];
    const int c = threadIdx.x;
    if (c == 0) p.part_ml[part] = make_float2(mx, sum);
    if (c < d) p.part_o[part * d + c] = fmaf(f[0], s_o[0][r][c], fmaf(f[1], s_o[1][r][c], fmaf(f[2], s_o[2][r][c], f[3] * s_o[3][r][c])));
  }
}

template <int CH>
static int launch_vec(const PaArgs& a, int rows, unsigned first, unsigned items, cudaStream_t s) {
  if (rows == 1) return launch_early(paged_attn_vec_kernel<CH, 1>, items, 1, kPvThreads, 0, s, a, first);
  if (rows == 2) return launch_early(paged_attn_vec_kernel<CH, 2>, items, 1, kPvThreads, 0, s, a, first);
  return launch_early(paged_attn_vec_kernel<CH, 4>, items, 1, kPvThreads, 0, s, a, first);
}

static int paged_attn_vec(const PaArgs& a, int rows, unsigned first, unsigned items, cudaStream_t s) {
  switch ((a.d + 31) / 32) {
    case 1: return launch_vec<1>(a, rows, first, items, s);
    case 2: return launch_vec<2>(a, rows, first, items, s);
    case 3: return launch_vec<3>(a, rows, first, items, s);
    default: return launch_vec<4>(a, rows, first, items, s);
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

// One row's P (d x d): 8 lanes a row of it (thread: row pr + 32 x, columns 4 (pq + 8 y) .. + 3).
template <int V>
HOA_DEVICE void load_path(const float* __restrict__ Pg, int d, int pr, int pq, float4 (&P)[4][4]) {
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

// out row g = P q, or 0 where no key was `seen` (an idle row's P may hold anything)
HOA_DEVICE void apply_path(const PaArgs& p, long long g, int pr, int pq, const float4 (&P)[4][4], const float4 (&q)[4], bool seen) {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      y = fmaf(P[x][k].x, q[k].x, fmaf(P[x][k].y, q[k].y, fmaf(P[x][k].z, q[k].z, fmaf(P[x][k].w, q[k].w, y))));
#pragma unroll
    for (int k = 1; k < 8; k <<= 1) y += __shfl_xor_sync(0xffffffffu, y, k);
    const int r = pr + 32 * x;
    if (pq == 0 && r < p.d) store_elem(p.out, g * p.d + r, p.out_dtype, seen ? y : 0.f);
  }
}

template <int V, int kWpr, bool kPaths>
__global__ void __launch_bounds__(kPjThreads) paged_attn_join_kernel(const __grid_constant__ PaArgs p) {
  static_assert(!kPaths || kWpr == 8, "P takes the whole CTA");
  __shared__ float4 s_o[8][32];
  __shared__ float s_l[8];
  const int d = p.d, slots = p.ns1 + p.ns2, warp = threadIdx.x >> 5, lid = threadIdx.x & 31;
  const int w = warp % kWpr;
  const long long g = (long long)blockIdx.x * (8 / kWpr) + warp / kWpr;
  if (p.leads) wait_previous();                        // (a call without items: nothing before it has waited for P)
  const bool ok = g < p.rows;                          // (uniform in the warps that share a row)
  float4 P[4][4];                                      // pass, chunk of 4 columns
  const int pr = threadIdx.x >> 3, pq = threadIdx.x & 7;
  if constexpr (kPaths) load_path<V>(p.paths + g * d * d, d, pr, pq, P);
  if (!p.leads) wait_previous();
  if (p.more) let_next_start();
  // a part without a key has l = 0; one that saw a score of NaN or +inf has l = NaN, which makes the row NaN
  float m = -INFINITY;
  if (ok)
    for (int s = lid; s < slots; s += 32) {
      const float2 ml = p.part_ml[s * p.rows + g];
      if (ml.y != 0.f) m = fmaxf(m, ml.y > 0.f ? ml.x : INFINITY);
    }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  if (ok && m != -INFINITY) {
#pragma unroll 4
    for (int s = w; s < slots; s += kWpr) {
      const float2 ml = p.part_ml[s * p.rows + g];
      const float f = ml.y != 0.f ? exp2f(ml.x - m) : 0.f;
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
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= inv;
  if (w == 0 && lid == 0) p.lse[g] = l != 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
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
    apply_path(p, g, pr, pq, P, q, l != 0.f);
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

// out = P o for many rows, o fp32 from the join: a stream of P alone, every load of a CTA's row at once and nothing to
// wait for but o.  Measured at 128 rows x 24 heads of 120 (177 MB of P): fused with the join 48 us, apart 6 + 33.
template <int V>
__global__ void __launch_bounds__(kPjThreads) paged_attn_transport_kernel(const __grid_constant__ PaArgs p) {
  const int d = p.d, pr = threadIdx.x >> 3, pq = threadIdx.x & 7;
  const long long g = blockIdx.x;
  float4 P[4][4];
  load_path<V>(p.paths + g * d * d, d, pr, pq, P);     // (the launches before let this one start after they had waited for P)
  wait_previous();
  const bool seen = p.lse[g] != -INFINITY;             // (by the join; NaN counts as seen)
  float4 q[4];
  const float* o = p.o + g * d;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const int c = 4 * (pq + 8 * y);
    q[y] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (V == 4) {
      if (c < d) q[y] = *reinterpret_cast<const float4*>(o + c);
    } else {
      if (c < d) q[y].x = o[c];
      if (c + 1 < d) q[y].y = o[c + 1];
      if (c + 2 < d) q[y].z = o[c + 2];
      if (c + 3 < d) q[y].w = o[c + 3];
    }
  }
  apply_path(p, g, pr, pq, P, q, seen);
}

template <int V, int kWpr, bool kPaths>
static int launch_join(const PaArgs& a, cudaStream_t s) {
  const long long blocks = (a.rows + 8 / kWpr - 1) / (8 / kWpr);
  if (blocks > 0x7fffffffll) return HOA_ERR_UNSUPPORTED;
  return launch_early(paged_attn_join_kernel<V, kWpr, kPaths>, (unsigned)blocks, 1, kPjThreads, 0, s, a);
}

static int join(const PaArgs& a, cudaStream_t s) {
  // 16-byte accesses: four columns a lane of o, the parts and P
  const bool v4 = a.d % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.paths) |
                                    reinterpret_cast<uintptr_t>(a.part_o)) & 15) == 0;
  if (a.paths) {
    if (a.rows < 8 * 148) return v4 ? launch_join<4, 8, true>(a, s) : launch_join<1, 8, true>(a, s);
    PaArgs j = a;                                      // the join writes o, fp32
    j.paths = nullptr;
    j.out = a.o;
    j.out_dtype = HOA_F32;
    j.more = 1;
    const int st = v4 ? launch_join<4, 1, false>(j, s) : launch_join<1, 1, false>(j, s);
    if (st != HOA_OK) return st;
    if (a.rows > 0x7fffffffll) return HOA_ERR_UNSUPPORTED;
    return launch_early(v4 ? paged_attn_transport_kernel<4> : paged_attn_transport_kernel<1>, (unsigned)a.rows, 1, kPjThreads, 0, s, a);
  }
  // eight warps a row where one a row would leave SMs without work and there are parts to share
  if (a.rows < 148 * 16 && a.ns1 + a.ns2 > 4) return v4 ? launch_join<4, 8, false>(a, s) : launch_join<1, 8, false>(a, s);
  return v4 ? launch_join<4, 1, false>(a, s) : launch_join<1, 1, false>(a, s);
}

}  // namespace hoa

using namespace hoa;

static bool pa_shape_ok(int B, int Tq, int H, int Hk, int d, int page, int n_shared, int W, int num_sms) {
  return B >= 1 && Tq >= 1 && Hk >= 1 && H >= Hk && H % Hk == 0 && d >= 1 && page >= 1 && n_shared >= 0 && W >= 0 &&
         num_sms >= 1;
}

static size_t pa_bytes(const PaPlan& pl, int B, int Tq, int H, int d) {
  // the parts (O, then m and l), and one token's o before its transport
  return ((size_t)pl.ns1 + pl.ns2) * B * Tq * H * (8 + 4 * (size_t)d) + (Tq == 1 ? 4 * (size_t)B * H * d : 0) + 256;
}

extern "C" size_t hoa_paged_attn_workspace_bytes(int B, int Tq, int H, int Hk, int d, int page, int n_shared, int W,
                                                 int num_sms) {
  if (!pa_shape_ok(B, Tq, H, Hk, d, page, n_shared, W, num_sms)) return 0;
  size_t most = 0;                                 // enough for whichever kernels take the call
  for (int k = 0; k < 4; ++k) {
    const size_t n = pa_bytes(pa_plan(B, Tq, H, Hk, d, page, n_shared, W, num_sms, k == 1, k > 1, k > 2), B, Tq, H, d);
    most = n > most ? n : most;
  }
  return most;
}

static int run_items(int kind, const PaArgs& a, long long first, long long items, cudaStream_t s) {
  if (items == 0) return HOA_OK;
  if (pa_is_tc(kind)) return paged_attn_tc(a, kind == kPaTc128, (unsigned)first, (unsigned)items, s);
  if (kind == kPaMma) return paged_attn_mma(a, (unsigned)first, (unsigned)items, s);
  if (kind < kPaSimt) return paged_attn_vec(a, pa_tile_rows(kind), (unsigned)first, (unsigned)items, s);
  return paged_attn_simt(a, pa_tile_rows(kind), (unsigned)first, (unsigned)items, s);
}

extern "C" int hoa_paged_attn_fwd(const void* q, const long long* q_strides, const void* k_pages, const void* v_pages,
                                  const long long* page_strides, int dtype, const int* shared, int n_shared,
                                  const int* table, long long table_stride, int W, const int* lens, const float* paths,
                                  void* out, int out_dtype, float* lse, float softmax_scale, int B, int Tq, int H, int Hk,
                                  int d, int page, int n_pages, int num_sms, void* workspace, size_t workspace_bytes,
                                  int* status, void* stream) {
  if (!q || !q_strides || !k_pages || !v_pages || !page_strides || !lens || !out || !lse || !workspace ||
      (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
      !pa_shape_ok(B, Tq, H, Hk, d, page, n_shared, W, num_sms) || n_pages < 1 || (n_shared > 0 && !shared) ||
      (W > 0 && !table) || (paths && Tq != 1))
    return HOA_ERR_INVALID_ARG;
  if ((dtype != HOA_F32 && dtype != HOA_BF16) || (out_dtype != HOA_F32 && out_dtype != HOA_BF16) || d > 128)
    return HOA_ERR_UNSUPPORTED;
  // key positions, row numbers (a tile past the last one included) and item numbers are ints
  if ((long long)(n_shared + (long long)W) * page > 0x7fff0000ll) return HOA_ERR_UNSUPPORTED;
  if ((long long)B * Tq > 0x7fff0000ll / H) return HOA_ERR_UNSUPPORTED;
  const int e = dtype == HOA_BF16 ? 2 : 4;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                         (uintptr_t)(page_strides[0] * e) | (uintptr_t)(page_strides[1] * e) | (uintptr_t)(page_strides[2] * e);
  const bool rows16 = (bits & 15) == 0;              // every token's row is 16-byte aligned
  const bool tensor = dtype == HOA_BF16 && d % 8 == 0 && rows16;
  const PaPlan pl = pa_plan(B, Tq, H, Hk, d, page, n_shared, W, num_sms, dtype == HOA_F32 && d % 4 == 0 && rows16, tensor,
                            tensor && softmax_scale > 0.f);
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
  a.leads = 1;
  a.part_o = static_cast<float*>(workspace);
  const size_t parts = (size_t)(pl.ns1 + pl.ns2) * a.rows * d;
  a.o = a.part_o + parts;
  // (m, l) pairs are read 8 bytes at a time: the floats before them rounded up to 16 bytes
  a.part_ml = reinterpret_cast<float2*>(a.part_o + ((parts + (Tq == 1 ? (size_t)a.rows * d : 0) + 3) & ~(size_t)3));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int st;
  if (pl.kind1 == pl.kind2) {                      // one launch for both parts
    st = run_items(pl.kind1, a, 0, items1 + items2, s);
  } else {
    st = run_items(pl.kind1, a, 0, items1, s);
    a.leads = items1 == 0;
    if (st == HOA_OK) st = run_items(pl.kind2, a, items1, items2, s);
  }
  if (st != HOA_OK) return st;
  a.leads = items1 + items2 == 0;
  return join(a, s);
}
