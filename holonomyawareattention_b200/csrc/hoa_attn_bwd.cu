// Gradients of causal attention over the transported q^, k^, v^ (kernel (3)'s backward
// pass; the reference differentiates core/attention_fast_chunked.py:119-168 with autograd).
//
//   s_ij = scale q_i . k_j  (j <= q_offset + i),  p_ij = exp(s_ij - lse_i),  D_i = do_i . o_i
//   dv_j = sum_i p_ij do_i
//   ds_ij = p_ij (do_i . v_j - D_i),   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i
//
// The probabilities are recomputed from the forward's log-sum-exp.  Two kernels, one per
// output side: a CTA owns a tile of keys (dk, dv) or of queries (dq) and walks the tiles of
// the other side, so every sum has one owner and a fixed order, and no atomics; S and dP
// are computed twice (7 products instead of 5).
//
// This file: the dispatch, D, and the form with every product in fp32 on the CUDA cores
// (fp32 inputs, and bf16 ones whose head dim the tensor-core form does not take).
#include "hoa_attn_bwd.cuh"

namespace hoa {

constexpr int kAbT = 64, kAbThreads = 256;
constexpr int kAbLdP = kAbT + 4;

// Tiles are row-major with rows of DA + 4 floats: 8 lanes that read a float4 each of rows 16
// bytes apart modulo 128 (DA + 4 = 4 or 20 mod 32) hit 8 different bank groups.
template <int DA> struct AbCfg {
  static constexpr int kLd = DA + 4, CPT = DA / 16;
  static constexpr size_t kTile = (size_t)kAbT * kLd, kP = (size_t)kAbT * kAbLdP;
  static constexpr size_t kSmem = (4 * kTile + 2 * kP + 2 * kAbT) * sizeof(float);
};

// 64 rows from `row0` of x (rows, d) -> tile, zero outside
template <int DA>
HOA_DEVICE void ab_load(float* tile, const void* x, int dtype, long long base, int row0, int rows, int d) {
  for (int i = threadIdx.x; i < kAbT * DA; i += kAbThreads) {
    const int r = i / DA, e = i % DA;
    tile[r * AbCfg<DA>::kLd + e] = row0 + r < rows && e < d ? load_elem(x, base + (long long)(row0 + r) * d + e, dtype) : 0.f;
  }
}

// acc[a][b] = X[ty + 16 a] . Y[tx + 16 b]
template <int DA>
HOA_DEVICE void ab_nt(const float* X, const float* Y, int ty, int tx, float (&acc)[4][4]) {
  constexpr int kLd = AbCfg<DA>::kLd;
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] = 0.f;
#pragma unroll 2
  for (int e = 0; e < DA; e += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      x[a] = *reinterpret_cast<const float4*>(X + (ty + 16 * a) * kLd + e);
      y[a] = *reinterpret_cast<const float4*>(Y + (tx + 16 * a) * kLd + e);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        acc[a][b] = fmaf(x[a].x, y[b].x, acc[a][b]);
        acc[a][b] = fmaf(x[a].y, y[b].y, acc[a][b]);
        acc[a][b] = fmaf(x[a].z, y[b].z, acc[a][b]);
        acc[a][b] = fmaf(x[a].w, y[b].w, acc[a][b]);
      }
  }
}

// acc[a][c] += sum_k P[k][4 ty + a] Y[k][tx + 16 c]
template <int DA>
HOA_DEVICE void ab_tn(const float* P, const float* Y, int ty, int tx, float (&acc)[4][AbCfg<DA>::CPT]) {
  constexpr int kLd = AbCfg<DA>::kLd, CPT = AbCfg<DA>::CPT;
#pragma unroll 4
  for (int k = 0; k < kAbT; ++k) {
    const float4 p = *reinterpret_cast<const float4*>(P + k * kAbLdP + 4 * ty);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const float y = Y[k * kLd + tx + 16 * c];
      acc[0][c] = fmaf(p.x, y, acc[0][c]);
      acc[1][c] = fmaf(p.y, y, acc[1][c]);
      acc[2][c] = fmaf(p.z, y, acc[2][c]);
      acc[3][c] = fmaf(p.w, y, acc[3][c]);
    }
  }
}

// kKeys: the CTA's own tile holds keys (outputs dk, dv), else queries (output dq).
template <int DA, bool kKeys>
__global__ void __launch_bounds__(kAbThreads) attn_bwd_simt_kernel(AttnBwdArgs p) {
  using C = AbCfg<DA>;
  constexpr int CPT = C::CPT;
  extern __shared__ __align__(16) float smem[];
  float* Q = smem;
  float* dO = Q + C::kTile;
  float* K = dO + C::kTile;
  float* V = K + C::kTile;
  float* P = V + C::kTile;           // P and dS: [query][key] for keys, [key][query] for queries
  float* dS = P + C::kP;
  float* lse = dS + C::kP;
  float* D = lse + kAbT;
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int chain = blockIdx.x, d = p.d;                             // (all chains' longest walks first)
  const int nq = (p.Tq + kAbT - 1) / kAbT, nk = (p.Tk + kAbT - 1) / kAbT;
  const long long qbase = (long long)chain * p.Tq * d, kbase = (long long)chain * p.Tk * d;
  const int own = kKeys ? blockIdx.y : nq - 1 - blockIdx.y;
  int first = 0, last = nq;
  if (kKeys) {
    first = max(0, (own * kAbT - p.q_offset) / kAbT);              // the first query tile that sees one of the keys
  } else {
    last = min((p.q_offset + own * kAbT + kAbT - 1) / kAbT, nk - 1) + 1;
  }
  auto load_keys = [&](int t) {
    ab_load<DA>(K, p.k, p.dtype, kbase, t * kAbT, p.Tk, d);
    ab_load<DA>(V, p.v, p.dtype, kbase, t * kAbT, p.Tk, d);
  };
  auto load_queries = [&](int t) {
    ab_load<DA>(Q, p.q, p.dtype, qbase, t * kAbT, p.Tq, d);
    ab_load<DA>(dO, p.dout, p.dtype, qbase, t * kAbT, p.Tq, d);
    if (tid < kAbT) {
      const bool in = t * kAbT + tid < p.Tq;
      lse[tid] = in ? p.lse[(long long)chain * p.Tq + t * kAbT + tid] : 0.f;
      D[tid] = in ? p.delta[(long long)chain * p.Tq + t * kAbT + tid] : 0.f;
    }
  };
  if (kKeys) load_keys(own); else load_queries(own);

  float acc0[4][CPT], acc1[4][CPT];
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < CPT; ++c) acc0[a][c] = acc1[a][c] = 0.f;

  for (int t = first; t < last; ++t) {
    if (kKeys) load_queries(t); else load_keys(t);
    __syncthreads();
    const int q0 = (kKeys ? t : own) * kAbT, k0 = (kKeys ? own : t) * kAbT;
    float s[4][4], g[4][4];
    ab_nt<DA>(Q, K, ty, tx, s);
    ab_nt<DA>(dO, V, ty, tx, g);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int i = ty + 16 * a, j = tx + 16 * b;
        const bool see = k0 + j <= p.q_offset + q0 + i && q0 + i < p.Tq && k0 + j < p.Tk;
        const float pr = see ? expf(fmaf(s[a][b], p.scale, -lse[i])) : 0.f;
        const float ds = see ? pr * (g[a][b] - D[i]) : 0.f;
        if (kKeys) {
          P[i * kAbLdP + j] = pr;
          dS[i * kAbLdP + j] = ds;
        } else {
          dS[j * kAbLdP + i] = ds;
        }
      }
    __syncthreads();
    if (kKeys) {
      ab_tn<DA>(P, dO, ty, tx, acc0);
      ab_tn<DA>(dS, Q, ty, tx, acc1);
    } else {
      ab_tn<DA>(dS, K, ty, tx, acc1);
    }
    __syncthreads();
  }

  const int rows = kKeys ? p.Tk : p.Tq;
  const long long base = kKeys ? kbase : qbase;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const int r = own * kAbT + 4 * ty + a;
    if (r >= rows) continue;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int e = tx + 16 * c;
      if (e >= d) continue;
      const long long at = base + (long long)r * d + e;
      if (kKeys) store_elem(p.dv, at, p.dtype, acc0[a][c]);
      store_elem(kKeys ? p.dk : p.dq, at, p.dtype, acc1[a][c] * p.scale);
    }
  }
}

// D_i = do_i . o_i, 8 lanes a row; kVec: 8 elements a load (d % 8 == 0, 16-byte boundaries).
template <bool kVec>
__global__ void __launch_bounds__(256) attn_bwd_delta_kernel(AttnBwdArgs p, long long rows) {
  const long long r = (long long)blockIdx.x * 32 + threadIdx.x / 8;
  const int l = threadIdx.x & 7;
  float t = 0.f;
  if (r < rows) {
    if (kVec) {
      for (int e = 8 * l; e < p.d; e += 64) {
        float x[8];
        if (p.dtype == HOA_BF16) {
          const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.dout) + r * p.d + e);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[2 * k] = __uint_as_float(w[k] << 16);
            x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
          }
        } else {
          const float4* f = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.dout) + r * p.d + e);
          const float4 a = f[0], b = f[1];
          x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        }
        const float4* f = reinterpret_cast<const float4*>(p.o + r * p.d + e);
        const float4 a = f[0], b = f[1];
        t = fmaf(x[0], a.x, fmaf(x[1], a.y, fmaf(x[2], a.z, fmaf(x[3], a.w, t))));
        t = fmaf(x[4], b.x, fmaf(x[5], b.y, fmaf(x[6], b.z, fmaf(x[7], b.w, t))));
      }
    } else {
      for (int e = l; e < p.d; e += 8) t = fmaf(load_elem(p.dout, r * p.d + e, p.dtype), p.o[r * p.d + e], t);
    }
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (r < rows && l == 0) p.delta[r] = t;
}

template <int DA, bool kKeys>
static int launch_simt(const AttnBwdArgs& a, int BH, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(attn_bwd_simt_kernel<DA, kKeys>, AbCfg<DA>::kSmem, done)) return HOA_ERR_LAUNCH;
  const int tiles = ceil_div(kKeys ? a.Tk : a.Tq, kAbT);
  if (tiles > 65535) return HOA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)BH, (unsigned)tiles);
  attn_bwd_simt_kernel<DA, kKeys><<<grid, kAbThreads, AbCfg<DA>::kSmem, s>>>(a);
  return launch_status();
}

template <int DA>
static int launch_both(const AttnBwdArgs& a, int BH, cudaStream_t s) {
  const int st = launch_simt<DA, true>(a, BH, s);
  return st == HOA_OK ? launch_simt<DA, false>(a, BH, s) : st;
}

}  // namespace hoa

using namespace hoa;

extern "C" size_t hoa_attn_bwd_workspace_bytes(int BH, int Tq) {
  return BH < 1 || Tq < 1 ? 0 : (size_t)BH * Tq * sizeof(float);
}

extern "C" int hoa_attn_bwd(const void* qh, const void* kh, const void* vh, const float* o, const float* lse, const void* dout,
                            int dtype, void* dq, void* dk, void* dv, float softmax_scale, int BH, int Tq, int Tk, int q_offset,
                            int d, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  if (!qh || !kh || !vh || !o || !lse || !dout || !dq || !dk || !dv || !workspace || BH < 1 || Tq < 1 || Tk < 1 || d < 1)
    return HOA_ERR_INVALID_ARG;
  if (q_offset < 0 || (long long)q_offset + Tq > Tk) return HOA_ERR_INVALID_ARG;
  if ((dtype != HOA_F32 && dtype != HOA_BF16) || d > 128 || BH > 65535) return HOA_ERR_UNSUPPORTED;
  if (Tk > 0x7fffff00) return HOA_ERR_UNSUPPORTED;                   // (tile starts are counted with ints)
  if (workspace_bytes < hoa_attn_bwd_workspace_bytes(BH, Tq)) return HOA_ERR_WORKSPACE;
  AttnBwdArgs a{qh, kh, vh, o, lse, dout, reinterpret_cast<float*>(workspace), dq, dk, dv, dtype, softmax_scale, Tq, Tk, q_offset, d,
                status, wait_bound_cycles()};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const long long rows = (long long)BH * Tq;
  if (rows > 32ll * 0x7fffffff) return HOA_ERR_UNSUPPORTED;
  const uintptr_t od = reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(dout);
  if (d % 8 == 0 && (od & 15) == 0) attn_bwd_delta_kernel<true><<<(unsigned)((rows + 31) / 32), 256, 0, s>>>(a, rows);
  else attn_bwd_delta_kernel<false><<<(unsigned)((rows + 31) / 32), 256, 0, s>>>(a, rows);
  if (int st = launch_status()) return st;
  uintptr_t at = 0;                                                  // TMA and the outputs' 16-byte stores
  for (const void* x : {qh, kh, vh, dout, (const void*)dq, (const void*)dk, (const void*)dv}) at |= reinterpret_cast<uintptr_t>(x);
  if (dtype == HOA_BF16 && d % 8 == 0 && (at & 15) == 0) return attn_bwd_tc(a, BH, s);
  switch ((d + 15) / 16) {
    case 1: return launch_both<16>(a, BH, s);
    case 2: return launch_both<32>(a, BH, s);
    case 3: return launch_both<48>(a, BH, s);
    case 4: return launch_both<64>(a, BH, s);
    case 5: return launch_both<80>(a, BH, s);
    case 6: return launch_both<96>(a, BH, s);
    case 7: return launch_both<112>(a, BH, s);
    default: return launch_both<128>(a, BH, s);
  }
}
