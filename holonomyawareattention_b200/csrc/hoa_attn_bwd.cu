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
// This file: the dispatch, D, and the form for fp32, every product in fp32 on the CUDA cores.
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

// 64 rows from `row0` of x (rows, d) -> registers, zero outside (kVec: d % 4 == 0, 16-byte boundaries) -> tile
template <int DA> struct AbRegs {
  static constexpr int N4 = DA / 4, K = kAbT * N4 / kAbThreads;      // float4s of a thread
  float4 v[K];
  template <bool kVec>
  HOA_DEVICE void load(const void* px, long long base, int row0, int rows, int d) {
    const float* x = reinterpret_cast<const float*>(px);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = threadIdx.x + k * kAbThreads, r = row0 + i / N4, e = i % N4 * 4;
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r >= rows || e >= d) continue;
      const long long at = base + (long long)r * d + e;
      if (kVec) {
        v[k] = *reinterpret_cast<const float4*>(x + at);
      } else {
        v[k].x = x[at];
        if (e + 1 < d) v[k].y = x[at + 1];
        if (e + 2 < d) v[k].z = x[at + 2];
        if (e + 3 < d) v[k].w = x[at + 3];
      }
    }
  }
  HOA_DEVICE void store(float* tile) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = threadIdx.x + k * kAbThreads;
      *reinterpret_cast<float4*>(tile + i / N4 * AbCfg<DA>::kLd + i % N4 * 4) = v[k];
    }
  }
};

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

// acc[a][c] += sum over k0 <= k < k1 of P[k][8 ty + a] Y[k][tx + 16 c]
template <int DA>
HOA_DEVICE void ab_tn(const float* P, const float* Y, int k0, int k1, int ty, int tx, float (&acc)[8][AbCfg<DA>::CPT]) {
  constexpr int kLd = AbCfg<DA>::kLd, CPT = AbCfg<DA>::CPT;
#pragma unroll 4
  for (int k = k0; k < k1; ++k) {
    const float4 p0 = *reinterpret_cast<const float4*>(P + k * kAbLdP + 8 * ty);
    const float4 p1 = *reinterpret_cast<const float4*>(P + k * kAbLdP + 8 * ty + 4);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const float y = Y[k * kLd + tx + 16 * c];
      acc[0][c] = fmaf(p0.x, y, acc[0][c]);
      acc[1][c] = fmaf(p0.y, y, acc[1][c]);
      acc[2][c] = fmaf(p0.z, y, acc[2][c]);
      acc[3][c] = fmaf(p0.w, y, acc[3][c]);
      acc[4][c] = fmaf(p1.x, y, acc[4][c]);
      acc[5][c] = fmaf(p1.y, y, acc[5][c]);
      acc[6][c] = fmaf(p1.z, y, acc[6][c]);
      acc[7][c] = fmaf(p1.w, y, acc[7][c]);
    }
  }
}

// kKeys: the CTA's own tile holds keys (outputs dk, dv), else queries (output dq).  The second products take half of the
// threads each, 8 rows a thread (4 rows a thread would ask more of shared memory than of the FMA pipes): dv and dk, or the
// two halves of the keys for dq.  The next tile of the other side is loaded while one is worked on (head dims up to 64;
// above, the registers do not hold it).
template <int DA, bool kKeys, bool kVec>
HOA_DEVICE void attn_bwd_simt(const AttnBwdArgs& p) {
  using C = AbCfg<DA>;
  constexpr int CPT = C::CPT;
  constexpr bool kAhead = DA <= 64;
  extern __shared__ __align__(16) float smem[];
  float* Q = smem;
  float* dO = Q + C::kTile;
  float* K = dO + C::kTile;
  float* V = K + C::kTile;
  float* P = V + C::kTile;           // P and dS: [query][key] for keys, [key][query] for queries
  float* dS = P + C::kP;
  float* lse = dS + C::kP;
  float* D = lse + kAbT;
  // a warp has 4 x 8 of the 16 x 16 threads of the first products: its 16-byte loads meet 4 and 8 different rows (2 and 16
  // with rows of 16 threads)
  const int tid = threadIdx.x, ty = tid / 64 * 4 + tid % 32 / 8, tx = tid % 64 / 32 * 8 + tid % 8;
  const int half = tid / 128, ty8 = tid % 128 / 16, tx16 = tid % 16;
  const int chain = blockIdx.x, d = p.d;                             // (all chains' longest walks first)
  const int nq = (p.Tq + kAbT - 1) / kAbT, nk = (p.Tk + kAbT - 1) / kAbT;
  const long long qbase = (long long)chain * p.Tq * d, kbase = (long long)chain * p.Tk * d;
  const int own = kKeys ? blockIdx.y : nq - 1 - blockIdx.y;
  if (own < 0 || own >= (kKeys ? nk : nq)) return;
  int first = 0, last = nq;
  if (kKeys) {
    first = max(0, (own * kAbT - p.q_offset) / kAbT);              // the first query tile that sees one of the keys
  } else {
    last = min((p.q_offset + own * kAbT + kAbT - 1) / kAbT, nk - 1) + 1;
  }
  AbRegs<DA> r0, r1;
  float stat = 0.f;                                                // threads 0-63: lse, 64-127: D, of the streamed queries
  auto load_keys = [&](int t) {
    r0.template load<kVec>(p.k, kbase, t * kAbT, p.Tk, d);
    r1.template load<kVec>(p.v, kbase, t * kAbT, p.Tk, d);
  };
  auto load_queries = [&](int t) {
    r0.template load<kVec>(p.q, qbase, t * kAbT, p.Tq, d);
    r1.template load<kVec>(p.dout, qbase, t * kAbT, p.Tq, d);
  };
  auto load_stats = [&](int t) {
    const int q = t * kAbT + (tid & 63);
    if (tid < 128) stat = q < p.Tq ? (tid < 64 ? p.lse : p.delta)[(long long)chain * p.Tq + q] : 0.f;
  };
  auto store_queries = [&]() {
    r0.store(Q);
    r1.store(dO);
    if (tid < 128) lse[tid] = stat;                                // (D lies behind lse)
  };
  auto store_keys = [&]() {
    r0.store(K);
    r1.store(V);
  };
  // The kernel before, which leaves D, starts when all before it has completed, so q, k, v, do and lse are there: they are
  // loaded while it runs (8 chains of 128, d = 48: 21.3 -> 20.5 us).
  if (kKeys) {
    load_keys(own);
    store_keys();
    if (first < last) load_queries(first);
    wait_previous();                                               // D
    if (first < last) load_stats(first);
  } else {
    load_queries(own);
    wait_previous();
    load_stats(own);
    store_queries();
    if (first < last) load_keys(first);
  }
  auto load = [&](int t) {
    if (kKeys) {
      load_queries(t);
      load_stats(t);
    } else {
      load_keys(t);
    }
  };

  float acc[8][CPT];
#pragma unroll
  for (int a = 0; a < 8; ++a)
#pragma unroll
    for (int c = 0; c < CPT; ++c) acc[a][c] = 0.f;

  for (int t = first; t < last; ++t) {
    if (!kAhead && t > first) load(t);
    if (kKeys) store_queries(); else store_keys();
    __syncthreads();
    if (kAhead && t + 1 < last) load(t + 1);
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
    if (kKeys) ab_tn<DA>(half ? dS : P, half ? Q : dO, 0, kAbT, ty8, tx16, acc);
    else ab_tn<DA>(dS, K, half * (kAbT / 2), (half + 1) * (kAbT / 2), ty8, tx16, acc);
    __syncthreads();
  }

  if (!kKeys) {                                                    // the second half's sums, through shared memory
    static_assert(C::kLd <= 2 * kAbLdP, "P and dS together hold 64 rows");
    float* X = P;
    if (half) {
#pragma unroll
      for (int a = 0; a < 8; ++a)
#pragma unroll
        for (int c = 0; c < CPT; ++c) X[(8 * ty8 + a) * C::kLd + tx16 + 16 * c] = acc[a][c];
    }
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
      for (int c = 0; c < CPT; ++c) acc[a][c] += X[(8 * ty8 + a) * C::kLd + tx16 + 16 * c];
  }
  const int rows = kKeys ? p.Tk : p.Tq;
  const long long base = kKeys ? kbase : qbase;
  const bool is_dv = kKeys && half == 0;
  float* out = reinterpret_cast<float*>(kKeys ? (is_dv ? p.dv : p.dk) : p.dq);
#pragma unroll
  for (int a = 0; a < 8; ++a) {
    const int r = own * kAbT + 8 * ty8 + a;
    if (r >= rows) continue;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int e = tx16 + 16 * c;
      if (e < d) out[base + (long long)r * d + e] = acc[a][c] * (is_dv ? 1.f : p.scale);
    }
  }
}

// Both sides in one launch (blockIdx.z): neither waits for the other, and few tiles leave SMs to both.
template <int DA, bool kVec>
__global__ void __launch_bounds__(kAbThreads, DA <= 64 ? 2 : 1) attn_bwd_simt_kernel(const __grid_constant__ AttnBwdArgs p) {
  if (blockIdx.z == 0) attn_bwd_simt<DA, true, kVec>(p);
  else attn_bwd_simt<DA, false, kVec>(p);
}

// D_i = do_i . o_i, 8 lanes a row; kVec: 8 elements a load (d % 8 == 0, 16-byte boundaries).
template <bool kVec>
__global__ void __launch_bounds__(256) attn_bwd_delta_kernel(AttnBwdArgs p, long long rows) {
  let_next_start();
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

template <int DA, bool kVec>
static int launch_sides(const AttnBwdArgs& a, int BH, cudaStream_t s) {
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(attn_bwd_simt_kernel<DA, kVec>, AbCfg<DA>::kSmem, done)) return HOA_ERR_LAUNCH;
  const int tiles = ceil_div(a.Tk, kAbT);                          // (Tq <= Tk)
  if (tiles > 65535) return HOA_ERR_UNSUPPORTED;
  return launch_early(attn_bwd_simt_kernel<DA, kVec>, dim3((unsigned)BH, (unsigned)tiles, 2), 1, kAbThreads, AbCfg<DA>::kSmem, s, a);
}

template <int DA>
static int launch_both(const AttnBwdArgs& a, int BH, cudaStream_t s) {
  uintptr_t at = 0;
  for (const void* x : {a.q, a.k, a.v, a.dout}) at |= reinterpret_cast<uintptr_t>(x);
  return a.d % 4 == 0 && (at & 15) == 0 ? launch_sides<DA, true>(a, BH, s) : launch_sides<DA, false>(a, BH, s);
}

}  // namespace hoa

using namespace hoa;

// D, and for bf16 rows that the tensor-core form takes through copies (`direct` 0) those
static size_t ab_bytes(int BH, int Tq, int Tk, int d, int dtype, bool direct, size_t* copies_at) {
  const size_t D = ((size_t)BH * Tq * sizeof(float) + 255) / 256 * 256;
  *copies_at = D;
  return D + (dtype == HOA_BF16 && !(direct && d % 8 == 0) ? attn_bwd_tc_bytes(BH, Tq, Tk, d) : 0);
}

extern "C" size_t hoa_attn_bwd_workspace_bytes(int BH, int Tq, int Tk, int d, int dtype, int aligned) {
  size_t at;
  return BH < 1 || Tq < 1 || Tk < 1 || d < 1 ? 0 : ab_bytes(BH, Tq, Tk, d, dtype, aligned != 0, &at);
}

extern "C" int hoa_attn_bwd(const void* qh, const void* kh, const void* vh, const float* o, const float* lse, const void* dout,
                            int dtype, void* dq, void* dk, void* dv, float softmax_scale, int BH, int Tq, int Tk, int q_offset,
                            int d, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  if (!qh || !kh || !vh || !o || !lse || !dout || !dq || !dk || !dv || !workspace || BH < 1 || Tq < 1 || Tk < 1 || d < 1)
    return HOA_ERR_INVALID_ARG;
  if (q_offset < 0 || (long long)q_offset + Tq > Tk) return HOA_ERR_INVALID_ARG;
  if (!(softmax_scale > 0.f && softmax_scale < INFINITY)) return HOA_ERR_INVALID_ARG;   // (masked scores are scale * -infinity)
  if ((dtype != HOA_F32 && dtype != HOA_BF16) || d > 128 || BH > 65535) return HOA_ERR_UNSUPPORTED;
  if (Tk > 0x7fffff00) return HOA_ERR_UNSUPPORTED;                   // (tile starts are counted with ints)
  uintptr_t at = 0;                                                  // TMA and the outputs' 16-byte stores
  for (const void* x : {qh, kh, vh, dout, (const void*)dq, (const void*)dk, (const void*)dv}) at |= reinterpret_cast<uintptr_t>(x);
  size_t copies_at;
  const size_t need = ab_bytes(BH, Tq, Tk, d, dtype, (at & 15) == 0, &copies_at);
  if (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return HOA_ERR_WORKSPACE;
  AttnBwdArgs a{qh, kh, vh, o, lse, dout, reinterpret_cast<float*>(workspace), dq, dk, dv, dtype, softmax_scale, Tq, Tk, q_offset, d,
                status, wait_bound_cycles()};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const long long rows = (long long)BH * Tq;
  if (rows > 32ll * 0x7fffffff) return HOA_ERR_UNSUPPORTED;
  const uintptr_t od = reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(dout);
  if (d % 8 == 0 && (od & 15) == 0) attn_bwd_delta_kernel<true><<<(unsigned)((rows + 31) / 32), 256, 0, s>>>(a, rows);
  else attn_bwd_delta_kernel<false><<<(unsigned)((rows + 31) / 32), 256, 0, s>>>(a, rows);
  if (int st = launch_status()) return st;
  if (dtype == HOA_BF16)
    return attn_bwd_tc(a, BH, need > copies_at ? reinterpret_cast<unsigned char*>(workspace) + copies_at : nullptr, s);
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
