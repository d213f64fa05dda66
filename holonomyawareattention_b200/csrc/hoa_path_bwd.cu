// Gradients through the path (the reference differentiates core/attention_fast_chunked.py:86-110
// and :171 with autograd): of the generators, and of q, k, v.
//
//   P_{t+1} = G_t P_t, G_t = expm(A_t), A_t = skew(edge_scale a_t)
//   q^ = P^T q, k^ = P^T k, v^ = P^T v, out = P o
//
// The gradient of P_s from its own uses has rank 4; with do^ = P^T dout,
//   P_s^T dP_s = q^ dq^T + k^ dk^T + v^ dv^T + do^ o^T      (vectors of position s).
// Every P is orthogonal, so seen from the first position the gradients of all later uses of
// G_t simply add up:  Z_t = sum_{s > t} skew(P_s^T dP_s), skew(X) = X - X^T, and
//   W_t = P_t Z_t P_t^T,   M_t = phi(ad_A) W_t,  phi(z) = (e^z - 1) / z,  ad_A X = A X - X A,
//   da_t[i, j] = edge_scale M_t[i, j] (i < j);   dq = P dq^, dk = P dk^, dv = P dv^
// (the derivative of expm at A is G times the integral of e^{-sA} . e^{sA} over s in [0, 1]).
// The closing edge t = T - 1 is on no path: its gradient is 0.
//
// P_t = R_t C_k as the forward left them.  The sums run in the chunk's frame, Y = C Z C^T,
// so that W = R Y R^T takes R alone.  Four kernels, over runs of 32 positions (of 8 in
// short sequences, which have few: 8 chains of 128, d = 48, take 71 us so and 84 in runs of 32):
//   sums    S_run = sum over the run of skew(X^T Y)               (one CTA a run)
//   suffix  S_run <- sum of all later runs                        (fp64, one thread an entry)
//   scan    Y_t for every position of a run, from its last one back (one CTA a run)
//   main    W, M, da, dq, dk, dv of every position                (tcgen05, below)
#include "hoa_split_f16.cuh"

namespace hoa {
using namespace sm100;

constexpr int kPbRun = 32, kPbRunMin = 8, kPbShort = 256;      // positions of a run, of one in sequences up to kPbShort

struct PathBwdArgs {
  const float* a; int banked, stride; const float* a_bias; float edge_scale;
  const float* R; const float* C; int chunk, K, rpc, NR;       // runs of a chunk, of a chain
  const void* x[3]; const float* o;                            // q^, k^, v^ (BH, T, d) in dtype, o in fp32
  const void* y[4];                                            // dq^, dk^, dv^, do^
  int dtype;
  float* da; void* dqkv; int out_dtype;
  int B, H, T, d;
  float* S;                                                    // (BH, NR, d, d)
  float* Y; float* F;                                          // of a group of runs: (runs, run, d, d), (runs, run, 3, d)
  float4* V;                                                   // two old iterates a CTA (main, large norms)
  long long run0; int runs, run, run_log;                      // the group, positions of a run
  int vec4;                                                    // rows of R, Y and the vectors from 16-byte (bf16: 8-byte) boundaries
  int* status;
  long long max_wait;
};

// chain, positions [t0, t1) and chunk of run r
struct PbRun { int chain, t0, t1, k; };
HOA_DEVICE PbRun pb_run(const PathBwdArgs& p, long long r) {
  PbRun x;
  x.chain = (int)(r / p.NR);
  const int i = (int)(r - (long long)x.chain * p.NR);
  x.k = i / p.rpc;
  x.t0 = x.k * p.chunk + (i - x.k * p.rpc) * p.run;
  x.t1 = min(min(x.t0 + p.run, (x.k + 1) * p.chunk), p.T);
  return x;
}

constexpr int kPsThreads = 256;

// The 8 vectors of `n` positions from t on -> rows 8 i + w of X (row stride ld, DP columns, zero past d):
// w = 0..3 q^, k^, v^, do^ and w = 4..7 dq^, dk^, dv^, o.  Rows past the n-th position are zero.
template <int DP>
HOA_DEVICE void pb_vectors(const PathBwdArgs& p, int chain, int t, int n, float* X, int ld) {
  static_assert(kPsThreads == 256, "a warp a vector");
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31, d = p.d;
  const void* src = w == 7 ? (const void*)p.o : w < 3 ? p.x[w] : w == 3 ? p.y[3] : p.y[w - 4];
  const bool f32 = w == 7 || p.dtype == HOA_F32;
  const long long at = ((long long)chain * p.T + t) * d;
  float* out = X + w * ld;
  if (p.vec4) {
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i >= n || 4 * l >= d) continue;
      if (f32) {
        v[i] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + at + i * d + 4 * l);
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(src) + at + i * d + 4 * l);
        v[i] = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                           __uint_as_float(u.y & 0xffff0000u));
      }
    }
    if (4 * l < DP)
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<float4*>(out + 8 * i * ld + 4 * l) = v[i];
  } else {
#pragma unroll
    for (int e = l; e < DP; e += 32)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        out[8 * i * ld + e] = i < n && e < d ? load_elem(src, at + i * d + e, f32 ? HOA_F32 : HOA_BF16) : 0.f;
  }
}

// A d x d matrix over the CTA's 8 warps: warp w has rows w DP / 8 + i, lane l columns l + 32 b, rows in pairs.
template <int DP> struct PbTile {
  static constexpr int NR = DP / 8, NB = (DP + 31) / 32;
  F2 v[NR / 2][NB];
};

// Y += skew of position i's vectors (rows 8 i .. of X)
template <int DP>
HOA_DEVICE void pb_add(const float* X, int ld, int i, PbTile<DP>& Y) {
  using T = PbTile<DP>;
  const int r0 = (threadIdx.x >> 5) * T::NR, l = threadIdx.x & 31;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float* x = X + (8 * i + w) * ld;
    const float* y = x + 4 * ld;
    F2 xc[T::NB], yc[T::NB];
#pragma unroll
    for (int b = 0; b < T::NB; ++b) {
      const int c = min(l + 32 * b, DP - 1);
      xc[b] = f2(-x[c]);
      yc[b] = f2(y[c]);
    }
#pragma unroll
    for (int a = 0; a < T::NR / 2; ++a) {
      const float2 xr = *reinterpret_cast<const float2*>(x + r0 + 2 * a), yr = *reinterpret_cast<const float2*>(y + r0 + 2 * a);
#pragma unroll
      for (int b = 0; b < T::NB; ++b) Y.v[a][b] = f2_fma(f2(xr.x, xr.y), yc[b], f2_fma(f2(yr.x, yr.y), xc[b], Y.v[a][b]));
    }
  }
}

template <int DP>
HOA_DEVICE void pb_store(const PbTile<DP>& Y, float* out, int d) {
  using T = PbTile<DP>;
  const int r0 = (threadIdx.x >> 5) * T::NR, l = threadIdx.x & 31;
#pragma unroll
  for (int a = 0; a < T::NR / 2; ++a)
#pragma unroll
    for (int b = 0; b < T::NB; ++b) {
      const float2 v = f2_get(Y.v[a][b]);
      const int r = r0 + 2 * a, c = l + 32 * b;
      if (c < d && r < d) out[r * d + c] = v.x;
      if (c < d && r + 1 < d) out[(r + 1) * d + c] = v.y;
    }
}

template <int DP>
__global__ void __launch_bounds__(kPsThreads) path_bwd_sums_kernel(const __grid_constant__ PathBwdArgs p) {
  __shared__ __align__(16) float X[64 * DP];
  const PbRun r = pb_run(p, blockIdx.x);
  PbTile<DP> Y;
#pragma unroll
  for (int a = 0; a < PbTile<DP>::NR / 2; ++a)
#pragma unroll
    for (int b = 0; b < PbTile<DP>::NB; ++b) Y.v[a][b] = f2(0.f);
  for (int t = r.t0; t < r.t1; t += 8) {
    const int n = min(8, r.t1 - t);
    __syncthreads();
    pb_vectors<DP>(p, r.chain, t, n, X, DP);
    __syncthreads();
    for (int i = 0; i < n; ++i) pb_add<DP>(X, DP, i, Y);
  }
  pb_store<DP>(Y, p.S + (long long)blockIdx.x * p.d * p.d, p.d);
}

// S_r <- sum of S_{r'} over the chain's later runs r' > r
__global__ void __launch_bounds__(256) path_bwd_suffix_kernel(const __grid_constant__ PathBwdArgs p, long long entries) {
  wait_previous();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= entries) return;
  const long long dd = (long long)p.d * p.d;
  const long long chain = i / dd;
  float* s = p.S + chain * p.NR * dd + (i - chain * dd);
  double acc = 0.0;
  int r = p.NR - 1;
  for (; r >= 15; r -= 16) {
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = s[(r - k) * dd];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      s[(r - k) * dd] = (float)acc;
      acc += v[k];
    }
  }
  for (; r >= 0; --r) {
    const float v = s[r * dd];
    s[r * dd] = (float)acc;
    acc += v;
  }
}

template <int DP> struct PbScan {
  static constexpr int kLd = DP + 4;
  static constexpr size_t kSmem = (size_t)(2 * DP + 64) * kLd * sizeof(float);
};

// out[ty + 16 a][tx + 16 b] = X[ty + 16 a] . Y[tx + 16 b] over DP columns, rows of kLd floats, once all have read X and Y
template <int DP, int NA>
HOA_DEVICE void pb_nt(const float* X, const float* Y, float* out) {
  constexpr int kLd = PbScan<DP>::kLd, NB = DP / 16;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  F2 acc[NA][NB];
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[a][b] = f2(0.f);
#pragma unroll 1
  for (int e = 0; e < DP; e += 4) {
    float4 x[NA];
#pragma unroll
    for (int a = 0; a < NA; ++a) x[a] = *reinterpret_cast<const float4*>(X + (ty + 16 * a) * kLd + e);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float4 y = *reinterpret_cast<const float4*>(Y + (tx + 16 * b) * kLd + e);
#pragma unroll
      for (int a = 0; a < NA; ++a)                                 // (even and odd columns in the two halves)
        acc[a][b] = f2_fma(f2(x[a].x, x[a].y), f2(y.x, y.y), f2_fma(f2(x[a].z, x[a].w), f2(y.z, y.w), acc[a][b]));
    }
  }
  __syncthreads();
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const float2 v = f2_get(acc[a][b]);
      out[(ty + 16 * a) * kLd + tx + 16 * b] = v.x + v.y;
    }
  __syncthreads();
}

template <int DP>
__global__ void __launch_bounds__(kPsThreads) path_bwd_scan_kernel(const __grid_constant__ PathBwdArgs p) {
  constexpr int kLd = PbScan<DP>::kLd;
  extern __shared__ __align__(16) float smem[];
  float* C = smem;
  float* Z = C + DP * kLd;
  float* X = Z + DP * kLd;
  const int tid = threadIdx.x, d = p.d;
  const long long run = p.run0 + blockIdx.x;
  const PbRun r = pb_run(p, run);
  wait_previous();
  if (r.t0 >= r.t1) return;
  const float* Cg = p.C + ((long long)r.chain * p.K + r.k) * d * d;
  const float* Zg = p.S + run * d * d;
  for (int i = tid; i < DP * DP; i += kPsThreads) {
    const int a = i / DP, b = i % DP;
    const bool in = a < d && b < d;
    C[a * kLd + b] = in ? Cg[a * d + b] : 0.f;
    Z[a * kLd + b] = in ? -Zg[a * d + b] : 0.f;            // Z^T = -Z
  }
  __syncthreads();
  pb_nt<DP, DP / 16>(C, Z, Z);                             // C Z
  pb_nt<DP, DP / 16>(Z, C, Z);                             // (C Z) C^T
  PbTile<DP> Y;
  {
    using T = PbTile<DP>;
    const int r0 = (tid >> 5) * T::NR, l = tid & 31;
#pragma unroll
    for (int a = 0; a < T::NR / 2; ++a)
#pragma unroll
      for (int b = 0; b < T::NB; ++b) {
        const int c = min(l + 32 * b, DP - 1);
        Y.v[a][b] = f2(Z[(r0 + 2 * a) * kLd + c], Z[(r0 + 2 * a + 1) * kLd + c]);
      }
  }
  for (int tb = r.t0 + (r.t1 - r.t0 - 1) / 8 * 8; tb >= r.t0; tb -= 8) {
    const int n = min(8, r.t1 - tb);
    __syncthreads();
    pb_vectors<DP>(p, r.chain, tb, n, X, kLd);
    __syncthreads();
    pb_nt<DP, 4>(X, C, X);                                 // the vectors in the chunk's frame
    float* F = p.F + ((long long)blockIdx.x * p.run + (tb - r.t0)) * 3 * d;
    for (int i = tid; i < n * 3 * d; i += kPsThreads) {
      const int e = i % d, w = i / d % 3, j = i / (3 * d);
      F[i] = X[(8 * j + 4 + w) * kLd + e];
    }
    for (int i = n - 1; i >= 0; --i) {
      pb_store<DP>(Y, p.Y + ((long long)blockIdx.x * p.run + (tb + i - r.t0)) * d * d, d);
      pb_add<DP>(X, kLd, i, Y);
    }
  }
}

// ---------------------------------------------------------------------------
// main: a CTA takes PP positions at a time, 128 / PP rows of its tiles each (head dims up to 32: 4,
// up to 64: 2, else 1), so that short rows fill the 128 lanes too.  Products on tcgen05 with fp32
// accuracy: each factor is two f16 parts (hoa_split_f16.cuh), a product three tensor-core
// products.  With |R| <= 1 and the entries of Y scaled below 2^10 (a power of two, per position),
// entries of W = R Y R^T, at most ||Y||_F <= 128 2^10, are taken 2^-4 times: no part leaves f16's range, as a
// commutator's Frobenius norm grows by less than 2.7 (below), so an entry stays below 2^13 2.7 < 65504;
// what f16 drops of small ones, 2^-25, is far below 2^-22 of the usual ones.
//
//   U = R Y          both from shared memory (R's slabs are the K-major left operand)
//   W = U R^T        U in TMEM; the same slabs, as the K-major right operand, are R^T
//   V_0 = W;  V_k = alpha_k [A, V_{k-1}] (+ V_{k-2}),  M = sum_k gamma_k V_k
// A is the left operand in TMEM for all k.  A and V are skew, so [A, V] = A V - (A V)^T: one
// product, transposed through shared memory.  M stays in registers (a thread owns a row and
// every G-th 16 columns).  The right factors of the PP positions lie side by side: the product of one's
// left rows with another's right columns is computed and not used.
//
// The sum: with x >= 2 ||A||_2 (from ||A||_inf and ||A||_F / sqrt 2),
//   x <= 4   Taylor: alpha_k = 1 / (k + 1), gamma = 1, ended once what is left, ||V_k||_F r / (1 - r) with r = x / (k + 2),
//            is below 2^-22 of ||W||_F, what the products are good for.
//   x > 4    Chebyshev (Taylor's terms would grow before they fall): alpha = 2 / x (1 / x first),
//            V_{k-2} added, gamma_k = (2 - [k = 0]) / x * integral of J_k over [0, x]
//            = (2 - [k = 0]) / x * 2 sum_m J_{k + 2m + 1}(x), the Bessel functions by Miller's
//            backward recurrence in fp64; about x + 15 products.  x <= kPbMaxX, else NaN.
//
// What bounds it: the chain of a position's dependent products and the element work between them
// (d = 96: 61.6K cycles with one CTA on the SM, 66K each with two; the schedulers issue 35-40%, the tensor pipe
// is busy 21%).  Two CTAs are what registers (128 a thread: M, a matrix being loaded and a chunk being
// split), 256 TMEM columns and 106 KB allow.  Measured, all four kernels: 65536 positions of 96 8.5 ms,
// 131072 of 48 6.2, 24000 of 120 6.15 (plain: 169, 49, 93).  Not kept: the next pass's matrices loaded ahead
// or the next chunk's TMEM loads (spills; 10.6 to 13 ms at d = 96), 3 or 4 warpgroups at 96 (10.3),
// products issued by a whole warp with uniform descriptors (its registers spill the rest: 13.8).
// ---------------------------------------------------------------------------
constexpr float kPbR = 256.f, kPbA = 16.f;
constexpr int kPbCoef = 640;
constexpr float kPbMaxX = 480.f;

template <int DP> struct PbLayout {
  static constexpr int RS = DP <= 32 ? 32 : DP <= 64 ? 64 : 128, PP = 128 / RS;    // rows of a position, positions
  static constexpr int G = DP <= 16 ? 1 : DP <= 32 ? 2 : DP <= 48 ? 3 : DP <= 96 ? 2 : 4;
  static constexpr int NT = 128 * G;
  static constexpr int NC = DP / 16, NCG = (NC + G - 1) / G;
  static constexpr int ND = PP > 1 ? 128 : DP;                     // columns of a product
  static constexpr int kDim = DP < 120 ? DP : 120;
  // R: rows of 64 columns a slab, all positions' rows stacked; hi, then lo
  static constexpr int kRowsR = PP > 1 ? 128 : DP;
  static constexpr int kSlabR = kRowsR * 128, kMatR = (DP + 63) / 64 * kSlabR, kTwoR = 2 * kMatR;
  // Y, V: DP rows of 64 columns a slab, the positions side by side
  static constexpr int kSlabV = DP * 128, kMatV = (ND + 63) / 64 * kSlabV, kTwoV = 2 * kMatV;
  static constexpr int kLdT = DP + 4;
  static constexpr int kT = (PP > 1 ? 128 : kDim) * kLdT * 4;      // A V, to be read transposed
  static constexpr int kR = ((kTwoR > kT ? kTwoR : kT) + 1023) / 1024 * 1024;
  static constexpr int offV = kR;
  // (R as the left factor is read as 128 rows a slab: past its own end into what follows)
  static constexpr int kMats = kR + kTwoV > kTwoR + 128 * 128 ? kR + kTwoV : kTwoR + 128 * 128;
  static constexpr int offVec = kMats;                             // dq^, dk^, dv^ in the chunk's frame
  static constexpr int offPart = offVec + PP * 3 * DP * 4;
  static constexpr int offRed = offPart + 3 * NT * 4;
  static constexpr int offPos = offRed + 2 * 32 * 4;               // of each position: top, norm bound, terms
  static constexpr int offCoef = offPos + 4 * 4 * 4;
  static constexpr int offBar = offCoef + PP * kPbCoef * 4;
  static constexpr int kAlloc = offBar + 64 + 1024;
  static constexpr int kMinBlocks = kAlloc <= 113 * 1024 ? 2 : 1;
  static constexpr uint32_t kCols = ND + DP <= 256 ? 256 : 512;
  static constexpr uint32_t colD = 0, colHi = ND, colLo = ND + DP / 2;
  static constexpr int kGen = (kDim * (kDim - 1) / 2 + kDim / 2 + NT - 1) / NT;
  static constexpr int kScratch = 2 * NCG * 4 * NT;                // float4s of a CTA's old iterates
  static_assert(NT <= 1024 && kPbRunMin % PP == 0, "a pass stays in its run");
};

// gamma_k (k >= 0) for x, and how many terms they need
HOA_DEVICE int pb_chebyshev(double x, float* coef) {
  // J_n by the recurrence J_{n-1} = 2 n / x J_n - J_{n+1} downwards from J_{N+1} = 0 and any small J_N; the first
  // pass finds what to divide by (J_0 + 2 (J_2 + J_4 + ...) = 1), the second one leaves the coefficients
  const double i2x = 2.0 / x;
  const int N = min(kPbCoef - 2, (int)(x + 40.0 + 8.0 * cbrt(x)));
  double start = 1e-100;
  int terms = 1;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    double j1 = 0.0, j0 = start, even = 0.0, odd = 0.0;              // sums of J_n, J_{n+2}, ... so far, by the parity of n
#pragma unroll 1
    for (int n = N; n >= 1; --n) {
      double& tail = n & 1 ? odd : even;
      tail += j0;
      if (pass == 1) {
        const float v = (float)(tail * (n == 1 ? 2.0 : 4.0) / x);
        coef[n - 1] = v;
        if (terms == 1 && fabsf(v) > 2e-9f) terms = max(1, n - 1);
      }
      const double j = n * i2x * j0 - j1;
      j1 = j0;
      j0 = j;
    }
    start /= j0 + 2.0 * even;
  }
  return terms;
}

template <int DP>
__global__ void __launch_bounds__(PbLayout<DP>::NT, PbLayout<DP>::kMinBlocks)
path_bwd_kernel(const __grid_constant__ PathBwdArgs p) {
  using L = PbLayout<DP>;
  constexpr int G = L::G, NT = L::NT, NCG = L::NCG, PP = L::PP, RS = L::RS, NW = NT / 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* gen = reinterpret_cast<float*>(sm);                        // R's place, once R is done with
  float* T = reinterpret_cast<float*>(sm);
  float* vec = reinterpret_cast<float*>(sm + L::offVec);
  float* part = reinterpret_cast<float*>(sm + L::offPart);
  float* red = reinterpret_cast<float*>(sm + L::offRed);           // [2][32]
  unsigned* s_top = reinterpret_cast<unsigned*>(sm + L::offPos);   // [4] the largest |Y|, as bits
  float* s_x = reinterpret_cast<float*>(sm + L::offPos) + 4;       // [4] x
  int* s_terms = reinterpret_cast<int*>(sm + L::offPos) + 8;       // [4] Chebyshev: products
  float* coef = reinterpret_cast<float*>(sm + L::offCoef);
  uint64_t* done = reinterpret_cast<uint64_t*>(sm + L::offBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lid = tid & 31;
  const int d = p.d;
  if (tid == 0) {
    mbar_init(done, 1);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (tid < 4) s_top[tid] = 0;
  if (warp == 0) {
    tmem_alloc(tmem_slot, L::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
  const int lrow = (warp & 3) * 32 + lid, group = warp >> 2;        // TMEM lane
  const int mine = (warp & 3) * 32 / RS, row0 = (warp & 3) * 32 - mine * RS, row = row0 + lid;   // position, row of its matrix
  const bool works = row0 < DP;                                     // (the warp has rows of a matrix)
  const uint32_t laneD = lanes + L::colD + (PP > 1 ? mine * RS : 0);
  uint32_t phase = 0;
  bool bad = false;

  // ---- the positions' matrices from global memory, DP / 4 threads a row, 4 columns each
  constexpr int n4 = DP / 4, RG = NT / n4, kRows = (PP * DP + RG - 1) / RG;
  const int pr = tid / n4, pc = (tid % n4) * 4;
  float4 pv[kRows];
  auto load_mat = [&](const float* m, int live) {                   // of `live` positions, d x d each
    int r0 = pr;
    asm volatile("" : "+r"(r0));
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int q = r0 + k * RG, w = PP > 1 ? q / DP : 0, r = q - w * DP;
      pv[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r0 >= RG || w >= live || r >= d || pc >= d) continue;
      const float* at = m + (w * d + r) * d + pc;
      if (p.vec4) {
        pv[k] = *reinterpret_cast<const float4*>(at);
      } else {
        pv[k].x = at[0];
        if (pc + 1 < d) pv[k].y = at[1];
        if (pc + 2 < d) pv[k].z = at[2];
        if (pc + 3 < d) pv[k].w = at[3];
      }
    }
  };
  auto put_half = [&](uint8_t* at, int mat, float4 v, float scale) {
    uint2 hi, lo;
    st_split2(f2_mul(f2(v.x, v.y), f2(scale)), hi.x, lo.x);
    st_split2(f2_mul(f2(v.z, v.w), f2(scale)), hi.y, lo.y);
    *reinterpret_cast<uint2*>(at) = hi;
    *reinterpret_cast<uint2*>(at + mat) = lo;
  };
  auto put_R = [&]() {
    int r0 = pr;
    asm volatile("" : "+r"(r0));
    uint8_t* slab = sm + (pc >> 6) * L::kSlabR + (pc & 7) * 2;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int q = r0 + k * RG, w = PP > 1 ? q / DP : 0, r = q - w * DP + w * RS;
      if (r0 >= RG || q >= PP * DP) continue;
      put_half(slab + sw128_offset(r, (pc & 63) >> 3), L::kMatR, pv[k], kPbR);
    }
  };
  auto put_Y = [&](const float* scales) {                           // a scale a position
    int r0 = pr;
    asm volatile("" : "+r"(r0));
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int q = r0 + k * RG, w = PP > 1 ? q / DP : 0, r = q - w * DP, c = pc + w * RS;
      if (r0 >= RG || q >= PP * DP) continue;
      put_half(sm + L::offV + (c >> 6) * L::kSlabV + (c & 7) * 2 + sw128_offset(r, (c & 63) >> 3), L::kMatV, pv[k], scales[w]);
    }
  };
  // ---- a thread's own 16 columns (chunk c) of its row
  auto put_right = [&](int c, const F2 (&v)[8]) {
    if (row >= DP) return;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint4 h, l;
      st_split2(v[4 * q], h.x, l.x);
      st_split2(v[4 * q + 1], h.y, l.y);
      st_split2(v[4 * q + 2], h.z, l.z);
      st_split2(v[4 * q + 3], h.w, l.w);
      const int ch = 2 * c + q + (PP > 1 ? mine * RS / 8 : 0);
      uint8_t* at = sm + L::offV + (ch >> 3) * L::kSlabV + sw128_offset(row, ch & 7);
      *reinterpret_cast<uint4*>(at) = h;
      *reinterpret_cast<uint4*>(at + L::kMatV) = l;
    }
  };
  auto put_left = [&](int c, const F2 (&v)[8]) {
    float h[8], l[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t hi, lo;
      st_split2(v[e], hi, lo);
      h[e] = __uint_as_float(hi);
      l[e] = __uint_as_float(lo);
    }
    tmem_st8(lanes + L::colHi + 8 * c, h);
    tmem_st8(lanes + L::colLo + 8 * c, l);
  };
  auto load_D = [&](int c, float (&v)[16]) {
    tmem_ld16(laneD + 16 * c, v);
    tmem_wait_ld();
    tmem_touch(v);
  };
  // this row's columns 16 c .. of a d x d matrix, times f; 0 outside
  auto mask_row = [&](int c, float f, const float (&v)[16], F2 (&x)[8]) {
    int n = row < d ? d - 16 * c : 0;
    asm volatile("" : "+r"(n));
    if (n >= 16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = f2_mul(f2(v[2 * e], v[2 * e + 1]), f2(f));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = f2(2 * e < n ? v[2 * e] * f : 0.f, 2 * e + 1 < n ? v[2 * e + 1] * f : 0.f);
    }
  };

  // ---- products.  Left R from shared memory or the left factor in TMEM; right: the slabs at V by rows, or R^T
  const uint32_t base = smem_u32(sm);
  const uint64_t rK[2] = {desc_sw128(base), desc_sw128(base + L::kMatR)};
  const uint64_t vN[2] = {desc_sw128_mn(base + L::offV, L::kSlabV), desc_sw128_mn(base + L::offV + L::kMatV, L::kSlabV)};
  constexpr uint32_t idN = make_idesc(0, 128, L::ND, true), idK = make_idesc(0, 128, L::ND, false);
  // hi_only: one of the three products alone, 2^-11 of the result off
  auto issue = [&](bool left_R, bool right_R, bool hi_only = false) {
    if (warp != 0 || !elect_one() || bad) return;
    tc_fence_after();
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int a = pass == 1, b = pass == 0;                       // hi lo, lo hi, hi hi
      if (pass < 2 && hi_only) continue;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint64_t kk = (uint64_t)(((k >> 2) * L::kSlabR + (k & 3) * 32) >> 4);
        const uint32_t acc = k > 0 || (pass == 1 || (pass == 2 && !hi_only)) ? 1u : 0u;
        const uint64_t rd = right_R ? rK[b] + kk : vN[b] + (uint64_t)(k * 2048 >> 4);
        if (left_R) mma_bf16(tmem + L::colD, rK[a] + kk, rd, idN, acc);
        else mma_bf16_ts(tmem + L::colD, tmem + (a ? L::colLo : L::colHi) + 8 * k, rd, right_R ? idK : idN, acc);
      }
    }
    tc_commit(done);
  };
  // what every thread wrote (shared memory, TMEM) -> the tensor core, after a barrier
  auto publish = [&]() {
    tmem_wait_st();
    fence_proxy_async_smem();
    tc_fence_before();
  };
  auto wait = [&]() {
    if (!bad) {
      const unsigned c0 = (unsigned)clock();
      bad = !mbar_wait_abortable(done, phase, s_abort, p.max_wait);
      if (!bad && (unsigned)clock() - c0 > (unsigned)p.max_wait) {
        bad = true;
        *s_abort = 1;
      }
      if (!bad) phase ^= 1;
    }
    tc_fence_after();
  };
  // the sum of the NW per-warp values in `at` that belong to position w
  auto sum_of = [&](const float* at, int w) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if ((i & 3) * 32 / RS == w) s += at[i];
    return s;
  };
  auto warp_sum = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };

  wait_previous();
  float4* scratch = p.V + (long long)blockIdx.x * L::kScratch + tid;
  constexpr int kLogPP = PP == 4 ? 2 : PP == 2 ? 1 : 0;
  const long long passes = ((long long)p.runs << p.run_log) / PP;
  for (long long u = blockIdx.x; u < passes; u += gridDim.x) {
    const long long lr = u >> (p.run_log - kLogPP);
    const PbRun r = pb_run(p, p.run0 + lr);
    const int t = r.t0 + (int)(u - (lr << (p.run_log - kLogPP))) * PP;
    if (t >= r.t1) continue;                                        // (block-uniform)
    const int live = min(PP, r.t1 - t);
    const int b = r.chain / p.H, h = r.chain - b * p.H;
    const long long pos = ((long long)b * p.T + t) * p.H + h;       // position w: pos + w H
    // ---- R and Y as factors
    load_mat(p.R + ((long long)r.chain * p.T + t) * d * d, live);
    put_R();
    load_mat(p.Y + u * PP * d * d, live);
    for (int i = tid; i < PP * 3 * DP; i += NT) {
      const int w = i / (3 * DP), e = i % DP;
      vec[i] = w < live && e < d ? p.F[((u * PP + w) * 3 + i / DP % 3) * d + e] : 0.f;
    }
    {
      unsigned top[PP];
#pragma unroll
      for (int w = 0; w < PP; ++w) top[w] = 0;
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int w = PP > 1 ? (pr + k * RG) / DP : 0;
        // (as bits: a NaN is above infinity)
        const unsigned v = max(max(__float_as_uint(fabsf(pv[k].x)), __float_as_uint(fabsf(pv[k].y))),
                               max(__float_as_uint(fabsf(pv[k].z)), __float_as_uint(fabsf(pv[k].w))));
#pragma unroll
        for (int i = 0; i < PP; ++i) top[i] = i == w ? max(top[i], v) : top[i];
      }
#pragma unroll
      for (int w = 0; w < PP; ++w) {
        const unsigned v = __reduce_max_sync(0xffffffffu, top[w]);
        if (lid == 0) atomicMax(&s_top[w], v);
      }
    }
    __syncthreads();
    bool lost = false;                                              // nothing finite can come of this thread's position
    int e_y = 0;
    {
      float scales[PP];
#pragma unroll
      for (int w = 0; w < PP; ++w) {
        const float top = __uint_as_float(s_top[w]);
        const bool fin = top <= 3.0e38f;
        const int e = fin && top > 0.f ? max(-100, min(100, 9 - ilogbf(top))) : 0;
        scales[w] = ldexpf(1.f, e);
        if (w == mine) {
          e_y = e;
          lost = !fin;
        }
      }
      put_Y(scales);
    }
    publish();
    __syncthreads();
    issue(true, false);                                             // U = R Y, in units of 2^-e_y / kPbR
    // ---- meanwhile: the generators on their way, and dq, dk, dv = R (.)
    float g[PP][L::kGen];
#pragma unroll
    for (int w = 0; w < PP; ++w) {
      const float* ag = p.a + (pos + (long long)w * p.H) * p.stride;
#pragma unroll
      for (int k = 0; k < L::kGen; ++k) {
        const int i = tid + k * NT;
        g[w][k] = i < p.stride && w < live ? ag[i] : 0.f;
        if (p.a_bias != nullptr && i < p.stride) g[w][k] += p.a_bias[(long long)h * p.stride + i];
      }
    }
    {
      float y[3] = {0.f, 0.f, 0.f};
      if (works) {
        const float* my = vec + mine * 3 * DP;
#pragma unroll 1
        for (int c = group; c < L::NC; c += G) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int ch = 2 * c + q;
            const uint8_t* at = sm + (ch >> 3) * L::kSlabR + sw128_offset(min(row, DP - 1) + mine * RS, ch & 7);
            const uint4 hi = *reinterpret_cast<const uint4*>(at), lo = *reinterpret_cast<const uint4*>(at + L::kMatR);
            const float2 m[4] = {f2_get(st_join2(hi.x, lo.x)), f2_get(st_join2(hi.y, lo.y)), f2_get(st_join2(hi.z, lo.z)),
                                 f2_get(st_join2(hi.w, lo.w))};
#pragma unroll
            for (int w = 0; w < 3; ++w)
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const float4 x = *reinterpret_cast<const float4*>(my + w * DP + 8 * ch + 2 * e);
                y[w] = fmaf(m[e].x, x.x, fmaf(m[e].y, x.y, fmaf(m[e + 1].x, x.z, fmaf(m[e + 1].y, x.w, y[w]))));
              }
          }
        }
      }
#pragma unroll
      for (int w = 0; w < 3; ++w) part[w * NT + group * 128 + lrow] = y[w];
    }
    wait();
    if (works) {
#pragma unroll 1
      for (int c = group; c < L::NC; c += G) {
        float v[16];
        F2 x[8];
        load_D(c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = f2_mul(f2(v[2 * e], v[2 * e + 1]), f2(1.f / (16.f * kPbR)));
        put_left(c, x);
      }
    }
    publish();
    __syncthreads();
    issue(false, true);                                             // W = U R^T, in units of 16 2^-e_y / kPbR
    if (tid < 4) s_top[tid] = 0;                                    // (read before the last barrier)
    for (int i = tid; i < live * 3 * d; i += NT) {
      const int q = i / d, e = i - q * d, pw = q / 3, w = q - 3 * pw;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < G; ++k) s += part[w * NT + k * 128 + pw * RS + e];
      store_elem(p.dqkv, (pos + (long long)pw * p.H) * 3 * d + w * d + e, p.out_dtype, s * (1.f / kPbR));
    }
    wait();
#pragma unroll
    for (int w = 0; w < PP; ++w)
#pragma unroll
      for (int k = 0; k < L::kGen; ++k)
        if (tid + k * NT < p.stride) gen[w * p.stride + tid + k * NT] = g[w][k];
    __syncthreads();
    // ---- V_0 = W as the right factor (units: 2^(4 - e_y)), A as the left one; the norms of W and of A
    F2 M[NCG][8];
    float rs = 0.f;
    {
      F2 sq = f2(0.f), sw = f2(0.f);
#pragma unroll
      for (int ci = 0; ci < NCG; ++ci) {
        const int c = group + ci * G;
        if (!works || c >= L::NC) continue;
        float v[16];
        load_D(c, v);
        mask_row(c, 1.f / kPbR, v, M[ci]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sw = f2_fma(M[ci][e], M[ci][e], sw);
        put_right(c, M[ci]);
      }
#pragma unroll 1
      for (int c = works ? group : L::NC; c < L::NC; c += G) {
        F2 x[8];
        int at = row;
        asm volatile("" : "+r"(at));                                // (its index math stays here: no registers across the products)
        gen_row16(gen + mine * p.stride, p.banked != 0, p.stride, d, at, lid, 16 * c, p.edge_scale * kPbA, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 a = f2_get(x[e]);
          rs += fabsf(a.x) + fabsf(a.y);
          sq = f2_fma(x[e], x[e], sq);
        }
        put_left(c, x);
      }
      part[group * 128 + lrow] = rs;
      const float2 a = f2_get(sq), w = f2_get(sw);
      const float ta = warp_sum(a.x + a.y), tw = warp_sum(w.x + w.y);
      if (lid == 0) {
        part[NT + warp] = ta;
        red[warp] = tw;
      }
    }
    publish();
    __syncthreads();
    issue(false, false);                                            // A V_0
    {
      float inf = 0.f;
#pragma unroll
      for (int q = 0; q < RS / 32; ++q) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < G; ++k) s += part[k * 128 + mine * RS + lid + 32 * q];
        if (lid + 32 * q < DP) inf = s <= 3.0e38f ? fmaxf(inf, s) : INFINITY;
      }
      inf = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(inf)));
      // (a bound: rounded up)
      const float x = 2.00002f / kPbA * fminf(inf, sqrtf(0.5f * sum_of(part + NT, mine)));
      lost |= !(x <= kPbMaxX);
      // one warp of each position leaves what all need to know; Taylor for what is lost, ended at once
      if (row0 == 0 && group == G - 1 && lid == 0) {
        s_x[mine] = lost ? 0.f : x;
        s_terms[mine] = !lost && x > 4.f ? pb_chebyshev((double)x, coef + mine * kPbCoef) : 0;
      }
    }
    // ---- the series
    float wq[PP];
#pragma unroll
    for (int w = 0; w < PP; ++w) wq[w] = sum_of(red, w);
    for (int k = 1;; ++k) {
      // (while the product runs) the norm above which another term is needed, of each position; Chebyshev: a number of terms
      // and the one below which the next product may do with its high parts: V_{k+1}, at most x / (k + 2) of V_k, is then
      // below 2^-12.5 of W, and 2^-11 sqrt 2 of it below 2^-23
      float need[PP], fine[PP];
      if (k > 1) {
#pragma unroll
        for (int w = 0; w < PP; ++w) {
          const float rr = s_x[w] / (float)(k + 2), left = rr / (1.f - rr);
          const bool cheb = s_terms[w] > 0;
          need[w] = cheb ? (k < s_terms[w] ? -1.f : INFINITY) : k >= 64 ? INFINITY : rr >= 1.f ? -1.f : 5.7e-14f * wq[w] / (left * left);
          fine[w] = cheb ? -1.f : 2.98e-8f * wq[w] / (rr * rr);
        }
      }
      wait();
#pragma unroll 1
      for (int c = works ? group : L::NC; c < L::NC; c += G) {
        float v[16];
        load_D(c, v);
        if (row < d)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(T + lrow * L::kLdT + 16 * c + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
      }
      __syncthreads();
      const int terms = s_terms[mine];
      const bool cheb = terms > 0;
      const float alpha = cheb ? (k == 1 ? 1.f / kPbA : 2.f / kPbA) / s_x[mine] : 1.f / (kPbA * (float)(k + 1));
      const float gamma = cheb ? (k <= terms ? coef[mine * kPbCoef + k] : 0.f) : 1.f;
      F2 vv = f2(0.f);
#pragma unroll
      for (int ci = 0; ci < NCG; ++ci) {
        const int c = group + ci * G;
        if (!works || c >= L::NC) continue;
        float v[16];
        F2 x[8];
        load_D(c, v);
        int at = (16 * c + mine * RS) * L::kLdT + row;
        asm volatile("" : "+r"(at));
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] -= T[at + e * L::kLdT];   // (rows past d: whatever lies there, masked below)
        mask_row(c, alpha, v, x);
        if (cheb) {
          float4* at4 = scratch + (long long)(((k & 1) * NCG + ci) * 4) * NT;
          if (k == 1) {
            float4* old = scratch + (long long)(ci * 4) * NT;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float2 lo = f2_get(M[ci][2 * q]), hi = f2_get(M[ci][2 * q + 1]);
              old[q * NT] = make_float4(lo.x, lo.y, hi.x, hi.y);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) M[ci][e] = f2_mul(M[ci][e], f2(coef[mine * kPbCoef]));
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float4 o = at4[q * NT];
              x[2 * q] = f2_add(x[2 * q], f2(o.x, o.y));
              x[2 * q + 1] = f2_add(x[2 * q + 1], f2(o.z, o.w));
            }
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 lo = f2_get(x[2 * q]), hi = f2_get(x[2 * q + 1]);
            at4[q * NT] = make_float4(lo.x, lo.y, hi.x, hi.y);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          M[ci][e] = f2_fma(x[e], f2(gamma), M[ci][e]);
          vv = f2_fma(x[e], x[e], vv);
        }
        put_right(c, x);
      }
      if (k > 1) {
        const float2 v = f2_get(vv);
        const float sum = warp_sum(v.x + v.y);
        if (lid == 0) red[(k & 1) * 32 + warp] = sum;
      }
      publish();
      __syncthreads();
      bool more = k == 1, hi_only = k > 1;                          // (the first check comes with the second term)
      if (k > 1)
#pragma unroll
        for (int w = 0; w < PP; ++w) {
          const float sum = sum_of(red + (k & 1) * 32, w);
          more |= sum > need[w];
          hi_only &= sum <= fine[w];
        }
      if (!more) break;
      issue(false, false, hi_only);
    }
    // ---- da: M by rows through shared memory, its upper triangle in the generators' layout to global memory
    {
      const float f = lost ? __int_as_float(0x7fffffff) : ldexpf(1.f, -e_y), es = 16.f * p.edge_scale;
#pragma unroll
      for (int ci = 0; ci < NCG; ++ci) {
        const int c = group + ci * G;
        if (!works || c >= L::NC || row >= d) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 lo = f2_get(f2_mul(M[ci][2 * q], f2(es))), hi = f2_get(f2_mul(M[ci][2 * q + 1], f2(es)));
          *reinterpret_cast<float4*>(T + lrow * L::kLdT + 16 * c + 4 * q) = make_float4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
        }
      }
    }
    if (__syncthreads_or(bad)) break;
#pragma unroll 1
    for (int w = 0; w < live; ++w) {
      float* dg = p.da + (pos + (long long)w * p.H) * p.stride;
      const float* Tw = T + w * RS * L::kLdT;
      if (t + w == p.T - 1) {                                       // the closing edge
        for (int i = tid; i < p.stride; i += NT) dg[i] = 0.f;
      } else if (p.banked) {
        // gen_banked_slot's lines of 32 slots: those of a pair of blocks, then 16 a diagonal block
        const int nb = d >> 5, off = nb * (nb - 1) / 2 * 32;
#pragma unroll 1
        for (int line = warp; line < off + 16 * nb; line += NW) {
          float v;
          if (line < off) {
            int pair = line >> 5, a = 0;
            while (pair >= nb - 1 - a) pair -= nb - 1 - a++;
            const int u0 = line & 31;
            v = Tw[(32 * a + u0) * L::kLdT + 32 * (a + 1 + pair) + (lid ^ (4 * (u0 & 7)))];
          } else {
            // slot (k, s): offsets u + v = s mod 32 with w = u - ceil(s / 2) = k + 1 - s mod 2; the one with u = v is unused
            const int o = (line - off) >> 4, k = (line - off) & 15, e = lid & 1;
            const int u0 = (k + 1 - e + ((lid + 1) >> 1)) & 31, v0 = (lid - u0) & 31;
            v = u0 == v0 ? 0.f : Tw[(32 * o + min(u0, v0)) * L::kLdT + 32 * o + max(u0, v0)];
          }
          dg[line * 32 + lid] = v;
        }
      } else {
        constexpr int NJ = (DP + 31) / 32;
#pragma unroll 2
        for (int i = warp; i < d - 1; i += NW) {
          float* o = dg + i * (2 * d - i - 1) / 2 - i - 1;
          float m[NJ];
#pragma unroll
          for (int k = 0; k < NJ; ++k) m[k] = Tw[i * L::kLdT + min(lid + 32 * k, DP - 1)];
#pragma unroll
          for (int k = 0; k < NJ; ++k)
            if (lid + 32 * k > i && lid + 32 * k < d) o[lid + 32 * k] = m[k];
        }
      }
    }
    __syncthreads();                                                // the next pass writes R there
  }
  if (tid == 0 && bad) mbar_wait(done, phase);                      // the product that it gave up on may still read shared memory
  if (__syncthreads_or(bad) && tid == 0 && p.status != nullptr) *reinterpret_cast<volatile int*>(p.status) = HOA_ERR_TIMEOUT;
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, L::kCols);
}

// ---------------------------------------------------------------------------
struct PbPlan {
  int rpc, K, NR, run_log;
  long long group;                                     // runs of one pass of scan and main
  size_t off_Y, off_F, off_V, bytes;
};

static int pb_sms() {
  static const int n = []() {                          // of the device that calls first: every GPU here is the same
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) v = 148;
    return v;
  }();
  return n;
}

// CTAs of the main kernel and float4s of their old iterates, by the padded head dim
template <int DP> static size_t pb_scratch(int sms) { return (size_t)sms * PbLayout<DP>::kMinBlocks * PbLayout<DP>::kScratch * sizeof(float4); }
static size_t pb_scratch_of(int d, int sms) {
  switch ((d + 15) / 16) {
    case 1: return pb_scratch<16>(sms);
    case 2: return pb_scratch<32>(sms);
    case 3: return pb_scratch<48>(sms);
    case 4: return pb_scratch<64>(sms);
    case 5: return pb_scratch<80>(sms);
    case 6: return pb_scratch<96>(sms);
    case 7: return pb_scratch<112>(sms);
    default: return pb_scratch<128>(sms);
  }
}

// The matrices Y of a pass take 1 GiB at most (4 d^2 bytes a position): longer inputs go through in several passes.
static bool pb_plan(int B, int H, int T, int d, int chunk, int sms, PbPlan& x) {
  if (B < 1 || H < 1 || T < 1 || d < 2 || d > 120 || chunk < 1 || sms < 1) return false;
  x.K = (int)(((long long)T + chunk - 1) / chunk);
  // (by the length alone: a sequence's gradients are the same bits in a batch of any size)
  const int run = T <= kPbShort ? kPbRunMin : kPbRun;
  x.run_log = T <= kPbShort ? 3 : 5;
  x.rpc = ((chunk < T ? chunk : T) + run - 1) / run;
  const long long NR = (long long)x.K * x.rpc, runs = NR * B * H;
  if ((long long)B * H > 0x7fffffff || NR > 0x7fffffff || runs > 0x7fffffff || (long long)T + chunk > 0x7fffff00) return false;
  x.NR = (int)NR;
  const size_t dd = (size_t)d * d * sizeof(float);
  x.group = (long long)((1ull << 30) / (dd * run));
  if (x.group < 1) x.group = 1;
  if (x.group > runs) x.group = runs;
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  x.off_Y = up((size_t)runs * dd);
  x.off_F = x.off_Y + up((size_t)x.group * run * dd);
  x.off_V = x.off_F + up((size_t)x.group * run * 3 * d * sizeof(float));
  x.bytes = x.off_V + pb_scratch_of(d, sms);
  return true;
}

template <int DP>
static int launch_path_bwd(PathBwdArgs a, const PbPlan& x, int sms, cudaStream_t s) {
  using L = PbLayout<DP>;
  static std::atomic<unsigned long long> done_scan{0}, done_main{0};
  if (!allow_smem(path_bwd_scan_kernel<DP>, PbScan<DP>::kSmem, done_scan) || !allow_smem(path_bwd_kernel<DP>, L::kAlloc, done_main))
    return HOA_ERR_LAUNCH;
  const long long runs = (long long)a.B * a.H * x.NR, entries = (long long)a.B * a.H * a.d * a.d;
  if ((entries + 255) / 256 > 0x7fffffff) return HOA_ERR_UNSUPPORTED;
  path_bwd_sums_kernel<DP><<<(unsigned)runs, kPsThreads, 0, s>>>(a);
  if (int st = launch_status()) return st;
  if (int st = launch_early(path_bwd_suffix_kernel, (unsigned)((entries + 255) / 256), 1, 256, 0, s, a, entries)) return st;
  for (long long r = 0; r < runs; r += x.group) {
    a.run0 = r;
    a.runs = (int)(runs - r < x.group ? runs - r : x.group);
    if (int st = launch_early(path_bwd_scan_kernel<DP>, (unsigned)a.runs, 1, kPsThreads, PbScan<DP>::kSmem, s, a)) return st;
    const long long passes = ((long long)a.runs << x.run_log) / L::PP, most = (long long)sms * L::kMinBlocks;
    if (int st = launch_early(path_bwd_kernel<DP>, (unsigned)(passes < most ? passes : most), 1, L::NT, L::kAlloc, s, a)) return st;
  }
  return HOA_OK;
}

}  // namespace hoa

using namespace hoa;

extern "C" size_t hoa_path_bwd_workspace_bytes(int B, int H, int T, int d, int chunk) {
  PbPlan x;
  return pb_plan(B, H, T, d, chunk, pb_sms(), x) ? x.bytes : 0;
}

extern "C" int hoa_path_bwd(const float* a_all, int a_dtype, const float* a_bias, float edge_scale, const float* R, const float* C,
                            int chunk, const void* qh, const void* kh, const void* vh, const float* o, const void* dqh,
                            const void* dkh, const void* dvh, const void* doh, int hat_dtype, float* da, void* dqkv, int out_dtype,
                            int B, int H, int T, int d, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  if (!a_all || !R || !C || !qh || !kh || !vh || !o || !dqh || !dkh || !dvh || !doh || !da || !dqkv || !workspace)
    return HOA_ERR_INVALID_ARG;
  if (B < 1 || H < 1 || T < 1 || d < 2 || chunk < 1) return HOA_ERR_INVALID_ARG;
  const int stride = gen_row_stride(a_dtype, d);
  if (d > 120 || stride == 0 || gen_elem_dtype(a_dtype) != HOA_F32 || (hat_dtype != HOA_F32 && hat_dtype != HOA_BF16) ||
      (out_dtype != HOA_F32 && out_dtype != HOA_BF16))
    return HOA_ERR_UNSUPPORTED;
  const int sms = pb_sms();
  PbPlan x;
  if (!pb_plan(B, H, T, d, chunk, sms, x)) return HOA_ERR_UNSUPPORTED;
  if (workspace_bytes < x.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return HOA_ERR_WORKSPACE;
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  uintptr_t at = reinterpret_cast<uintptr_t>(R);
  for (const void* v : {qh, kh, vh, (const void*)o, dqh, dkh, dvh, doh}) at |= reinterpret_cast<uintptr_t>(v);
  const int vec4 = d % 4 == 0 && (at & 15) == 0;
  PathBwdArgs p{a_all, gen_is_banked(a_dtype) ? 1 : 0, stride, a_bias, edge_scale, R, C, chunk, x.K, x.rpc, x.NR,
                {qh, kh, vh}, o, {dqh, dkh, dvh, doh}, hat_dtype, da, dqkv, out_dtype, B, H, T, d,
                reinterpret_cast<float*>(ws), reinterpret_cast<float*>(ws + x.off_Y), reinterpret_cast<float*>(ws + x.off_F),
                reinterpret_cast<float4*>(ws + x.off_V), 0, 0, 1 << x.run_log, x.run_log, vec4, status, wait_bound_cycles()};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch ((d + 15) / 16) {
    case 1: return launch_path_bwd<16>(p, x, sms, s);
    case 2: return launch_path_bwd<32>(p, x, sms, s);
    case 3: return launch_path_bwd<48>(p, x, sms, s);
    case 4: return launch_path_bwd<64>(p, x, sms, s);
    case 5: return launch_path_bwd<80>(p, x, sms, s);
    case 6: return launch_path_bwd<96>(p, x, sms, s);
    case 7: return launch_path_bwd<112>(p, x, sms, s);
    default: return launch_path_bwd<128>(p, x, sms, s);
  }
}
