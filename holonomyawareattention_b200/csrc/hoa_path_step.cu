// The path step: one generated token of every row (b, h).
//
//   P' = expm(skew(edge_scale a)) P          the edge from the row's last token to this one
//   q^ = P'^T q,  k^ = P'^T k,  v^ = P'^T v   k^ and v^ go to the row's page, slot lens[b] - 1
// (core/attention_fast_chunked.py:86-94 and :108-110 for one position.)  A row at
// its first token (lens 1) has no edge: P' = I.  A row without a token (lens 0)
// keeps P, gets q^ = 0 and writes nothing.
#include <cuda_fp16.h>

#include <type_traits>

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

// ---------------------------------------------------------------------------
// One CTA of 256 threads per row (b, h), its products on tcgen05 with fp32
// accuracy: every factor x is split into x s = hi + lo, two f16 of 11 bits each (s a
// power of two that puts the factor's bound near 2^10), and a product is the three
// tensor-core products hi hi + hi lo + lo hi with fp32 accumulation; lo lo, 2^-22 of
// it, is left out.  f16 runs at twice the rate of tf32 and has its 11 bits; its
// short exponent is no loss, because the bounds are known: theta <= 0.6 after
// scaling, |P| <= 1.
//
//   P1  A2 = A A                                  scale 2^-s from ||A2||_1 >= ||A||_2^2
//   P2  A4 = A2 T,        T = x1 A + x2 A2
//   P3  E = E0 + L R,     L = x3 A2 + A4, R = x5 A + x6 A2 + x7 A4, E0 = A + y2 A2 + L
//   (s times  E <- 2 E + E E)
//   P4  P' = P + E P
// G = I + E: the identity stays out of every product, so that the accumulator's
// rounding scales with the small factor.
//
// A right factor lies row by row in shared memory (128-byte swizzled slabs of 64
// columns, the MN-major operand), a left factor in TMEM (lane = row); P1 takes both
// from shared memory, where the same slabs are also the K-major operand.  No matrix
// is kept in registers between products: a thread owns a row and every other 16
// columns, and reads A and A2 back from their own halves (A from T) - 2^-22 of them,
// as the products.  TMEM: D, left hi and lo, 2 DP of the 512 columns, and 64 KB of
// shared memory at d = 120, so two CTAs run on an SM and one's products overlap the
// other's element work.
// ---------------------------------------------------------------------------
using namespace sm100;

constexpr int kStThreads = 256;
constexpr float kSA2 = 2048.f, kST = 16384.f, kSL = 4096.f, kSR = 4096.f, kSE = 512.f, kSP = 256.f;

template <int DP>
struct StLayout {
  static constexpr int NKB = (DP + 63) / 64, NC = DP / 16;
  static constexpr int kSlab = DP * 128;                 // bytes: DP rows of 64 f16
  static constexpr int kMat = NKB * kSlab;               // one f16 matrix
  static constexpr int kLd = DP + 4;                     // floats of a row of E P: rows of a warp on different banks
  static constexpr int kRight = 2 * kMat + (128 - DP) * 128;   // hi, lo; P1 reads 128 rows as its left factor
  static constexpr int kDelta = DP * kLd * 4;
  static constexpr int offVec = ((kRight > kDelta ? kRight : kDelta) + 127) / 128 * 128;
  static constexpr int offSum = offVec + 3 * DP * 4;     // row sums (2 x 128), later the partial q^, k^, v^
  static constexpr int offMax = offSum + 3 * 128 * 4;
  static constexpr int offBar = offMax + 32;
  static constexpr int kAlloc = offBar + 32 + 1024;
  static constexpr uint32_t kCols = DP <= 16 ? 32 : DP <= 32 ? 64 : DP <= 64 ? 128 : 256;
  static constexpr uint32_t colD = 0, colHi = DP, colLo = DP + DP / 2;
};

HOA_DEVICE void st_split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

HOA_DEVICE float2 st_join2(uint32_t hi, uint32_t lo) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  return make_float2(h.x + l.x, h.y + l.y);
}

template <int DP>
struct StUnit {
  using L = StLayout<DP>;
  uint8_t* sm;
  uint32_t tmem;           // + this warp's lanes
  int row, half;           // the thread's row (= TMEM lane), which of every two 16-column chunks

  // 16 columns of chunk c of the right factor (this thread's row) / of the left factor
  HOA_DEVICE uint32_t* right(int part, int c, int q) const {   // q: which 8 columns
    const int ch = 2 * c + q;
    return reinterpret_cast<uint32_t*>(sm + part * L::kMat + (ch >> 3) * L::kSlab + sw128_offset(row, ch & 7));
  }
  HOA_DEVICE void put_right(int c, const float (&v)[16], float s) const {
    if (row >= DP) return;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint4 h, l;
      st_split2(v[8 * q] * s, v[8 * q + 1] * s, h.x, l.x);
      st_split2(v[8 * q + 2] * s, v[8 * q + 3] * s, h.y, l.y);
      st_split2(v[8 * q + 4] * s, v[8 * q + 5] * s, h.z, l.z);
      st_split2(v[8 * q + 6] * s, v[8 * q + 7] * s, h.w, l.w);
      *reinterpret_cast<uint4*>(right(0, c, q)) = h;
      *reinterpret_cast<uint4*>(right(1, c, q)) = l;
    }
  }
  HOA_DEVICE void get_right(int c, float (&v)[16], float s) const {   // s: 1 / the factor's scale
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int r = row < DP ? row : 0;
      const int ch = 2 * c + q;
      const uint8_t* at = sm + (ch >> 3) * L::kSlab + sw128_offset(r, ch & 7);
      const uint4 h = *reinterpret_cast<const uint4*>(at), l = *reinterpret_cast<const uint4*>(at + L::kMat);
      const uint32_t hh[4] = {h.x, h.y, h.z, h.w}, ll[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = st_join2(hh[e], ll[e]);
        v[8 * q + 2 * e] = f.x * s;
        v[8 * q + 2 * e + 1] = f.y * s;
      }
    }
  }
  // (TMEM accesses are warp-collective: every lane of the warp calls these)
  HOA_DEVICE void put_left(int c, const float (&v)[16], float s) const {
    float h[8], l[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t hi, lo;
      st_split2(v[2 * e] * s, v[2 * e + 1] * s, hi, lo);
      h[e] = __uint_as_float(hi);
      l[e] = __uint_as_float(lo);
    }
    tmem_st8(tmem + L::colHi + 8 * c, h);
    tmem_st8(tmem + L::colLo + 8 * c, l);
  }
  HOA_DEVICE void load_left(int c, float (&h)[8], float (&l)[8]) const {
    tmem_ld8(tmem + L::colHi + 8 * c, h);
    tmem_ld8(tmem + L::colLo + 8 * c, l);
  }
  HOA_DEVICE static void join_left(float (&h)[8], float (&l)[8], float (&v)[16], float s) {
    tmem_touch(h);
    tmem_touch(l);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 f = st_join2(__float_as_uint(h[e]), __float_as_uint(l[e]));
      v[2 * e] = f.x * s;
      v[2 * e + 1] = f.y * s;
    }
  }
};

// the three products of one fp32-accurate product, by one thread: D (+)= X Y
template <int DP, bool kSmemLeft>
HOA_DEVICE void st_product(uint8_t* sm, uint32_t tmem, bool accumulate, uint64_t* done) {
  using L = StLayout<DP>;
  constexpr uint32_t id = make_idesc(0, 128, DP, true);        // f16, right factor MN-major
  const uint32_t base = smem_u32(sm);
  const uint64_t r[2] = {desc_sw128_mn(base, L::kSlab), desc_sw128_mn(base + L::kMat, L::kSlab)};
  const uint64_t x[2] = {desc_sw128(base), desc_sw128(base + L::kMat)};
  const uint32_t t[2] = {tmem + L::colHi, tmem + L::colLo};
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int a = pass == 2, b = pass == 1;                    // hi hi, hi lo, lo hi
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const uint64_t rk = r[b] + (uint64_t)(k * 2048 >> 4);
      const uint32_t acc = accumulate || pass > 0 || k > 0 ? 1u : 0u;
      if (kSmemLeft) mma_bf16(tmem + L::colD, x[a] + (uint64_t)(((k >> 2) * L::kSlab + (k & 3) * 32) >> 4), rk, id, acc);
      else mma_bf16_ts(tmem + L::colD, t[a] + 8 * k, rk, id, acc);
    }
  }
  tc_commit(done);
}

template <int DP>
__global__ void __launch_bounds__(kStThreads, 2) path_step_kernel(const __grid_constant__ StepArgs p) {
  using L = StLayout<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* vec = reinterpret_cast<float*>(sm + L::offVec);
  float* sum = reinterpret_cast<float*>(sm + L::offSum);
  float* s_max = reinterpret_cast<float*>(sm + L::offMax);     // one per warp
  uint64_t* done = reinterpret_cast<uint64_t*>(sm + L::offBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  float* delta = reinterpret_cast<float*>(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lid = tid & 31;
  const int d = p.d, dd = d * d;
  if (tid == 0) {
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, L::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  StUnit<DP> un{sm, tmem + ((uint32_t)(warp & 3) << 21), (warp & 3) * 32 + lid, warp >> 2};
  const int row = un.row;
  uint32_t phase = 0;
  bool bad = false;
  constexpr int CH = (L::NC + 1) / 2;                          // 16-column chunks of a thread, at most

  // shared-memory and TMEM writes of every thread -> the tensor core; thread 0 issues; all wait
  auto product = [&](auto smem_left, bool accumulate) {
    tmem_wait_st();
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (tid == 0) {
      tc_fence_after();
      st_product<DP, decltype(smem_left)::value>(sm, tmem, accumulate, done);
    }
    bad |= !mbar_wait(done, phase);
    phase ^= 1;
    tc_fence_after();
  };
  using Yes = std::true_type;
  using No = std::false_type;

  const int units = p.B * p.H;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int b = u / p.H, h = u % p.H;
    const int len = p.lens[b];
    const float* P = p.P + (long long)u * dd;
    float* Po = p.P_out + (long long)u * dd;
    if (len <= 0) {                                            // (block-uniform)
      for (int i = tid; i < dd; i += kStThreads) Po[i] = P[i];
      for (int i = tid; i < d; i += kStThreads) store_elem(p.qh, (long long)u * d + i, p.dtype, 0.f);
      continue;
    }
    for (int i = tid; i < 3 * d; i += kStThreads)
      vec[i] = load_elem(p.qkv, b * p.qkv_stride + (long long)h * 3 * d + i, p.qkv_dtype);
    if (len > 1) {
      // ---- A: rows q and d-2-q of the strict upper triangle together have d entries; a warp takes
      // every eighth such pair, a lane every 32nd entry
      constexpr int QW = (DP / 2 + 7) / 8, EW = (DP + 31) / 32;
      float av[QW][EW];
      const float* g = p.a + (long long)u * p.stride;
      const float* bias = p.a_bias ? p.a_bias + (long long)h * p.stride : nullptr;
      const int nq = d / 2;                                    // pairs (the middle row alone when d is even)
      auto entry = [&](int x, int y, int& i, int& j) -> bool {
        const int q = warp + 8 * x, e = lid + 32 * y;
        const int first = d - 1 - q;
        i = e < first ? q : d - 2 - q;
        j = e < first ? q + 1 + e : i + 1 + (e - first);
        return q < nq && e < d && (e < first || i != q);
      };
      float mx = 0.f;
#pragma unroll
      for (int x = 0; x < QW; ++x)
#pragma unroll
        for (int y = 0; y < EW; ++y) {
          int i, j;
          av[x][y] = 0.f;
          if (entry(x, y, i, j)) {
            const int at = p.banked ? gen_banked_slot(i, j, d) : i * (2 * d - i - 1) / 2 + j - i - 1;
            av[x][y] = g[at];
            if (bias) av[x][y] += bias[at];
            av[x][y] *= p.edge_scale;
          }
          mx = fmaxf(mx, fabsf(av[x][y]));
        }
      for (int i = tid; i < (2 * L::kMat) / 16; i += kStThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (lid == 0) s_max[warp] = mx;
      __syncthreads();
      mx = s_max[0];
#pragma unroll
      for (int w = 1; w < 8; ++w) mx = fmaxf(mx, s_max[w]);
      // s = 2^(10 - exponent): entries of A s below 2^10
      int ex = 0;
      frexpf(mx, &ex);
      ex = mx > 0.f ? min(max(ex, -60), 60) : 0;
      const float sA = ldexpf(1.f, 10 - ex), iA = ldexpf(1.f, ex - 10);
#pragma unroll
      for (int x = 0; x < QW; ++x)
#pragma unroll
        for (int y = 0; y < EW; ++y) {
          int i, j;
          if (entry(x, y, i, j)) {
            const float v = av[x][y] * sA;
            const __half hi = __float2half_rn(v), lo = __float2half_rn(v - __half2float(hi));
            uint8_t* up = sm + (j >> 6) * L::kSlab + sw128_offset(i, (j & 63) >> 3) + (j & 7) * 2;
            uint8_t* dn = sm + (i >> 6) * L::kSlab + sw128_offset(j, (i & 63) >> 3) + (i & 7) * 2;
            *reinterpret_cast<__half*>(up) = hi;
            *reinterpret_cast<__half*>(up + L::kMat) = lo;
            *reinterpret_cast<__half*>(dn) = __hneg(hi);
            *reinterpret_cast<__half*>(dn + L::kMat) = __hneg(lo);
          }
        }
      // ---- P1: A2, and the scaling: ||A2||_1 (A2 is symmetric: row sums) bounds ||A||_2^2
      product(Yes{}, false);
      float rs = 0.f;
#pragma unroll
      for (int x = 0; x < CH; ++x) {
        const int c = 2 * x + un.half;
        if (c < L::NC) {
          float v[16];
          tmem_ld16(un.tmem + L::colD + 16 * c, v);
          tmem_wait_ld();
          tmem_touch(v);
#pragma unroll
          for (int e = 0; e < 16; ++e) rs += fabsf(v[e]);
        }
      }
      sum[un.half * 128 + row] = rs;
      __syncthreads();
      float top = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = lid + 32 * x;
        if (r < d) top = fmaxf(top, sum[r] + sum[128 + r]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float theta = sqrtf(top) * iA;
      int nsq = 0;
      while (theta > kStTheta && nsq < 64) { theta *= 0.5f; ++nsq; }
      const float sa = ldexpf(iA, -nsq), sa2 = sa * sa;        // A = (hi + lo) sa, A2 = D sa2 once scaled
      // ---- P2: A4 = A2 T
#pragma unroll
      for (int x = 0; x < CH; ++x) {
        const int c = 2 * x + un.half;
        if (c < L::NC) {
          float a[16], a2[16];
          tmem_ld16(un.tmem + L::colD + 16 * c, a2);
          un.get_right(c, a, sa);
          tmem_wait_ld();
          tmem_touch(a2);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            a2[e] *= sa2;
            a[e] = kStX1 * a[e] + kStX2 * a2[e];
          }
          un.put_left(c, a2, kSA2);
          un.put_right(c, a, kST);
        }
      }
      product(No{}, false);
      // ---- P3: E = E0 + L R
#pragma unroll
      for (int x = 0; x < CH; ++x) {
        const int c = 2 * x + un.half;
        if (c < L::NC) {
          float a4[16], t[16], a2[16], hh[8], ll[8];
          tmem_ld16(un.tmem + L::colD + 16 * c, a4);
          un.load_left(c, hh, ll);
          un.get_right(c, t, 1.f / kST);
          tmem_wait_ld();
          tmem_touch(a4);
          un.join_left(hh, ll, a2, 1.f / kSA2);
          float r[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float a = (t[e] - kStX2 * a2[e]) * (1.f / kStX1), q = a4[e] * (1.f / (kSA2 * kST));
            const float l = kStX3 * a2[e] + q;
            r[e] = kStX5 * a + kStX6 * a2[e] + kStX7 * q;
            a4[e] = l;
            t[e] = (a + kStY2 * a2[e] + l) * (kSL * kSR);
          }
          un.put_left(c, a4, kSL);
          un.put_right(c, r, kSR);
          tmem_st16(un.tmem + L::colD + 16 * c, t);
        }
      }
      product(No{}, true);
      // ---- E, squared nsq times: (I + E)^2 = I + (2 E + E E)
      for (int s = 0;; ++s) {
#pragma unroll
        for (int x = 0; x < CH; ++x) {
          const int c = 2 * x + un.half;
          if (c < L::NC) {
            float e1[16], e0[16], hh[8], ll[8];
            tmem_ld16(un.tmem + L::colD + 16 * c, e1);
            if (s > 0) un.load_left(c, hh, ll);
            tmem_wait_ld();
            tmem_touch(e1);
            if (s > 0) {
              un.join_left(hh, ll, e0, 2.f / kSE);
#pragma unroll
              for (int e = 0; e < 16; ++e) e1[e] = fmaf(e1[e], 1.f / (kSE * kSE), e0[e]);
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) e1[e] *= 1.f / (kSL * kSR);
            }
            un.put_left(c, e1, kSE);
            if (s < nsq) un.put_right(c, e1, kSE);
          }
        }
        if (s >= nsq) break;
        product(No{}, false);
      }
      // ---- P4: E P.  Pad rows and columns of the right factor are zero already.
      if (d % 4 == 0) {
        const int n4 = d / 4;
        for (int i = tid; i < dd / 4; i += kStThreads) {
          const int r = i / n4, c = (i % n4) * 4;
          const float4 v = reinterpret_cast<const float4*>(P)[i];
          uint2 hi, lo;
          st_split2(v.x * kSP, v.y * kSP, hi.x, lo.x);
          st_split2(v.z * kSP, v.w * kSP, hi.y, lo.y);
          uint8_t* at = sm + (c >> 6) * L::kSlab + sw128_offset(r, (c & 63) >> 3) + (c & 7) * 2;
          *reinterpret_cast<uint2*>(at) = hi;
          *reinterpret_cast<uint2*>(at + L::kMat) = lo;
        }
      } else {
        for (int i = tid; i < dd; i += kStThreads) {
          const int r = i / d, c = i % d;
          const float v = P[i] * kSP;
          const __half hi = __float2half_rn(v), lo = __float2half_rn(v - __half2float(hi));
          uint8_t* at = sm + (c >> 6) * L::kSlab + sw128_offset(r, (c & 63) >> 3) + (c & 7) * 2;
          *reinterpret_cast<__half*>(at) = hi;
          *reinterpret_cast<__half*>(at + L::kMat) = lo;
        }
      }
      product(No{}, false);
#pragma unroll
      for (int x = 0; x < CH; ++x) {
        const int c = 2 * x + un.half;
        if (c < L::NC) {
          float v[16];
          tmem_ld16(un.tmem + L::colD + 16 * c, v);
          tmem_wait_ld();
          tmem_touch(v);
          if (row < d) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<float4*>(delta + row * L::kLd + 16 * c + e) =
                  make_float4(v[e] * (1.f / (kSE * kSP)), v[e + 1] * (1.f / (kSE * kSP)), v[e + 2] * (1.f / (kSE * kSP)),
                              v[e + 3] * (1.f / (kSE * kSP)));
          }
        }
      }
    }
    if (__syncthreads_or(bad)) break;
    // ---- P' = P + E P, to global memory and in place of E P
    if (len > 1 && d % 4 == 0) {
      const int n4 = d / 4;
      for (int i = tid; i < dd / 4; i += kStThreads) {
        float4* at = reinterpret_cast<float4*>(delta + (i / n4) * L::kLd + (i % n4) * 4);
        const float4 v = reinterpret_cast<const float4*>(P)[i], e = *at;
        const float4 y = make_float4(v.x + e.x, v.y + e.y, v.z + e.z, v.w + e.w);
        reinterpret_cast<float4*>(Po)[i] = y;
        *at = y;
      }
    } else {
      for (int i = tid; i < dd; i += kStThreads) {
        const int r = i / d, c = i % d;
        const float y = len > 1 ? P[i] + delta[r * L::kLd + c] : (r == c ? 1.f : 0.f);
        Po[i] = y;
        delta[r * L::kLd + c] = y;
      }
    }
    __syncthreads();
    // ---- q^, k^, v^ = P'^T q, ...: a thread per column and half of the rows
    const int c = tid & 127, part = tid >> 7;
    float y0 = 0.f, y1 = 0.f, y2 = 0.f;
    if (c < d) {
#pragma unroll 4
      for (int r = part; r < d; r += 2) {
        const float x = delta[r * L::kLd + c];
        y0 = fmaf(x, vec[r], y0);
        y1 = fmaf(x, vec[d + r], y1);
        y2 = fmaf(x, vec[2 * d + r], y2);
      }
      if (part) { sum[c] = y0; sum[128 + c] = y1; sum[256 + c] = y2; }
    }
    __syncthreads();
    if (c < d && part == 0) {
      const int pos = len - 1, pg = pos / p.page;
      const int id = pg < p.W ? p.table[b * p.tstride + pg] : -1;
      store_elem(p.qh, (long long)u * d + c, p.dtype, y0 + sum[c]);
      if (id >= 0 && id < p.n_pages) {
        const long long at = id * p.ps + h * p.hs + (long long)(pos % p.page) * p.ts + c;
        store_elem(p.kp, at, p.dtype, y1 + sum[128 + c]);
        store_elem(p.vp, at, p.dtype, y2 + sum[256 + c]);
      } else if (c == 0) {
        st_fail(p.status);
      }
    }
    __syncthreads();                                           // the next row overwrites shared memory
  }
  if (__syncthreads_or(bad) && tid == 0 && p.status != nullptr) *reinterpret_cast<volatile int*>(p.status) = HOA_ERR_TIMEOUT;
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, L::kCols);
}

template <int DP>
static int launch_step(const StepArgs& s, int num_sms, cudaStream_t stream) {
  using L = StLayout<DP>;
  if (cudaFuncSetAttribute(path_step_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc) != cudaSuccess)
    return HOA_ERR_LAUNCH;
  const int units = s.B * s.H;
  path_step_kernel<DP><<<(unsigned)(units < 2 * num_sms ? units : 2 * num_sms), kStThreads, L::kAlloc, stream>>>(s);
  return launch_status();
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
  static const int num_sms = []() {                        // of the device that calls first: every GPU here is the same
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      n = 148;
    return n;
  }();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch ((d + 15) / 16) {
    case 1: return launch_step<16>(s, num_sms, st);
    case 2: return launch_step<32>(s, num_sms, st);
    case 3: return launch_step<48>(s, num_sms, st);
    case 4: return launch_step<64>(s, num_sms, st);
    case 5: return launch_step<80>(s, num_sms, st);
    case 6: return launch_step<96>(s, num_sms, st);
    case 7: return launch_step<112>(s, num_sms, st);
    case 8: return launch_step<128>(s, num_sms, st);
    default: return HOA_ERR_UNSUPPORTED;
  }
}
