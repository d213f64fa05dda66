// The path step: one generated token of every row (b, h).
//
//   P' = expm(skew(edge_scale a)) P          the edge from the row's last token to this one
//   q^ = P'^T q,  k^ = P'^T k,  v^ = P'^T v   k^ and v^ go to the row's page, slot lens[b] - 1
// (core/attention_fast_chunked.py:86-94 and :108-110 for one position.)  A row at
// its first token (lens 1) has no edge: P' = I.  A row without a token (lens 0)
// keeps P, gets q^ = 0 and writes nothing.
#include <type_traits>

#include "hoa_split_f16.cuh"

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
  long long max_wait;                                      // bound of a wait for a product, SM cycles (wait_bound_cycles())
};

HOA_DEVICE void st_fail(int* status) {
  if (status != nullptr) *reinterpret_cast<volatile int*>(status) = HOA_ERR_PAGES;
}

// ---------------------------------------------------------------------------
// One CTA of 256 threads per row (b, h), its products on tcgen05 with fp32
// accuracy: every factor x is split into x s = hi + lo, two f16 of 11 bits each (s a
// power of two that puts the factor's bound near 2^10), and a product is the three
// tensor-core products hi lo + lo hi + hi hi with fp32 accumulation (the small ones
// first: sums are cut off after each 16 columns); lo lo, 2^-22 of it, is left out.  f16 runs at twice the rate of tf32 and has its 11 bits; its
// short exponent is no loss, because the bounds are known: theta <= 0.6 after
// scaling, |P| <= 1.  (A itself is split at 16 A: entries up to 4094 fit, and what
// f16 drops of small ones, 2^-29, is below fp32's rounding of P'.)
//
//   P1  A2 = A A                                  scale 2^-s from ||A2||_1 >= ||A||_2^2
//   P2  A4 = A2 T,        T = x1 A + x2 A2
//   P3  E = E0 + L R,     L = x3 A2 + A4, R = x5 A + x6 A2 + x7 A4, E0 = A + y2 A2 + L  (s > 0: A added after L R)
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
// as the products.  TMEM: D, left hi and lo, 2 DP of the 512 columns, and 98 KB of
// shared memory at d = 120 (64 of them the right factor, 28 the next row's generators),
// so two CTAs run on an SM and one's products overlap the other's element work.
//
// Measured at 128 rows x 24 heads of 120 (446 MB, 42.7 GFLOP of fp32-accurate work): 266 us, 1.68 TB/s and 160 TFLOP/s,
// against 2.9 ms on the CUDA cores; 256 heads of 96: 20 us, one head's latency (22.8K cycles from its generators to its
// outputs).  The tensor pipe is busy 25%, the schedulers issue 48%: the rest is each CTA's chain of products (1.5K cycles
// each) and the element work between them (split, join, store: 2 to 5K).  More threads a row (384, 512) spill and are
// slower (283, 292 us), so are 8 columns a chunk (262) and a rolled loop over the products (292: a product takes the
// issuing lane about 95 cycles either way, but rolled they no longer follow one another closely).
// ---------------------------------------------------------------------------
using namespace sm100;

constexpr int kStGroups = 2, kStThreads = 128 * kStGroups;     // warpgroups: each has all 128 rows and every kStGroups-th chunk
constexpr float kSA = 16.f, kSA2 = 2048.f, kST = 16384.f, kSL = 4096.f, kSR = 4096.f, kSE = 512.f, kSP = 256.f;

template <int DP>
struct StLayout {
  static constexpr int NKB = (DP + 63) / 64, NC = DP / 16;
  static constexpr int kSlab = DP * 128;                 // bytes: DP rows of 64 f16
  static constexpr int kMat = NKB * kSlab;               // one f16 matrix
  static constexpr int kLd = DP + 4;                     // floats of a row of E P: rows of a warp on different banks
  static constexpr int kRight = 2 * kMat + (128 - DP) * 128;   // hi, lo; P1 reads 128 rows as its left factor
  static constexpr int kDim = DP < 120 ? DP : 120;       // the largest head dim
  static constexpr int kDelta = kDim * kLd * 4;
  static constexpr int kPart = kStThreads * 12 * 4;            // partial sums of q^, k^, v^, in place of E P
  static constexpr int kWork = kRight > kDelta ? kRight : kDelta;
  static constexpr int offGen = ((kWork > kPart ? kWork : kPart) + 127) / 128 * 128;   // the next row's generators
  static constexpr int kGen = (kDim * (kDim - 1) / 2 + kDim / 2) * 4;   // (either layout: banked has d / 2 unused slots)
  static constexpr int offVec = offGen + (kGen + 127) / 128 * 128;
  static constexpr int offSum = offVec + 3 * DP * 4;           // row sums, of each group
  static constexpr int offBar = offSum + kStThreads * 4;
  static constexpr int kAlloc = offBar + 32 + 1024;
  static constexpr uint32_t kCols = DP <= 16 ? 32 : DP <= 32 ? 64 : DP <= 64 ? 128 : 256;
  static constexpr uint32_t colD = 0, colHi = DP, colLo = DP + DP / 2;
};

// What a thread owns of the matrices: a row (= TMEM lane), and every kStGroups-th 16 columns.
template <int DP>
struct StUnit {
  using L = StLayout<DP>;
  uint8_t* sm;
  uint32_t tmem;           // + this warp's lanes
  int row, group;

  // 16 columns (chunk c) of this thread's row of the right factor
  HOA_DEVICE void put_right(int c, const F2 (&v)[8]) const {
    if (row >= DP) return;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint4 h, l;
      st_split2(v[4 * q], h.x, l.x);
      st_split2(v[4 * q + 1], h.y, l.y);
      st_split2(v[4 * q + 2], h.z, l.z);
      st_split2(v[4 * q + 3], h.w, l.w);
      const int ch = 2 * c + q;
      uint8_t* at = sm + (ch >> 3) * L::kSlab + sw128_offset(row, ch & 7);
      *reinterpret_cast<uint4*>(at) = h;
      *reinterpret_cast<uint4*>(at + L::kMat) = l;
    }
  }
  HOA_DEVICE void get_right(int c, F2 (&v)[8]) const {
    const int r = row < DP ? row : 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int ch = 2 * c + q;
      const uint8_t* at = sm + (ch >> 3) * L::kSlab + sw128_offset(r, ch & 7);
      const uint4 h = *reinterpret_cast<const uint4*>(at), l = *reinterpret_cast<const uint4*>(at + L::kMat);
      v[4 * q] = st_join2(h.x, l.x);
      v[4 * q + 1] = st_join2(h.y, l.y);
      v[4 * q + 2] = st_join2(h.z, l.z);
      v[4 * q + 3] = st_join2(h.w, l.w);
    }
  }
  // the same of the left factor (TMEM accesses are warp-collective: every lane calls these)
  HOA_DEVICE void put_left(int c, const F2 (&v)[8]) const {
    float h[8], l[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint32_t hi, lo;
      st_split2(v[e], hi, lo);
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
  HOA_DEVICE static void join_left(float (&h)[8], float (&l)[8], F2 (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = st_join2(__float_as_uint(h[e]), __float_as_uint(l[e]));
  }
};

HOA_DEVICE void cp_async(uint32_t dst, const float* src, bool wide) {
  if (wide) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

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
    const int a = pass == 1, b = pass == 0;                    // hi lo, lo hi, hi hi
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

// V: floats of a global access to P (4 where d % 4 == 0, else 1).
template <int DP, int V>
__global__ void __launch_bounds__(kStThreads, 2) path_step_kernel(const __grid_constant__ StepArgs p) {
  using L = StLayout<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* gen = reinterpret_cast<float*>(sm + L::offGen);
  float* vec = reinterpret_cast<float*>(sm + L::offVec);
  float* sum = reinterpret_cast<float*>(sm + L::offSum);
  uint64_t* done = reinterpret_cast<uint64_t*>(sm + L::offBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* delta = reinterpret_cast<float*>(sm);
  float* part = reinterpret_cast<float*>(sm);
  const int tid = threadIdx.x, warp = tid >> 5, lid = tid & 31;
  const int d = p.d, dd = d * d;
  if (tid == 0) {
    mbar_init(done, 1);
    *s_abort = 0;
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
  const StUnit<DP> un{sm, tmem + ((uint32_t)(warp & 3) << 21), (warp & 3) * 32 + lid, warp >> 2};
  const int row = un.row;
  uint32_t phase = 0;
  bool bad = false;

  // f(c, x) for this thread's chunks c, x the values there; the next chunk's are on their way meanwhile
  auto chunks = [&](auto load, auto f) {
    int c = un.group;
    if (c >= L::NC) return;
    auto x = load(c), y = x;
    tmem_wait_ld();
    x.touch();
#pragma unroll 1
    while (true) {
      const int n = c + kStGroups;
      if (n < L::NC) y = load(n);
      f(c, x);
      if (n >= L::NC) break;
      tmem_wait_ld();
      y.touch();
      x = y;
      c = n;
    }
  };
  struct Acc {
    float v[16];
    HOA_DEVICE void touch() { tmem_touch(v); }
  };
  struct AccLeft {
    float v[16], h[8], l[8];
    HOA_DEVICE void touch() { tmem_touch(v); tmem_touch(h); tmem_touch(l); }
  };
  auto load_acc = [&](int c) {
    Acc x;
    tmem_ld16(un.tmem + L::colD + 16 * c, x.v);
    return x;
  };
  auto load_left = [&](int c) {
    AccLeft x;
    tmem_ld16(un.tmem + L::colD + 16 * c, x.v);
    un.load_left(c, x.h, x.l);
    return x;
  };

  // V columns of P a thread, rows pr, pr + RG, ... (pn of them): a pass over P is contiguous
  const int n4 = d / V, RG = kStThreads / n4, pc = (tid % n4) * V, step = RG * d;
  int pr = tid / n4;
  const int pn = pr < RG && pr < d ? (d - pr + RG - 1) / RG : 0;
  constexpr int kRows = (DP + (kStThreads * V / DP) - 1) / (kStThreads * V / DP);
  using PV = typename std::conditional<V == 4, float4, float>::type;
  PV pv[kRows];
  auto load_P = [&](const float* P) {
    const float* at = P + pr * d + pc;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      pv[k] = PV{};
      if (k < pn) pv[k] = *reinterpret_cast<const PV*>(at);
      at += step;
    }
  };
  // P as the right factor; its pad rows and columns are zero already (every right factor's are)
  auto put_P = [&]() {
    asm volatile("" : "+r"(pr));
    uint8_t* slab = sm + (pc >> 6) * L::kSlab + (pc & 7) * 2;
    const uint32_t ch = (pc & 63) >> 3;
    int r = pr;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      uint8_t* at = slab + sw128_offset(r, ch);
      if constexpr (V == 4) {
        uint2 hi, lo;
        st_split2(f2_mul(f2(pv[k].x, pv[k].y), f2(kSP)), hi.x, lo.x);
        st_split2(f2_mul(f2(pv[k].z, pv[k].w), f2(kSP)), hi.y, lo.y);
        if (k < pn) {
          *reinterpret_cast<uint2*>(at) = hi;
          *reinterpret_cast<uint2*>(at + L::kMat) = lo;
        }
      } else {
        const float v = pv[k] * kSP;
        const __half hi = __float2half_rn(v), lo = __float2half_rn(v - __half2float(hi));
        if (k < pn) {
          *reinterpret_cast<__half*>(at) = hi;
          *reinterpret_cast<__half*>(at + L::kMat) = lo;
        }
      }
      r += RG;
    }
  };

  // shared-memory and TMEM writes of every thread -> the tensor core; thread 0 issues
  auto issue = [&](auto smem_left, bool accumulate) {
    tmem_wait_st();
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && !bad) {
      tc_fence_after();
      st_product<DP, decltype(smem_left)::value>(sm, tmem, accumulate, done);
    }
  };
  // A thread that has given up waits for no more products, and thread 0 issues none: the row's chain runs out on what is
  // there, without touching memory outside the CTA, and the CTA leaves before it stores the row.  (The clock is read
  // around the wait as well: a try may be suspended for longer than a short bound.)
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
  using Yes = std::true_type;
  using No = std::false_type;

  // a row's generators -> shared memory, one row ahead
  const bool wide = ((reinterpret_cast<uintptr_t>(p.a) | (uintptr_t)(p.stride * 4)) & 15) == 0;
  const int units = p.B * p.H;
  auto fetch = [&](int u) {
    if (u < units) {
      const float* g = p.a + (long long)u * p.stride;
      const uint32_t dst = smem_u32(gen);
      const int n = wide ? p.stride / 4 : p.stride;
      for (int i = tid; i < n; i += kStThreads) cp_async(dst + i * (wide ? 16 : 4), g + i * (wide ? 4 : 1), wide);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  wait_previous();
  fetch(blockIdx.x);

  // the token's vectors and its page, read one row ahead too
  constexpr int kQ = (3 * DP + kStThreads - 1) / kStThreads;
  float qv[kQ];
  int len = 0, id = -1;
  auto peek_len = [&](int u) { return u < units ? p.lens[u / p.H] : 0; };
  auto peek = [&](int u, int n) {
    if (n <= 0) return;
    const int b = u / p.H, h = u - b * p.H, pg = (n - 1) / p.page;
#pragma unroll
    for (int k = 0; k < kQ; ++k) {
      const int i = tid + k * kStThreads;
      qv[k] = i < 3 * d ? load_elem(p.qkv, b * p.qkv_stride + (long long)h * 3 * d + i, p.qkv_dtype) : 0.f;
    }
    id = pg < p.W ? p.table[b * p.tstride + pg] : -1;
  };
  len = peek_len(blockIdx.x);
  peek(blockIdx.x, len);

  for (int u = blockIdx.x, next = 0; u < units; u += gridDim.x, len = next) {
    const int h = u % p.H;
    next = peek_len(u + gridDim.x);
    const float* P = p.P + (long long)u * dd;
    float* Po = p.P_out + (long long)u * dd;
    if (len <= 0) {                                            // (block-uniform)
      for (int i = tid; i < dd; i += kStThreads) Po[i] = P[i];
      for (int i = tid; i < d; i += kStThreads) store_elem(p.qh, (long long)u * d + i, p.dtype, 0.f);
      asm volatile("cp.async.wait_all;" ::: "memory");
      fetch(u + gridDim.x);
      peek(u + gridDim.x, next);
      continue;
    }
    asm volatile("" : "+r"(pr));                               // (as the row's index math below)
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                           // the staged generators are in; the last row's sums were read
#pragma unroll
    for (int k = 0; k < kQ; ++k)
      if (tid + k * kStThreads < 3 * d) vec[tid + k * kStThreads] = qv[k];
    const int at_page = id;
    peek(u + gridDim.x, next);
    if (len > 1) {
      // ---- A, row by row: entry (r, c) is +-the generator of {r, c}
      if (p.a_bias) {
        const float* bias = p.a_bias + (long long)h * p.stride;
        for (int i = tid; i < p.stride; i += kStThreads) gen[i] += bias[i];
        __syncthreads();
      }
      // (0 in the pad)  y = 16 columns from c0 on, in units of 1 / kSA
      auto row_of_A = [&](int c0, F2 (&y)[8]) {
        int at = row;
        asm volatile("" : "+r"(at));                           // (its index math stays here: no registers across the products)
        gen_row16(gen, p.banked != 0, p.stride, d, at, lid, c0, p.edge_scale * kSA, y);
      };
      if ((row & ~31) < DP) {
#pragma unroll 1
        for (int c = un.group; c < L::NC; c += kStGroups) {
          F2 y[8];
          row_of_A(16 * c, y);
          un.put_right(c, y);
        }
      }
      // ---- P1: A2, and the scaling: ||A2||_1 (A2 is symmetric: row sums) bounds ||A||_2^2
      issue(Yes{}, false);
      wait();
      float rs = 0.f;
      chunks(load_acc, [&](int, Acc& x) {
#pragma unroll
        for (int e = 0; e < 16; ++e) rs += fabsf(x.v[e]);
      });
      sum[un.group * 128 + row] = rs;
      __syncthreads();
      float top = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = lid + 32 * x;
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < kStGroups; ++g) t += sum[g * 128 + r];
        if (r < d) top = fmaxf(top, t);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      float theta = sqrtf(top) * (1.f / kSA);
      int nsq = 0;
      while (theta > kStTheta && nsq < 64) { theta *= 0.5f; ++nsq; }
      const float sa = ldexpf(1.f / kSA, -nsq), sa2 = sa * sa;        // A = (hi + lo) sa, A2 = D sa2 once scaled
      // ---- P2: A4 = A2 T
      {
        const F2 ca = f2(kStX1 * kST * sa), ca2 = f2(kStX2 * kST / kSA2), cl = f2(kSA2 * sa2);
        chunks(load_acc, [&](int c, Acc& x) {
          F2 a[8], a2[8];
          un.get_right(c, a);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            a2[e] = f2_mul(f2(x.v[2 * e], x.v[2 * e + 1]), cl);
            a[e] = f2_fma(a[e], ca, f2_mul(a2[e], ca2));
          }
          un.put_left(c, a2);
          un.put_right(c, a);
        });
      }
      issue(No{}, false);
      wait();
      // ---- P3: E = E0 + L R, in units of 1 / (kSL kSR)
      auto p3 = [&](auto squares) {
        // with t = T kST, a = A2 kSA2, q = A4 kSA2 kST and A = (T - x2 A2) / x1:
        //   l = L kSL,  r = R kSR,  e = E0 kSL kSR
        const F2 la = f2(kStX3 * kSL / kSA2), lq = f2(kSL / (kSA2 * kST));
        const F2 rt = f2(kStX5 / kStX1 * kSR / kST), ra = f2((kStX6 - kStX5 * kStX2 / kStX1) * kSR / kSA2),
                 rq = f2(kStX7 * kSR / (kSA2 * kST));
        // The tensor core cuts its sums off (it does not round), 3 DP / 16 times over what stands in D before the product,
        // and each squaring doubles that: where there are squarings, A, most of E0, stays out of it and is added behind
        // the product.  Measured error of P', d = 72 and five squarings: 1.8e-6 with A in E0, 6.5e-7 without (fp32 all
        // through: 5.0e-7), for 14 us of 297 at 128 rows x 24 heads of 120.
        const F2 et = f2(squares ? 0.f : kSL * kSR / (kStX1 * kST)),
                 ea = f2((squares ? kStY2 : kStY2 - kStX2 / kStX1) * kSL * kSR / kSA2), el = f2(kSR);
        chunks(load_left, [&](int c, AccLeft& x) {
          F2 t[8], a2[8];
          un.get_right(c, t);
          un.join_left(x.h, x.l, a2);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const F2 q = f2(x.v[2 * e], x.v[2 * e + 1]);
            const F2 l = f2_fma(q, lq, f2_mul(a2[e], la));
            const float2 e0 = f2_get(f2_fma(l, el, squares ? f2_mul(a2[e], ea) : f2_fma(a2[e], ea, f2_mul(t[e], et))));
            t[e] = f2_fma(q, rq, f2_fma(a2[e], ra, f2_mul(t[e], rt)));
            a2[e] = l;
            x.v[2 * e] = e0.x;
            x.v[2 * e + 1] = e0.y;
          }
          un.put_left(c, a2);
          un.put_right(c, t);
          tmem_st16(un.tmem + L::colD + 16 * c, x.v);
        });
      };
      if (nsq > 0) p3(Yes{}); else p3(No{});
      issue(No{}, true);
      // ---- E, squared nsq times: (I + E)^2 = I + (2 E + E E)
      load_P(P);
      wait();
      if (nsq == 0) {
        put_P();
      } else {
#pragma unroll 1
        for (int c = (row & ~31) < DP ? un.group : L::NC; c < L::NC; c += kStGroups) {
          F2 y[8];
          row_of_A(16 * c, y);
          Acc x = load_acc(c);
          tmem_wait_ld();
          x.touch();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 v = f2_get(f2_fma(y[e], f2(kSL * kSR * sa), f2(x.v[2 * e], x.v[2 * e + 1])));
            x.v[2 * e] = v.x;
            x.v[2 * e + 1] = v.y;
          }
          tmem_st16(un.tmem + L::colD + 16 * c, x.v);
        }
        tmem_wait_st();
      }
      chunks(load_acc, [&](int c, Acc& x) {
        F2 e1[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) e1[e] = f2_mul(f2(x.v[2 * e], x.v[2 * e + 1]), f2(kSE / (kSL * kSR)));
        un.put_left(c, e1);
        if (nsq > 0) un.put_right(c, e1);
      });
#pragma unroll 1
      for (int s = 1; s <= nsq; ++s) {
        issue(No{}, false);
        wait();
        chunks(load_left, [&](int c, AccLeft& x) {
          F2 e1[8];
          un.join_left(x.h, x.l, e1);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            e1[e] = f2_fma(e1[e], f2(2.f), f2_mul(f2(x.v[2 * e], x.v[2 * e + 1]), f2(1.f / kSE)));
          un.put_left(c, e1);
          if (s < nsq) un.put_right(c, e1);
        });
      }
      if (nsq > 0) {
        load_P(P);
        put_P();
      }
      // ---- P4: E P
      issue(No{}, false);
      fetch(u + gridDim.x);                                    // (the staged row has been read)
      load_P(P);                                               // again, for P + E P (from L2)
      wait();
      chunks(load_acc, [&](int c, Acc& x) {
        if (row < d) {
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(delta + row * L::kLd + 16 * c + e) = make_float4(x.v[e], x.v[e + 1], x.v[e + 2], x.v[e + 3]);
        }
      });
    } else {
      fetch(u + gridDim.x);                                    // (P' = I: the staged row goes unused)
    }
    if (__syncthreads_or(bad)) break;
    asm volatile("" : "+r"(pr));
    // ---- P' = P + E P to global memory, and this thread's part of q^, k^, v^ = P'^T q, ...
    float y[3][V];
#pragma unroll
    for (int w = 0; w < 3; ++w)
#pragma unroll
      for (int e = 0; e < V; ++e) y[w][e] = 0.f;
    if (len <= 1) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) pv[k] = PV{};
    }
    {
      // four rows' shared-memory reads at a time; a row past the last one reads the last one and counts as zero
      constexpr int kB = 4;
      const float es = len > 1 ? 1.f / (kSE * kSP) : 0.f;
      float* op = Po + pr * d + pc;
#pragma unroll
      for (int k0 = 0; k0 < kRows; k0 += kB) {
        PV dv[kB];
        float q[kB][3];
#pragma unroll
        for (int k = 0; k < kB; ++k) {
          const int r = min(pr + (k0 + k) * RG, d - 1);
          dv[k] = *reinterpret_cast<const PV*>(delta + r * L::kLd + pc);
          q[k][0] = vec[r];
          q[k][1] = vec[d + r];
          q[k][2] = vec[2 * d + r];
        }
#pragma unroll
        for (int k = 0; k < kB; ++k) {
          if (k0 + k >= kRows) break;
          const bool in = k0 + k < pn;
          float x[V];
          if constexpr (V == 4) {
            x[0] = fmaf(dv[k].x, es, pv[k0 + k].x);
            x[1] = fmaf(dv[k].y, es, pv[k0 + k].y);
            x[2] = fmaf(dv[k].z, es, pv[k0 + k].z);
            x[3] = fmaf(dv[k].w, es, pv[k0 + k].w);
          } else {
            x[0] = fmaf(dv[k], es, pv[k0 + k]);
          }
          if (len <= 1)
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = pr + (k0 + k) * RG == pc + e ? 1.f : 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            x[e] = in ? x[e] : 0.f;
            y[0][e] = fmaf(x[e], q[k][0], y[0][e]);
            y[1][e] = fmaf(x[e], q[k][1], y[1][e]);
            y[2][e] = fmaf(x[e], q[k][2], y[2][e]);
          }
          if (in) {
            if constexpr (V == 4) *reinterpret_cast<float4*>(op) = make_float4(x[0], x[1], x[2], x[3]);
            else *op = x[0];
          }
          op += step;
        }
      }
    }
    __syncthreads();                                           // E P has been read
    if (pr < RG) {
#pragma unroll
      for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int e = 0; e < V; ++e) part[(pr * 3 + w) * d + pc + e] = y[w][e];
    }
    __syncthreads();
    for (int i = tid; i < 3 * d; i += kStThreads) {
      float t = 0.f;
      for (int g = 0; g < RG; ++g) t += part[g * 3 * d + i];
      const int w = i / d, c = i - w * d;
      if (w == 0) {
        store_elem(p.qh, (long long)u * d + c, p.dtype, t);
      } else if (at_page >= 0 && at_page < p.n_pages) {
        const long long at = at_page * p.ps + h * p.hs + (long long)((len - 1) % p.page) * p.ts + c;
        store_elem(w == 1 ? p.kp : p.vp, at, p.dtype, t);
      } else if (c == 0) {
        st_fail(p.status);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (tid == 0 && bad) mbar_wait(done, phase);                 // the product that it gave up on may still read shared memory
  if (__syncthreads_or(bad) && tid == 0 && p.status != nullptr) *reinterpret_cast<volatile int*>(p.status) = HOA_ERR_TIMEOUT;
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, L::kCols);
}

template <int DP, int V>
static int launch_step_v(const StepArgs& s, int num_sms, cudaStream_t stream) {
  using L = StLayout<DP>;
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(path_step_kernel<DP, V>, L::kAlloc, done)) return HOA_ERR_LAUNCH;
  const int units = s.B * s.H;
  return launch_early(path_step_kernel<DP, V>, (unsigned)(units < 2 * num_sms ? units : 2 * num_sms), 1, kStThreads, L::kAlloc, stream, s);
}

template <int DP>
static int launch_step(const StepArgs& s, int num_sms, cudaStream_t stream) {
  const bool v4 = s.d % 4 == 0 && ((reinterpret_cast<uintptr_t>(s.P) | reinterpret_cast<uintptr_t>(s.P_out)) & 15) == 0;
  return v4 ? launch_step_v<DP, 4>(s, num_sms, stream) : launch_step_v<DP, 1>(s, num_sms, stream);
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
      (dtype != HOA_F32 && dtype != HOA_BF16) || (long long)B * H > 0x7fff0000ll)   // (a CTA steps past the last unit by the grid)
    return HOA_ERR_UNSUPPORTED;
  StepArgs s{a, gen_is_banked(a_dtype) ? 1 : 0, stride, a_bias, edge_scale, P, P_out, qkv, qkv_dtype, qkv_stride, qh,
             k_pages, v_pages, dtype, page_strides[0], page_strides[1], page_strides[2], table, table_stride, lens,
             B, H, d, page, W, n_pages, status, wait_bound_cycles()};
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
