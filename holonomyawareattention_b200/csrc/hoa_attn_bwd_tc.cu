// Gradients of causal attention, bf16 form on tcgen05 / TMEM (formulas: hoa_attn_bwd.cu).
//
// One kernel in two roles.  A CTA owns 128 rows of one side - keys (outputs dk, dv) or
// queries (output dq) - and streams 64-row tiles of the other side:
//
//              own X0, X1   stream Y0, Y1   S = X0 Y0^T   G = X1 Y1^T    accumulators in TMEM
//   keys       K, V         Q, dO           S^T           dP^T           dV += P^T dO,  dK += dS^T Q
//   queries    Q, dO        K, V            S             dP                            dQ += dS K
//
// so a row of the CTA's matrices is a TMEM lane and a thread throughout, P and dS go back over S
// and G in two bf16 parts each (the left operands of the second products, from TMEM), and the streamed
// tile serves as the K-major right operand of the first products and, by rows, as the MN-major
// one of the second.
//
// Warps: W softmax warpgroups that take the streamed tiles in turn, one warp that issues the
// products, one for the TMA loads.  One's exponentials run beside the products of another's tile:
// head dims above 64 have W = 2 in a CTA (TMEM: S and G of two tiles, 4 x 64 columns, and 2 x 128 of
// accumulators: an SM's 512); up to 64 a CTA has W = 1 in 256 columns and 80 KB, and two run on an
// SM, so that one's start and end overlap the other's work too (256 x 512 x 48, P and dS of one part: 114 us
// with W = 2, 80 so).  CTAs with the longest walks, of all chains, start first.
//
// P and dS are hi + lo to 2^-16, so that a result is off by its own rounding (2^-8) and no more.  Of one part
// each they would add as much again: errors of 1.41 of the results' rounding, up to 1.8 in short sequences,
// 1.55 for dq at head dims up to 32, whose terms cancel; and 76, 212 and 491 us for the times below.
//
// Measured: 256 x 512 x 48 85 us, 16 x 4096 x 96 252 us (0.51 PFLOP/s of the formula's five products), 96 x 2048 x 120
// 574 us (0.42).  The tensor core is busy 52% (d = 96) and 35% (d = 48), issue 34% and 43%: the rest is the softmax's
// chain (TMEM loads, exponentials, the parts, stores and hand-overs) and a CTA's start and end, which with W = 2 nothing
// overlaps.  With P and dS of one part: own tiles in TMEM (their products 30 cycles instead of 46), a third S and G, P and
// dS in columns of their own, the second half's TMEM loads ahead: no gain.
#include "hoa_attn_bwd.cuh"
#include "hoa_f32x2.cuh"
#include "hoa_tma.cuh"

namespace hoa {
using namespace sm100;

constexpr int kBwOwn = 128, kBwStr = 64;

template <int DP>
struct BwLayout {
  static constexpr int W = DP <= 64 ? 1 : 2, kThreads = 128 * W + 64;
  static constexpr int NKB = (DP + 63) / 64;
  static constexpr int kOwnBlk = kBwOwn * 128, kStrBlk = kBwStr * 128;     // 64 columns of a tile
  static constexpr int kOwn = NKB * kOwnBlk, kStr = NKB * kStrBlk;
  static constexpr int kStage = 2 * kStr, NS = W == 1 ? 3 : 4;
  static constexpr int offStage = 2 * kOwn;
  static constexpr int offCol = offStage + NS * kStage;                    // -lse log2 e and -D of the streamed queries
  static constexpr int offBar = offCol + W * 2 * 128 * 4;
  static constexpr int kAlloc = offBar + 256 + 1024;
  static_assert(kAlloc <= 232448, "shared memory budget");
  static constexpr uint32_t kCols = 256 * W;
  // TMEM of a role: S and G of NB tiles, then the accumulators (keys: A0 and A1)
  template <bool kKeys> struct Role {
    static constexpr int NB = W;      // (a third one for queries, whose columns allow it: no gain)
    static constexpr uint32_t colA0 = 128 * NB, colA1 = colA0 + (kKeys ? DP : 0);
    static_assert(colA1 + DP <= kCols, "TMEM columns");
  };
};

HOA_DEVICE float bw_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
HOA_DEVICE float bw_pack(F2 x) {
  const float2 v = f2_get(x);
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return __uint_as_float(*reinterpret_cast<const uint32_t*>(&h));
}

// x = hi + lo to 2^-16, two bf16 each
HOA_DEVICE void bw_split(F2 x, float& hi, float& lo) {
  hi = bw_pack(x);
  const uint32_t u = __float_as_uint(hi);
  lo = bw_pack(f2_fma(f2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)), f2(-1.f), x));
}
// columns (8 of them a 16 keys or queries) of the high and low parts of matrix rows in the place of their 64 fp32 values:
// [hi lo] of the first 32, [hi lo] of the second, so that either half goes over what was loaded of it
HOA_DEVICE constexpr uint32_t bw_part(int kk, bool lo) { return (kk >> 1) * 32 + (lo ? 16 : 0) + (kk & 1) * 8; }

struct BwMaps { CUtensorMap x0, x1, y0, y1; };

template <int DP, bool kKeys>
HOA_DEVICE void attn_bwd_tc_role(const BwMaps& maps, const AttnBwdArgs& p) {
  using L = BwLayout<DP>;
  using Role = typename L::template Role<kKeys>;
  constexpr int W = L::W, NB = Role::NB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  float* cols = reinterpret_cast<float*>(sm + L::offCol);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::offBar);
  uint64_t* own_full = bars;
  uint64_t* full = bars + 1;         // [NS]
  uint64_t* empty = full + L::NS;    // [NS]
  uint64_t* s_full = empty + L::NS;  // [NB] S and G are there
  uint64_t* p_full = s_full + NB;    // [W] P and dS are there
  uint64_t* fin = p_full + W;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fin + 1);
  volatile int* s_abort = reinterpret_cast<volatile int*>(fin + 2);
  const int tid = threadIdx.x, warp = tid >> 5, lid = tid & 31;
  const int chain = blockIdx.x, d = p.d;
  // the longest walks first: early keys, late queries
  const int own0 = (kKeys ? (int)blockIdx.y : (int)((p.Tq + kBwOwn - 1) / kBwOwn - 1 - blockIdx.y)) * kBwOwn;
  if (own0 < 0) return;                                             // (a launch has tiles for the longer side)
  int first = 0, n;
  if (kKeys) {
    first = max(0, own0 - p.q_offset) / kBwStr;
    n = max(0, (p.Tq + kBwStr - 1) / kBwStr - first);
  } else {
    n = (p.q_offset + min(own0 + kBwOwn, p.Tq) - 1) / kBwStr + 1;
  }
  if (tid == 0) {
    for (uint64_t* b = bars; b <= fin; ++b) mbar_init(b, b >= p_full && b < fin ? 4 : 1);
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
  bool bad = false;
  wait_previous();                                                  // D, copied rows

  if (warp == 4 * W + 1) {
    // ------------------------------------------------------------------ TMA
    if (lid == 0 && n > 0) {
      mbar_arrive_expect_tx(own_full, 2u * L::kOwn);
      for (int kb = 0; kb < L::NKB; ++kb) {
        tma_load_3d(sm + kb * L::kOwnBlk, &maps.x0, own_full, kb * 64, own0, chain);
        tma_load_3d(sm + L::kOwn + kb * L::kOwnBlk, &maps.x1, own_full, kb * 64, own0, chain);
      }
      int issued = 0;
      for (int j = 0; j < n; ++j) {
        const int s = j % L::NS;
        if (j >= L::NS && !mbar_wait_abortable(&empty[s], (j / L::NS - 1) & 1, s_abort, p.max_wait)) { bad = true; break; }
        uint8_t* st = sm + L::offStage + s * L::kStage;
        mbar_arrive_expect_tx(&full[s], (uint32_t)L::kStage);
        for (int kb = 0; kb < L::NKB; ++kb) {
          tma_load_3d(st + kb * L::kStrBlk, &maps.y0, &full[s], kb * 64, (first + j) * kBwStr, chain);
          tma_load_3d(st + L::kStr + kb * L::kStrBlk, &maps.y1, &full[s], kb * 64, (first + j) * kBwStr, chain);
        }
        issued = j + 1;
      }
      // copies in flight land before the CTA exits (the last fill of each stage)
      for (int j = max(0, issued - L::NS); j < issued; ++j) bad |= !mbar_wait(&full[j % L::NS], (j / L::NS) & 1);
      bad |= !mbar_wait(own_full, 0);
    }
    __syncwarp();
  } else if (warp == 4 * W) {
    // ------------------------------------------------------------------ MMA
    if (n > 0) {
      // the whole warp runs this alike; one lane issues
      const uint32_t lead = elect_one() ? 1u : 0u, tm = warp_uniform(tmem), base = warp_uniform(smem_u32(sm));
      constexpr uint32_t idS = make_idesc(kFmtBF16, 128, kBwStr), idA = make_idesc(kFmtBF16, 128, DP, true);
      const uint64_t dX0 = desc_sw128(base), dX1 = desc_sw128(base + L::kOwn);
      bool ok = mbar_wait_abortable(own_full, 0, s_abort, p.max_wait);
      auto front = [&](int j) {
        const int s = j % L::NS;
        ok = __all_sync(0xffffffffu, ok && mbar_wait_abortable(&full[s], (j / L::NS) & 1, s_abort, p.max_wait));
        if (!ok) return;
        tc_fence_after();
        const uint32_t st = base + L::offStage + s * L::kStage;
        const uint64_t dY0 = desc_sw128(st), dY1 = desc_sw128(st + L::kStr);
        const uint32_t cS = tm + (j % NB) * 128;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {                        // (in turn: one's sums do not wait for the other's)
          const uint64_t ox = (uint64_t)(((kk >> 2) * L::kOwnBlk + (kk & 3) * 32) >> 4);
          const uint64_t oy = (uint64_t)(((kk >> 2) * L::kStrBlk + (kk & 3) * 32) >> 4);
          mma_bf16_warp(cS, dX0 + ox, dY0 + oy, idS, kk > 0 ? 1u : 0u, lead);
          mma_bf16_warp(cS + 64, dX1 + ox, dY1 + oy, idS, kk > 0 ? 1u : 0u, lead);
        }
        tc_commit_warp(&s_full[j % NB], lead);
      };
      ok = __all_sync(0xffffffffu, ok);
      // (S and G of tile j + NB - 1 go where those of tile j - 1 were: behind the products that read P and dS there)
      constexpr int kAhead = NB - 1;
      for (int j = 0; j < min(kAhead, n); ++j) front(j);
      for (int j = 0; j < n && ok; ++j) {
        if (j + kAhead < n && (kAhead > 0 || j == 0)) front(j + kAhead);
        ok = __all_sync(0xffffffffu, ok && mbar_wait_abortable(&p_full[j % W], (j / W) & 1, s_abort, p.max_wait));
        if (!ok) break;
        tc_fence_after();
        const uint32_t st = base + L::offStage + (j % L::NS) * L::kStage;
        const uint64_t mY0 = desc_sw128_mn(st, L::kStrBlk), mY1 = desc_sw128_mn(st + L::kStr, L::kStrBlk);
        const uint32_t cS = tm + (j % NB) * 128;
#pragma unroll
        for (int i = 0; i < kBwStr / 8; ++i) {
          const int kk = i >> 1;
          const uint32_t at = bw_part(kk, (i & 1) == 0), acc = j > 0 || i > 0 ? 1u : 0u;      // (the small parts first)
          if (kKeys) mma_bf16_ts_warp(tm + Role::colA0, cS + at, mY1 + (uint64_t)(kk * 2048 >> 4), idA, acc, lead);
          mma_bf16_ts_warp(tm + Role::colA1, cS + 64 + at, mY0 + (uint64_t)(kk * 2048 >> 4), idA, acc, lead);
        }
        tc_commit_warp(&empty[j % L::NS], lead);
        if (W == 1 && j + 1 < n) front(j + 1);                     // (over P and dS, behind the products that read them)
      }
      if (!ok) bad = true;
      tc_commit_warp(fin, lead);
      bad |= !mbar_wait(fin, 0);
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- softmax
    const int g = warp >> 2;                                      // takes the tiles g, g + W, ...
    const int r = tid & 127;                                      // row of the own tile = TMEM lane
    const uint32_t lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    constexpr float kLog2e = 1.4426950408889634f;
    const float c = p.scale * kLog2e;
    const long long qrow = (long long)chain * p.Tq;
    // (the scaling by -log2 e and -1 waits until the value is used: the load is on its way a tile long)
    // rows that are not there: exp2 of -infinity
    auto stat = [&](const float* x, int q, float past) { return q < p.Tq ? x[qrow + q] : past; };
    float my_l = 0.f, my_D = 0.f, next = 0.f;
    if (kKeys) {
      const int q = (first + g) * kBwStr + (r & 63);
      if (g < n) next = r < 64 ? stat(p.lse, q, INFINITY) : stat(p.delta, q, 0.f);
    } else {
      my_l = -kLog2e * stat(p.lse, own0 + r, INFINITY);
      my_D = -stat(p.delta, own0 + r, 0.f);
    }
    for (int j = g; j < n; j += W) {
      const int t0 = (first + j) * kBwStr;
      float* col = cols + (g * 2 + ((j / W) & 1)) * 128;
      if (kKeys) {
        col[r] = next * (r < 64 ? -kLog2e : -1.f);
        named_sync(1 + g, 128);
        const int q = t0 + W * kBwStr + (r & 63);
        if (j + W < n) next = r < 64 ? stat(p.lse, q, INFINITY) : stat(p.delta, q, 0.f);
      }
      bad |= !mbar_wait_abortable(&s_full[j % NB], (j / NB) & 1, s_abort, p.max_wait);
      tc_fence_after();
      const uint32_t cS = tmem + lane + (j % NB) * 128;
      // columns of this row that count: keys, its own key up to the query; queries, keys up to its own
      int lo = 0, hi = kBwStr;
      if (kKeys) lo = own0 + r - p.q_offset - t0; else hi = p.q_offset + own0 + r - t0 + 1;
      const bool masked = kKeys ? own0 + kBwOwn - 1 > p.q_offset + t0 : t0 + kBwStr - 1 > p.q_offset + own0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float s[32], gr[32];
        tmem_ld32(cS + 32 * half, s);
        tmem_ld32(cS + 64 + 32 * half, gr);
        tmem_wait_ld();
        tmem_touch(s);
        tmem_touch(gr);
        if (masked) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (kKeys ? 32 * half + e < lo : 32 * half + e >= hi) s[e] = -INFINITY;
        }
        float ph[16], pl[16], dh[16], dl[16];                      // P's and dS's high and low parts
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          F2 l[2], D[2];
          if (kKeys) {
            const float4 lv = *reinterpret_cast<const float4*>(col + 32 * half + e);
            const float4 dv = *reinterpret_cast<const float4*>(col + 64 + 32 * half + e);
            l[0] = f2(lv.x, lv.y);
            l[1] = f2(lv.z, lv.w);
            D[0] = f2(dv.x, dv.y);
            D[1] = f2(dv.z, dv.w);
          } else {
            l[0] = l[1] = f2(my_l);
            D[0] = D[1] = f2(my_D);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int i = e + 2 * k;
            const float2 z = f2_get(f2_fma(f2(s[i], s[i + 1]), f2(c), l[k]));
            const F2 pr = f2(bw_exp2(z.x), bw_exp2(z.y));
            if (kKeys) bw_split(pr, ph[i / 2], pl[i / 2]);
            bw_split(f2_mul(pr, f2_add(f2(gr[i], gr[i + 1]), D[k])), dh[i / 2], dl[i / 2]);
          }
        }
        if (kKeys) {
          tmem_st16(cS + 32 * half, ph);
          tmem_st16(cS + 32 * half + 16, pl);
        }
        tmem_st16(cS + 64 + 32 * half, dh);
        tmem_st16(cS + 64 + 32 * half + 16, dl);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lid == 0) mbar_arrive(&p_full[g]);
    }
    // ---- epilogue: rows of the own tile that exist; 16 columns of dv, dk (or dq) a warpgroup in turn
    if (n > 0) bad |= !mbar_wait_abortable(fin, 0, s_abort, p.max_wait);
    tc_fence_after();
    const int rows = kKeys ? p.Tk : p.Tq;
    const long long row_at = ((long long)chain * rows + own0 + r) * d;
    constexpr int kC = DP / 16;
#pragma unroll
    for (int i = 0; i < (kKeys ? 2 : 1) * kC; ++i) {
      if (i % W != g) continue;
      const bool is_dv = kKeys && i < kC;
      const int c16 = i % kC;
      float v[16];
      if (n > 0) {
        tmem_ld16(tmem + lane + (is_dv ? Role::colA0 : Role::colA1) + 16 * c16, v);
        tmem_wait_ld();
        tmem_touch(v);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0.f;
      }
      if (own0 + r >= rows || bad) continue;
      const float f = is_dv ? 1.f : p.scale;
      __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(!kKeys ? p.dq : is_dv ? p.dv : p.dk) + row_at + 16 * c16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (16 * c16 + 8 * h >= d) continue;
        uint4 w;
        uint32_t* u = &w.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(bw_pack(f2(v[8 * h + 2 * e] * f, v[8 * h + 2 * e + 1] * f)));
        *reinterpret_cast<uint4*>(out + 8 * h) = w;
      }
    }
  }

  bad = __syncthreads_or(bad || *s_abort != 0);
  if (bad && tid == 0 && p.status != nullptr) *reinterpret_cast<volatile int*>(p.status) = HOA_ERR_TIMEOUT;
  tc_fence_after();
  if (warp == 0) tmem_dealloc(tmem, L::kCols);
}

// Both roles in one launch (blockIdx.z): neither waits for the other.
template <int DP>
__global__ void __launch_bounds__(BwLayout<DP>::kThreads, BwLayout<DP>::W == 1 ? 2 : 1)
attn_bwd_tc_kernel(const __grid_constant__ BwMaps keys, const __grid_constant__ BwMaps queries, const __grid_constant__ AttnBwdArgs p) {
  if (blockIdx.z == 0) attn_bwd_tc_role<DP, true>(keys, p);
  else attn_bwd_tc_role<DP, false>(queries, p);
}

template <int DP>
static int launch_bwd_tc(const AttnBwdArgs& a, int BH, cudaStream_t s) {
  using L = BwLayout<DP>;
  BwMaps m[2];                                                      // of keys and of queries that own the tile
  auto map = [&](CUtensorMap* to, const void* x, int rows, int box) {
    return make_map(to, x, a.d, rows, BH, (uint64_t)a.d * 2, (uint64_t)rows * a.d * 2, box);
  };
  if (!map(&m[0].x0, a.k, a.Tk, kBwOwn) || !map(&m[0].x1, a.v, a.Tk, kBwOwn) || !map(&m[0].y0, a.q, a.Tq, kBwStr) ||
      !map(&m[0].y1, a.dout, a.Tq, kBwStr) || !map(&m[1].x0, a.q, a.Tq, kBwOwn) || !map(&m[1].x1, a.dout, a.Tq, kBwOwn) ||
      !map(&m[1].y0, a.k, a.Tk, kBwStr) || !map(&m[1].y1, a.v, a.Tk, kBwStr))
    return HOA_ERR_INVALID_ARG;
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(attn_bwd_tc_kernel<DP>, L::kAlloc, done)) return HOA_ERR_LAUNCH;
  const int tiles = ceil_div(a.Tk, kBwOwn);                         // (Tq <= Tk)
  if (tiles > 65535) return HOA_ERR_UNSUPPORTED;
  return launch_early(attn_bwd_tc_kernel<DP>, dim3((unsigned)BH, (unsigned)tiles, 2), 1, L::kThreads, L::kAlloc, s, m[0], m[1], a);
}

static int attn_bwd_tc_of(const AttnBwdArgs& a, int BH, cudaStream_t s) {
  switch ((a.d + 15) / 16) {
    case 1: return launch_bwd_tc<16>(a, BH, s);
    case 2: return launch_bwd_tc<32>(a, BH, s);
    case 3: return launch_bwd_tc<48>(a, BH, s);
    case 4: return launch_bwd_tc<64>(a, BH, s);
    case 5: return launch_bwd_tc<80>(a, BH, s);
    case 6: return launch_bwd_tc<96>(a, BH, s);
    case 7: return launch_bwd_tc<112>(a, BH, s);
    default: return launch_bwd_tc<128>(a, BH, s);
  }
}

// Rows of d elements <-> rows of d8 = d rounded up to 8, zeros behind; a thread 8 elements, blockIdx.y the tensor.
struct BwCopy { const void* src[4]; void* dst[4]; long long rows[4]; int d, d8; };

template <bool kPad>
__global__ void __launch_bounds__(256) attn_bwd_copy_kernel(const __grid_constant__ BwCopy p) {
  const int per = p.d8 / 8, t = blockIdx.y;
  const long long n = p.rows[t] * per;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / per;
    const int e = (int)(i - row * per) * 8;
    uint4 w = make_uint4(0, 0, 0, 0);
    unsigned short* u = reinterpret_cast<unsigned short*>(&w);
    if (kPad) {
      const unsigned short* src = reinterpret_cast<const unsigned short*>(p.src[t]) + row * p.d + e;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k < p.d) u[k] = src[k];
      reinterpret_cast<uint4*>(p.dst[t])[i] = w;
    } else {
      w = reinterpret_cast<const uint4*>(p.src[t])[i];
      unsigned short* dst = reinterpret_cast<unsigned short*>(p.dst[t]) + row * p.d + e;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (e + k < p.d) dst[k] = u[k];
    }
  }
}

static size_t bw_up(size_t v) { return (v + 255) / 256 * 256; }

size_t attn_bwd_tc_bytes(int BH, int Tq, int Tk, int d) {
  const size_t row = (size_t)(d + 7) / 8 * 16;
  return 3 * bw_up((size_t)BH * Tq * row) + 4 * bw_up((size_t)BH * Tk * row);
}

int attn_bwd_tc(const AttnBwdArgs& a, int BH, void* copies, cudaStream_t s) {
  if (copies == nullptr) return attn_bwd_tc_of(a, BH, s);
  // rows that TMA does not take (d % 8 != 0, or tensors off 16-byte boundaries) go through copies of rounded-up rows: the zeros
  // behind change no product.  2 x 1500 x 50: 39 us, 8 of them the copies.
  const int d8 = (a.d + 7) / 8 * 8;
  const long long q = (long long)BH * a.Tq, k = (long long)BH * a.Tk;
  unsigned char* at = reinterpret_cast<unsigned char*>(copies);
  auto take = [&](long long rows) {
    void* x = at;
    at += bw_up((size_t)rows * d8 * 2);
    return x;
  };
  AttnBwdArgs b = a;
  BwCopy in{{a.q, a.dout, a.k, a.v}, {take(q), take(q), take(k), take(k)}, {q, q, k, k}, a.d, d8};
  BwCopy out{{take(q), take(k), take(k)}, {a.dq, a.dk, a.dv}, {q, k, k}, a.d, d8};
  b.q = in.dst[0]; b.dout = in.dst[1]; b.k = in.dst[2]; b.v = in.dst[3];
  b.dq = const_cast<void*>(out.src[0]); b.dk = const_cast<void*>(out.src[1]); b.dv = const_cast<void*>(out.src[2]);
  b.d = d8;
  const long long ctas = (k * (d8 / 8) + 255) / 256;
  const unsigned grid = (unsigned)(ctas < 4096 ? ctas : 4096);
  attn_bwd_copy_kernel<true><<<dim3(grid, 4), 256, 0, s>>>(in);
  if (int st = launch_status()) return st;
  if (int st = attn_bwd_tc_of(b, BH, s)) return st;
  attn_bwd_copy_kernel<false><<<dim3(grid, 3), 256, 0, s>>>(out);
  return launch_status();
}

}  // namespace hoa
