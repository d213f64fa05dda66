// Paged attention for many query rows (bf16) on tcgen05 / TMEM.
//
// An item is up to two 128-row tiles of queries against a range of keys: the rows
// of the whole batch against the shared pages, or a row's own queries (a prompt)
// against its own pages.  The structure is that of attn_tc_kernel
// (hoa_attn_tc.cu): a softmax warpgroup per query tile, one warp that issues the
// products, one that issues the TMA loads; what differs:
//   * K and V tiles come page by page: a box of the 4-D map (d, token, head, page)
//     per page, the page id looked up one tile ahead by a lane each.  V stays
//     token-major as the cache holds it: it is the MN-major B operand of P V.
//   * Q rows are gathered (rows of different sequences, grouped heads, any
//     strides), so the softmax threads place their own row in the swizzled tile.
//   * every row has its own last key, and a row may see none.
//   * items of at most 128 rows (kDup) give both warpgroups the same rows and every
//     other key tile each: one alone takes 3.7K cycles for 128 keys, slower than HBM
//     brings them.  Their two O lie in the same lanes, where the first joins them.
//     Measured (d = 96, 16 heads, 32768 shared keys): 64 rows 95 -> 81 us, 24 rows
//     83 -> 70; 128 rows x 8 heads of 64 over 16384 keys 42 -> 37.
//   * the result is the item's unnormalised (m, l, O).
// What bounds it: 128 keys of a pair of tiles take 3.9K cycles, of which the issuing
// lane is busy 2.6K (scores 600 a tile, P V 730: about 95 cycles a product of 64, while
// the softmax warps use TMEM and the loads shared memory), the exponentials 2K (16 an SM
// cycle).  Prompts of 128 tokens in 16 rows over 4096 shared ones, 16 heads of 96 (51
// GFLOP): 105 us, 485 TFLOP/s.  Two score buffers of 64 keys (129 us against 112) and
// weights in columns of their own (110 against 107) overlap more and gain nothing.
// A key tile holds KT <= 128 keys, a whole number of pages (or of tiles in a page).
// Slots past the last key that any row of the item sees may hold NaN: their
// weights are 0, and the V rows are zeroed in shared memory before the product.
#include <cudaTypedefs.h>

#include "hoa_f32x2.cuh"
#include "hoa_paged_attn.cuh"
#include "hoa_sm100.cuh"

namespace hoa {
using namespace sm100;

constexpr int kPtThreads = 320;
constexpr int kPtRescaleLog2 = 8;

template <int DP16>
struct PtLayout {
  static constexpr int NKB = (DP16 + 63) / 64;        // 64-column slabs of a tile
  static constexpr int kBlk = 128 * 128;              // bytes: 128 rows x 128 B
  static constexpr int kQ = NKB * kBlk;               // one Q, K or V tile
  static constexpr int kStage = 2 * kQ;
  static constexpr int NS = NKB == 1 ? 4 : 2;
  static constexpr int offQ = 0;
  static constexpr int offStage = 2 * kQ;
  static constexpr int offBar = offStage + NS * kStage;
  static constexpr int kBytes = offBar + 256;
  static constexpr int kAlloc = kBytes + 1024;        // slack to align the base to 1024
  static_assert(kAlloc <= 232448, "shared memory budget");
  static constexpr uint32_t colS0 = 0, colS1 = 128, colO0 = 256, colO1 = 384;
};

HOA_DEVICE void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

HOA_DEVICE uint32_t pt_pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

struct PtArgs {
  int kt;              // keys of a tile
  int box;             // keys of a TMA box: kt or a page
  bool qvec;           // rows of q are 16-byte aligned
  long long max_wait;
};

template <int DP16, bool kDup>
__global__ void __launch_bounds__(kPtThreads, 1)
paged_attn_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                     const __grid_constant__ PaArgs p, const PtArgs pt, unsigned first) {
  using L = PtLayout<DP16>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::offBar);
  uint64_t* q_full = bars + 0;
  uint64_t* s_full = bars + 1;       // [2] per Q tile
  uint64_t* p_full = bars + 3;       // [2] per Q tile
  uint64_t* pv_done = bars + 5;      // [2] per Q tile
  uint64_t* fin = bars + 7;
  // K and V of a stage are handed over apart: K is free again once the last scores are computed, a round before V
  uint64_t* k_full = bars + 8;       // [NS]
  uint64_t* v_full = bars + 12;      // [NS]
  uint64_t* k_empty = bars + 16;     // [NS]
  uint64_t* v_empty = bars + 20;     // [NS]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
  volatile int* s_abort = reinterpret_cast<volatile int*>(bars + 25);
  int* s_seen = reinterpret_cast<int*>(bars + 26);   // [2] the last key that a row of the tile sees, + 1

  const int tid = threadIdx.x, warp = tid >> 5, lid = tid & 31;
  const int KT = pt.kt;
  if (tid == 0) {
    mbar_init(q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(fin, 1);
    for (int i = 0; i < L::NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    *s_abort = 0;
    s_seen[0] = s_seen[1] = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pa_begin(p.leads);
  const PaItem it = pa_item(p, first + blockIdx.x, kDup ? 128 : 256, KT);
  __syncthreads();
  PaRow my{};
  int seen = 0;
  if (warp < 8) {
    my = pa_row(p, it, it.row0 + (kDup ? tid & 127 : tid));     // warps 0-3: tile 0, warps 4-7: tile 1
    seen = my.ok ? max(0, min(my.seen - it.key_base, it.k1)) : 0;
    const int top = __reduce_max_sync(0xffffffffu, seen);
    if (lid == 0) atomicMax(&s_seen[warp >> 2], top);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int n_t[2], kmax = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    n_t[i] = s_seen[i] > it.k0 ? (s_seen[i] - it.k0 + KT - 1) / KT : 0;
    kmax = max(kmax, s_seen[i]);
  }
  const int nkt = max(n_t[0], n_t[1]);               // key tiles of the item
  if (kDup) {
    n_t[0] = (nkt + 1) / 2;
    n_t[1] = nkt / 2;
  }
  // the key tile that warpgroup i takes as its j-th
  auto tile = [](int i, int j) { return kDup ? 2 * j + i : j; };
  bool bad = false;

  if (warp == 9) {
    // ------------------------------------------------------------------ TMA
    const int nbox = KT / pt.box;
    // page of this lane's box of tile j, -1: no key of it is seen (or its page lies outside the pool)
    auto page_of = [&](int j) -> int {
      const int k = it.k0 + j * KT + lid * pt.box;
      if (lid >= nbox || j >= nkt || k >= kmax) return -1;
      const int pg = k / p.page;
      const int id = it.part == 1 ? p.shared[pg] : p.table[it.b * p.tstride + pg];
      if (id >= 0 && id < p.n_pages) return id;
      pa_fail(p.status);
      return -1;
    };
    int id = page_of(0);
    int issued[2] = {0, 0};                          // K, V tiles
    for (int j = 0; j < nkt && !bad; ++j) {
      const int s = j % L::NS, round = j / L::NS;
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, id >= 0)) * (uint32_t)(pt.box * 128 * L::NKB);
      const int y = (it.k0 + j * KT + lid * pt.box) % p.page;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        uint64_t* full = (kv ? v_full : k_full) + s;
        bool ok = true;
        if (lid == 0 && round > 0) ok = mbar_wait_abortable((kv ? v_empty : k_empty) + s, (round - 1) & 1, s_abort, pt.max_wait);
        if (!__all_sync(0xffffffffu, ok)) { bad = true; break; }
        if (lid == 0) mbar_arrive_expect_tx(full, bytes);
        __syncwarp();
        if (id >= 0) {
          uint8_t* st = sm + L::offStage + s * L::kStage + kv * L::kQ + lid * pt.box * 128;
          for (int kb = 0; kb < L::NKB; ++kb) tma_load_4d(st + kb * L::kBlk, kv ? &tv : &tk, full, kb * 64, y, it.kvh, id);
        }
        issued[kv] = j + 1;
      }
      id = page_of(j + 1);
    }
    // copies in flight land before the CTA exits (the last fill of each stage)
    if (lid == 0)
      for (int kv = 0; kv < 2; ++kv)
        for (int j = max(0, issued[kv] - L::NS); j < issued[kv]; ++j)
          bad |= !mbar_wait((kv ? v_full : k_full) + j % L::NS, (j / L::NS) & 1);
    __syncwarp();
  } else if (warp == 8) {
    // ------------------------------------------------------------------ MMA
    if (lid == 0) {
      const uint32_t idS = make_idesc(kFmtBF16, 128, KT);
      constexpr uint32_t idO = make_idesc(kFmtBF16, 128, DP16, true);
      constexpr int KSTEPS = DP16 / 16;
      const uint64_t dQ[2] = {desc_sw128(smem_u32(sm + L::offQ)), desc_sw128(smem_u32(sm + L::offQ + (kDup ? 0 : L::kQ)))};
      const uint32_t colS[2] = {tmem + L::colS0, tmem + L::colS1};
      const uint32_t colO[2] = {tmem + L::colO0, tmem + L::colO1};
      bool ok = mbar_wait_abortable(q_full, 0, s_abort, pt.max_wait);
      // Order: S0 S1 | PV0 S0' PV1 S1' | ...: a query tile's next scores are computed as soon as its own weights are
      // taken, so that the two softmax warpgroups run out of step and the products of one hide behind the other's
      // exponentials (with S0 S1 PV0 PV1 both waited for all four).
      int have = 0, v_have = 0;                      // K and V tiles known to have landed
      auto scores = [&](int i, int j) {
        const int t = tile(i, j), s = t % L::NS;
        if (t >= have) {
          ok = mbar_wait_abortable(&k_full[s], (t / L::NS) & 1, s_abort, pt.max_wait);
          if (!ok) return;
          have = t + 1;
        }
        tc_fence_after();
        const uint64_t dK = desc_sw128(smem_u32(sm + L::offStage + s * L::kStage));
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
          const uint64_t off = (uint64_t)(((kk >> 2) * L::kBlk + (kk & 3) * 32) >> 4);
          mma_bf16(colS[i], dQ[i] + off, dK + off, idS, kk > 0 ? 1u : 0u);
        }
        tc_commit(&s_full[i]);
        if (kDup || i == 1 || j >= n_t[1]) tc_commit(&k_empty[s]);      // the tile's last scores
      };
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (ok && n_t[i] > 0) scores(i, 0);
      for (int j = 0; j < max(n_t[0], n_t[1]) && ok; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (j >= n_t[i] || !ok) continue;
          const int t = tile(i, j), s = t % L::NS;
          const uint64_t dV = desc_sw128_mn(smem_u32(sm + L::offStage + s * L::kStage) + L::kQ, L::kBlk);
          ok = mbar_wait_abortable(&p_full[i], j & 1, s_abort, pt.max_wait);
          if (!ok) break;
          if (t >= v_have) {
            ok = mbar_wait_abortable(&v_full[s], (t / L::NS) & 1, s_abort, pt.max_wait);
            if (!ok) break;
            v_have = t + 1;
          }
          tc_fence_after();
          for (int kk = 0; kk < KT / 16; ++kk)         // 16 keys: 16 rows of 128 bytes of every V slab
            mma_bf16_ts(colO[i], colS[i] + kk * 8, dV + (uint64_t)(kk * 2048 >> 4), idO, (j > 0 || kk > 0) ? 1u : 0u);
          tc_commit(&pv_done[i]);
          if (kDup || i == 1 || j >= n_t[1]) tc_commit(&v_empty[s]);    // the tile's last weights
          if (j + 1 < n_t[i]) scores(i, j + 1);
        }
      }
      if (!ok) bad = true;
      tc_commit(fin);
      bad |= !mbar_wait(fin, 0);
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- softmax
    const int i = warp >> 2;                         // Q tile of this warpgroup
    const int r = tid & 127;                         // row in the tile = TMEM lane
    {
      const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q) + my.b * p.qsb + my.t * p.qst + my.h * p.qsh;
      uint8_t* dst = sm + L::offQ + i * L::kQ;
#pragma unroll
      for (int ch = 0; ch < L::NKB * 8; ++ch) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (kDup && i == 1) break;                    // (the rows are in place already)
        if (my.ok && ch * 8 < p.d) {
          if (pt.qvec) {
            v = *reinterpret_cast<const uint4*>(q + ch * 8);
          } else {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(q + ch * 8);
            v = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                           e[6] | (uint32_t)e[7] << 16);
          }
        }
        *reinterpret_cast<uint4*>(dst + (ch >> 3) * L::kBlk + sw128_offset(r, ch & 7)) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lid == 0) mbar_arrive(q_full);
    }
    const uint32_t lane = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t cS = tmem + (i ? L::colS1 : L::colS0) + lane;
    const uint32_t cO = tmem + (i ? L::colO1 : L::colO0) + lane;
    const int ni = n_t[i];
    const bool live = __any_sync(0xffffffffu, seen > it.k0);    // some row of the warp sees a key of the item
    const float c = p.scale_log2;
    float m_ref = -INFINITY, l_run = 0.f;
    for (int j = 0; j < ni; ++j) {
      bad |= !mbar_wait_abortable(&s_full[i], j & 1, s_abort, pt.max_wait);
      tc_fence_after();
      const int t = tile(i, j), k0 = it.k0 + t * KT;
      if (t == nkt - 1 && kmax - k0 < KT) {
        // V rows past the last key that is seen: zero (each warpgroup that runs this tile)
        const int s = t % L::NS;
        bad |= !mbar_wait_abortable(&v_full[s], (t / L::NS) & 1, s_abort, pt.max_wait);
        uint8_t* v = sm + L::offStage + s * L::kStage + L::kQ;
        if (r >= kmax - k0 && r < KT)
#pragma unroll
          for (int ch = 0; ch < L::NKB * 8; ++ch)
            *reinterpret_cast<uint4*>(v + (ch >> 3) * L::kBlk + r * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      if (live) {
        const int lim = min(seen - k0, KT);          // keys of the tile that the row sees
        float sv[4][32];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) tmem_ld32(cS + 32 * q4, sv[q4]);
        tmem_wait_ld();
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) tmem_touch(sv[q4]);
        if (lim < 128) {
#pragma unroll
          for (int k = 0; k < 128; ++k)
            if (k >= lim) sv[k >> 5][k & 31] = -INFINITY;
        }
        float mx[4];                                 // 4 independent partial maxima
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = sv[0][u];
#pragma unroll
        for (int k = 4; k < 128; ++k) mx[k & 3] = fmaxf(mx[k & 3], sv[k >> 5][k & 31]);
        const float m_cand = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;   // (c > 0)
        const bool move = m_cand > m_ref + (float)kPtRescaleLog2;    // also the first key seen (m_ref = -inf)
        const float m_new = move ? m_cand : m_ref;
        const float corr = move ? pa_ex2(m_ref - m_new) : 1.f;          // 0 at the first key seen
        if (__any_sync(0xffffffffu, move) && j > 0) {
          // rescale this warp's rows of O once the previous P V has completed
          bad |= !mbar_wait_abortable(&pv_done[i], (j - 1) & 1, s_abort, pt.max_wait);
          tc_fence_after();
#pragma unroll
          for (int c16 = 0; c16 < DP16 / 16; ++c16) {
            float ov[16];
            tmem_ld16(cO + 16 * c16, ov);
            tmem_wait_ld();
            tmem_touch(ov);
#pragma unroll
            for (int e = 0; e < 16; ++e) ov[e] *= corr;
            tmem_st16(cO + 16 * c16, ov);
          }
        }
        l_run *= corr;
        m_ref = m_new;
        const float ref = m_ref == -INFINITY ? 0.f : m_ref;          // no key seen yet: weights 0
        const F2 c2 = f2(c), r2 = f2(-ref);
        F2 ps[4] = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 4; ++h) {                // 32 keys -> 16 packed columns
          float pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 x = f2_get(f2_fma(f2(sv[h][2 * e], sv[h][2 * e + 1]), c2, r2));
            const float p0 = pa_ex2(x.x), p1 = pa_ex2(x.y);
            ps[e & 3] = f2_add(ps[e & 3], f2(p0, p1));
            // the weights are rounded to bf16 for the product only; l sums them unrounded
            pk[e] = __uint_as_float(pt_pack(p0, p1));
          }
          tmem_st16(cS + 16 * h, pk);
        }
        const float2 sum = f2_get(f2_add(f2_add(ps[0], ps[1]), f2_add(ps[2], ps[3])));
        l_run += sum.x + sum.y;
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lid == 0) mbar_arrive(&p_full[i]);
    }
    // ---- epilogue: the item's (m, l, O) of the rows that exist
    if (ni > 0) bad |= !mbar_wait_abortable(&pv_done[i], (ni - 1) & 1, s_abort, pt.max_wait);
    tc_fence_after();
    const long long part = (long long)it.slot * p.rows + my.grow;
    float f0 = 1.f, f1 = 0.f;                        // factors of this warpgroup's O, of the second one's
    if (kDup) {
      // the second warpgroup's (m, l) through shared memory (the Q slabs of the absent tile), its O from TMEM
      float2* s_ml = reinterpret_cast<float2*>(sm + L::offQ + L::kQ);
      if (i == 1) s_ml[r] = make_float2(m_ref, bad ? 0.f : l_run);
      tc_fence_before();
      named_sync(1, 256);
      tc_fence_after();
      if (i == 0) {
        const float2 o2 = s_ml[r];
        if (o2.y != 0.f) {                           // (NaN stays NaN)
          const float m = fmaxf(m_ref, o2.x);
          f0 = l_run != 0.f ? pa_ex2(m_ref - m) : 0.f;
          f1 = pa_ex2(o2.x - m);
          l_run = l_run * f0 + o2.y * f1;
          m_ref = m;
        }
      }
    }
    if (!kDup || i == 0) {
      const bool first_ran = ni > 0, second_ran = kDup && n_t[1] > 0;
      if (my.ok) p.part_ml[part] = make_float2(m_ref, bad ? 0.f : l_run);
      if (live) {
        float* orow = p.part_o + part * p.d;
#pragma unroll
        for (int c16 = 0; c16 < DP16 / 16; ++c16) {
          float ov[16], ow[kDup ? 16 : 1];
          if (first_ran) tmem_ld16(cO + 16 * c16, ov);
          if constexpr (kDup) {
            if (second_ran) tmem_ld16(tmem + L::colO1 + lane + 16 * c16, ow);
          }
          tmem_wait_ld();
          tmem_touch(ov);
          tmem_touch(ow);
          if (my.ok && !bad && l_run > 0.f) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (second_ran) ov[e] = (f0 > 0.f ? ov[e] * f0 : 0.f) + (f1 > 0.f ? ow[kDup ? e : 0] * f1 : 0.f);
#pragma unroll
            for (int e = 0; e < 16; e += 4)          // (d is a multiple of 8)
              if (16 * c16 + e < p.d)
                *reinterpret_cast<float4*>(orow + 16 * c16 + e) = make_float4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
          }
        }
      }
    }
  }

  wait_previous();
  bad = __syncthreads_or(bad || *s_abort != 0);
  if (bad && tid == 0 && p.status != nullptr) *reinterpret_cast<volatile int*>(p.status) = HOA_ERR_TIMEOUT;
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

static bool page_map(CUtensorMap* m, const void* base, const PaArgs& a, int box) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return false;
  cuuint64_t dims[4] = {(cuuint64_t)a.d, (cuuint64_t)a.page, (cuuint64_t)a.Hk, (cuuint64_t)a.n_pages};
  cuuint64_t strides[3] = {(cuuint64_t)a.ts * 2, (cuuint64_t)a.hs * 2, (cuuint64_t)a.ps * 2};
  cuuint32_t bx[4] = {64, (cuuint32_t)box, 1, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, bx, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP16, bool kDup>
static int launch_ptc_d(const CUtensorMap& mk, const CUtensorMap& mv, const PaArgs& a, const PtArgs& t, unsigned first,
                      unsigned items, cudaStream_t s) {
  using L = PtLayout<DP16>;
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(paged_attn_tc_kernel<DP16, kDup>, L::kAlloc, done)) return HOA_ERR_LAUNCH;
  return launch_early(paged_attn_tc_kernel<DP16, kDup>, items, 1, kPtThreads, L::kAlloc, s, mk, mv, a, t, first);
}

template <int DP16>
static int launch_ptc(const CUtensorMap& mk, const CUtensorMap& mv, const PaArgs& a, const PtArgs& t, bool dup, unsigned first,
                      unsigned items, cudaStream_t s) {
  return dup ? launch_ptc_d<DP16, true>(mk, mv, a, t, first, items, s) : launch_ptc_d<DP16, false>(mk, mv, a, t, first, items, s);
}

int paged_attn_tc(const PaArgs& a, bool dup, unsigned first, unsigned items, cudaStream_t s) {
  PtArgs t;
  t.kt = pa_tile_keys(a.page);
  t.box = a.page < t.kt ? a.page : t.kt;
  t.qvec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.qsb * 2) | (uintptr_t)(a.qst * 2) | (uintptr_t)(a.qsh * 2)) & 15) == 0;
  t.max_wait = wait_bound_cycles();
  CUtensorMap mk, mv;
  if (t.kt == 0 || !page_map(&mk, a.kp, a, t.box) || !page_map(&mv, a.vp, a, t.box)) return HOA_ERR_INVALID_ARG;
  switch ((a.d + 15) / 16) {
    case 1: return launch_ptc<16>(mk, mv, a, t, dup, first, items, s);
    case 2: return launch_ptc<32>(mk, mv, a, t, dup, first, items, s);
    case 3: return launch_ptc<48>(mk, mv, a, t, dup, first, items, s);
    case 4: return launch_ptc<64>(mk, mv, a, t, dup, first, items, s);
    case 5: return launch_ptc<80>(mk, mv, a, t, dup, first, items, s);
    case 6: return launch_ptc<96>(mk, mv, a, t, dup, first, items, s);
    case 7: return launch_ptc<112>(mk, mv, a, t, dup, first, items, s);
    case 8: return launch_ptc<128>(mk, mv, a, t, dup, first, items, s);
    default: return HOA_ERR_UNSUPPORTED;
  }
}

}  // namespace hoa
