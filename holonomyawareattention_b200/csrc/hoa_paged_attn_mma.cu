// Paged attention for few query rows (bf16): every warp streams its own keys.
//
// An item is at most 16 query rows against a range of keys; its 4 warps take the
// range's 16-key chunks in turn.  A warp copies a chunk of K and V to its own two
// shared-memory stages (16-byte asynchronous copies, a key's page looked up by one
// lane one chunk ahead), and runs
//   S (16 x 16) = Q K^T, online softmax, O (16 x d) += P V
// on m16n8k16 products whose accumulators and P stay in registers.  No barrier in
// the loop: warps meet once at the end, to join their (m, l, O).
//
// What bounds it is HBM: a key costs 4 d bytes (23.6 bytes an SM cycle at the
// measured copy rate, so 16 keys of d = 96 take 260 SM cycles): 16 warps an SM with a
// chunk of 6 KB each in flight keep 96 KB under way, twice what the latency needs -
// as long as a warp's own chain through a chunk stays short.  So, where pages hold
// whole chunks of adjacent tokens, a chunk's copies go to fixed offsets from one base;
// masks are applied only where a chunk has keys that some row does not see; and up to
// 8 query rows leave the lower half of the 16-row tile out of the softmax.  Measured: 8
// rows of 16 heads over 65536 shared tokens (460 MB) 85 us, 5.4 TB/s; 128 rows x 24
// heads of 120 with up to 512 tokens of their own (378 MB) 75 us, 5.0 TB/s.  The tensor
// cores' tcgen05 form (hoa_paged_attn_tc.cu) takes over where the rows of a head
// fill more of its 128-row tile.
#include "hoa_paged_attn.cuh"
#include "hoa_sm100.cuh"

namespace hoa {

constexpr int kPmWarps = 4, kPmKeys = 16, kPmStages = 2;

template <int D8>
struct PmCfg {
  static constexpr int d = 8 * D8, KS = (D8 + 1) / 2;      // k-steps of 16 over the head dim
  static constexpr int kRow = KS * 32 + 16;                // bytes of a key's row: an odd number of 16-byte chunks, so that
                                                           // the 8 rows of a matrix load fall on different banks
  static constexpr int kTile = kPmKeys * kRow;             // K or V chunk
  static constexpr int kStage = 2 * kTile;
  static constexpr int kWarp = kPmStages * kStage;
  static constexpr int kRing = kPmWarps * kWarp;
  static constexpr int kJoinRow = d + 4;                   // floats of a row of the join
  static constexpr int kJoin = kPmWarps * 16 * kJoinRow * 4;
  static constexpr int offRow = kRing > kJoin ? kRing : kJoin;   // per row: its place in the outputs, the warps' factors
  static constexpr int kSmem = offRow + 16 * 8 + 16 * 4 * 4;
  static constexpr int kMinBlocks = D8 <= 12 ? 4 : 3;
};

HOA_DEVICE void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
HOA_DEVICE void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
HOA_DEVICE void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

HOA_DEVICE void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
HOA_DEVICE void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
HOA_DEVICE void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
HOA_DEVICE uint32_t pm_pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// kHalf: at most 8 rows an item.
template <int D8, bool kHalf>
__global__ void __launch_bounds__(kPmWarps * 32, PmCfg<D8>::kMinBlocks)
paged_attn_mma_kernel(const __grid_constant__ PaArgs p, unsigned first) {
  using C = PmCfg<D8>;
  extern __shared__ __align__(16) uint8_t smem[];
  pa_begin(p.leads);
  PaItem it = pa_item(p, first + blockIdx.x, 16, kPmKeys);
  const int tid = threadIdx.x, w = tid >> 5, lid = tid & 31, r0 = lid >> 2, q2 = (lid & 3) * 2;
  const uint32_t ring = sm100::smem_u32(smem) + w * C::kWarp;

  // the pad chunk of a head dim that is 8 mod 16 enters the products: zero, once
  if (D8 & 1) {
    for (int i = lid; i < kPmStages * 2 * kPmKeys; i += 32)
      *reinterpret_cast<uint4*>(smem + w * C::kWarp + i * C::kRow + D8 * 16) = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }

  // no key past the last one that a row of the item sees is read: its slot may hold anything; keys before the last
  // one that every row sees need no mask
  // (lane l has row l % 16 of the item: where its q lies, and how many keys of the part it sees)
  int all_see, my_seen;
  long long my_q;
  {
    const PaRow row = pa_row(p, it, it.row0 + (lid & 15));
    my_seen = row.ok ? row.seen - it.key_base : 0;
    my_q = row.ok ? row.b * p.qsb + row.t * p.qst + row.h * p.qsh : -1;
    it.k1 = min(it.k1, __reduce_max_sync(0xffffffffu, my_seen));
    all_see = min(it.k1, __reduce_min_sync(0xffffffffu, row.ok ? my_seen : 0x7fffffff));
    if (tid < 16) reinterpret_cast<long long*>(smem + C::offRow)[tid] = row.ok ? row.grow : -1;
  }
  const int chunks = it.k1 > it.k0 ? (it.k1 - it.k0 + kPmKeys - 1) / kPmKeys : 0;
  const uint8_t* kp = reinterpret_cast<const uint8_t*>(p.kp);
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(p.vp);
  constexpr int NP = (kPmKeys * D8 + 31) / 32;          // 16-byte pieces of a lane
  // whole chunks of adjacent tokens: one offset a chunk (pieces 16 bytes apart); else one a key, on lanes 0-15
  const bool whole = p.page % kPmKeys == 0 && p.ts == C::d;
  auto key_of = [&](int c) -> long long {
    const int j = it.k0 + c * kPmKeys + (whole ? 0 : lid & 15);
    return c < chunks && j < it.k1 ? pa_key(p, it, j) : -1;
  };
  auto issue = [&](int stage, long long off, int c) {
    const uint32_t base = ring + stage * C::kStage;
    const int valid = it.k1 - it.k0 - c * kPmKeys;      // keys of the chunk that exist
    if (whole && valid >= kPmKeys && off >= 0) {
      const uint8_t* ks = kp + off * 2 + lid * 16;
      const uint8_t* vs = vp + off * 2 + lid * 16;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int x = lid + 32 * i, key = x / D8, ch = x % D8;
        if (kPmKeys * D8 % 32 == 0 || x < kPmKeys * D8) {
          const uint32_t dst = base + key * C::kRow + ch * 16;
          cp_async16(dst, ks + i * 512, 16);
          cp_async16(dst + C::kTile, vs + i * 512, 16);
        }
      }
      return;
    }
#pragma unroll 1
    for (int i = 0; i < NP; ++i) {
      const int x = lid + 32 * i, key = x / D8, ch = x % D8;
      long long o = __shfl_sync(0xffffffffu, off, key & 15);
      if (whole && o >= 0) o += key * C::d;
      if (x < kPmKeys * D8) {
        const uint32_t n = o >= 0 && key < valid ? 16u : 0u;   // 0: filled with zeros (a masked V row must not hold NaN)
        const long long at = (n ? o : 0) * 2 + ch * 16;
        cp_async16(base + key * C::kRow + ch * 16, kp + at, n);
        cp_async16(base + C::kTile + key * C::kRow + ch * 16, vp + at, n);
      }
    }
  };

  long long off = key_of(w);
#pragma unroll
  for (int s = 0; s < kPmStages; ++s) {
    if (w + s * kPmWarps < chunks) issue(s, off, w + s * kPmWarps);
    cp_commit();
    off = key_of(w + (s + 1) * kPmWarps);
  }

  // Q as A fragments: rows r0 and r0 + 8, columns 16 ks + q2 + {0, 1} and + 8
  uint32_t qf[C::KS][4];
  {
    const long long oa = __shfl_sync(0xffffffffu, my_q, r0), ob = __shfl_sync(0xffffffffu, my_q, r0 + 8);
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q);
    const bool even = ((reinterpret_cast<uintptr_t>(p.q) & 3) | ((p.qsb | p.qst | p.qsh) & 1)) == 0;   // rows 4-byte aligned
    auto pair = [&](long long o, int c) -> uint32_t {
      if (o < 0 || c >= C::d) return 0u;
      const uint16_t* at = reinterpret_cast<const uint16_t*>(q + o + c);
      if (even) return *reinterpret_cast<const uint32_t*>(at);
      return at[0] | (uint32_t)at[1] << 16;
    };
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      qf[ks][0] = pair(oa, 16 * ks + q2);
      qf[ks][1] = kHalf ? 0u : pair(ob, 16 * ks + q2);
      qf[ks][2] = pair(oa, 16 * ks + q2 + 8);
      qf[ks][3] = kHalf ? 0u : pair(ob, 16 * ks + q2 + 8);
    }
  }
  const int seen_a = __shfl_sync(0xffffffffu, my_seen, r0), seen_b = __shfl_sync(0xffffffffu, my_seen, r0 + 8);
  constexpr int NE = kHalf ? 2 : 4;                     // accumulator elements of a tile in use: row r0 (, row r0 + 8)

  float o[D8][4];
#pragma unroll
  for (int n = 0; n < D8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  // matrix loads: lane l gives row l % 8 of matrix l / 8
  const uint32_t k_at = ((lid >> 4) * 8 + (lid & 7)) * C::kRow + ((lid >> 3) & 1) * 16;   // matrices: keys 0-7 (k, k+8), keys 8-15
  const uint32_t v_at = C::kTile + (((lid >> 3) & 1) * 8 + (lid & 7)) * C::kRow + (lid >> 4) * 16;

  int stage = 0;
#pragma unroll 1
  for (int c = w; c < chunks; c += kPmWarps) {
    cp_wait<kPmStages - 1>();
    __syncwarp();
    const uint32_t base = ring + stage * C::kStage;
    float s[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < C::KS; ++ks) {
      uint32_t b[4];
      ldsm4(base + k_at + ks * 32, b);
      mma_16816(s[0], qf[ks], b[0], b[1]);
      mma_16816(s[1], qf[ks], b[2], b[3]);
    }
    const int j0 = it.k0 + c * kPmKeys;
    float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) s[n][e] *= p.scale_log2;
    if (j0 + kPmKeys > all_see) {
      const int na = min(seen_a, it.k1) - j0 - q2, nb = min(seen_b, it.k1) - j0 - q2;   // keys from q2 on that the rows see
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < NE; ++e)
          if (8 * n + (e & 1) >= (e < 2 ? na : nb)) s[n][e] = -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) x[e >> 1] = fmaxf(x[e >> 1], s[n][e]);
#pragma unroll
    for (int k = 1; k < 4; k <<= 1)
#pragma unroll
      for (int h = 0; h < NE / 2; ++h) x[h] = fmaxf(x[h], __shfl_xor_sync(0xffffffffu, x[h], k));
    if (__any_sync(0xffffffffu, x[0] > m[0] || (!kHalf && x[1] > m[1]))) {
      float f[2];
#pragma unroll
      for (int h = 0; h < NE / 2; ++h) {
        const float mn = fmaxf(m[h], x[h]);
        f[h] = mn == -INFINITY ? 1.f : exp2f(m[h] - mn);
        m[h] = mn;
        l[h] *= f[h];
      }
#pragma unroll
      for (int n = 0; n < D8; ++n)
#pragma unroll
        for (int e = 0; e < NE; ++e) o[n][e] *= f[e >> 1];
    }
    float ref[2];
#pragma unroll
    for (int h = 0; h < NE / 2; ++h) ref[h] = m[h] == -INFINITY ? 0.f : m[h];   // no key seen yet: weights 0
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        s[n][e] = pa_ex2(s[n][e] - ref[e >> 1]);
        l[e >> 1] += s[n][e];
      }
    // the weights are rounded to bf16 for the product only (2^-9 relative, as the output's own rounding); l sums them unrounded
    const uint32_t pf[4] = {pm_pack(s[0][0], s[0][1]), kHalf ? 0u : pm_pack(s[0][2], s[0][3]), pm_pack(s[1][0], s[1][1]),
                            kHalf ? 0u : pm_pack(s[1][2], s[1][3])};
#pragma unroll
    for (int n = 0; n < C::KS; ++n) {
      uint32_t b[4];
      ldsm4_t(base + v_at + n * 32, b);
      mma_16816(o[2 * n], pf, b[0], b[1]);
      if (2 * n + 1 < D8) mma_16816(o[2 * n + 1 < D8 ? 2 * n + 1 : 0], pf, b[2], b[3]);
    }
    __syncwarp();                                       // all lanes have read the stage
    if (c + kPmStages * kPmWarps < chunks) issue(stage, off, c + kPmStages * kPmWarps);
    cp_commit();
    off = key_of(c + (kPmStages + 1) * kPmWarps);
    stage ^= 1;
  }
#pragma unroll
  for (int k = 1; k < 4; k <<= 1)
#pragma unroll
    for (int h = 0; h < 2; ++h) l[h] += __shfl_xor_sync(0xffffffffu, l[h], k);

  // ---- join the warps
  wait_previous();
  cp_wait<0>();
  __syncthreads();
  float* jn = reinterpret_cast<float*>(smem);
  {
    float* a = jn + (w * 16 + r0) * C::kJoinRow;
    float* b = a + 8 * C::kJoinRow;
    if (q2 == 0) {
      a[C::d] = m[0]; a[C::d + 1] = l[0];
      b[C::d] = m[1]; b[C::d + 1] = l[1];
    }
#pragma unroll
    for (int n = 0; n < D8; ++n) {
      *reinterpret_cast<float2*>(a + 8 * n + q2) = make_float2(o[n][0], o[n][1]);
      *reinterpret_cast<float2*>(b + 8 * n + q2) = make_float2(o[n][2], o[n][3]);
    }
  }
  __syncthreads();
  const long long* s_row = reinterpret_cast<const long long*>(smem + C::offRow);
  float4* s_f = reinterpret_cast<float4*>(smem + C::offRow + 16 * 8);   // the warps' factors of a row
  constexpr int NR = kHalf ? 8 : 16;
  if (tid < NR && s_row[tid] >= 0) {
    const float* a = jn + tid * C::kJoinRow + C::d;
    constexpr int ws = 16 * C::kJoinRow;
    const float m0 = a[0], m1 = a[ws], m2 = a[2 * ws], m3 = a[3 * ws];
    const float mx = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)), ref = mx == -INFINITY ? 0.f : mx;
    const float4 f = make_float4(pa_ex2(m0 - ref), pa_ex2(m1 - ref), pa_ex2(m2 - ref), pa_ex2(m3 - ref));
    s_f[tid] = f;
    const float sum = fmaf(f.x, a[1], fmaf(f.y, a[ws + 1], fmaf(f.z, a[2 * ws + 1], f.w * a[3 * ws + 1])));
    p.part_ml[(long long)it.slot * p.rows + s_row[tid]] = make_float2(mx, sum);
  }
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < NR * (C::d / 4); i += kPmWarps * 32) {
    const int r = i / (C::d / 4), c = (i % (C::d / 4)) * 4;
    const long long row = s_row[r];
    if (row < 0) break;                                 // rows are in order: none after this one either
    const float4 f = s_f[r];
    const float ff[4] = {f.x, f.y, f.z, f.w};
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < kPmWarps; ++x) {
      const float4 v = *reinterpret_cast<const float4*>(jn + (x * 16 + r) * C::kJoinRow + c);
      y.x = fmaf(ff[x], v.x, y.x); y.y = fmaf(ff[x], v.y, y.y); y.z = fmaf(ff[x], v.z, y.z); y.w = fmaf(ff[x], v.w, y.w);
    }
    *reinterpret_cast<float4*>(p.part_o + ((long long)it.slot * p.rows + row) * C::d + c) = y;
  }
}

template <int D8, bool kHalf>
static int launch_mma_h(const PaArgs& a, unsigned first, unsigned items, cudaStream_t s) {
  using C = PmCfg<D8>;
  static std::atomic<unsigned long long> done{0};
  if (!allow_smem(paged_attn_mma_kernel<D8, kHalf>, C::kSmem, done)) return HOA_ERR_LAUNCH;
  return launch_early(paged_attn_mma_kernel<D8, kHalf>, items, 1, kPmWarps * 32, C::kSmem, s, a, first);
}

template <int D8>
static int launch_mma(const PaArgs& a, unsigned first, unsigned items, cudaStream_t s) {
  // the rows of an item: of the whole batch where the launch has items of part 1
  const bool part1 = first < (unsigned)a.tiles1 * a.Hk * a.ns1;
  const long long rows = (part1 ? a.B : 1) * (long long)a.Tq * a.G;
  return rows <= 8 ? launch_mma_h<D8, true>(a, first, items, s) : launch_mma_h<D8, false>(a, first, items, s);
}

int paged_attn_mma(const PaArgs& a, unsigned first, unsigned items, cudaStream_t s) {
  switch (a.d / 8) {
    case 1: return launch_mma<1>(a, first, items, s);
    case 2: return launch_mma<2>(a, first, items, s);
    case 3: return launch_mma<3>(a, first, items, s);
    case 4: return launch_mma<4>(a, first, items, s);
    case 5: return launch_mma<5>(a, first, items, s);
    case 6: return launch_mma<6>(a, first, items, s);
    case 7: return launch_mma<7>(a, first, items, s);
    case 8: return launch_mma<8>(a, first, items, s);
    case 9: return launch_mma<9>(a, first, items, s);
    case 10: return launch_mma<10>(a, first, items, s);
    case 11: return launch_mma<11>(a, first, items, s);
    case 12: return launch_mma<12>(a, first, items, s);
    case 13: return launch_mma<13>(a, first, items, s);
    case 14: return launch_mma<14>(a, first, items, s);
    case 15: return launch_mma<15>(a, first, items, s);
    case 16: return launch_mma<16>(a, first, items, s);
    default: return HOA_ERR_UNSUPPORTED;
  }
}

}  // namespace hoa
