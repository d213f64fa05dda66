// Pages of the generation cache: reserving, writing, copying, forking, freeing
// and compacting.  No counterpart in the reference, which keeps no cache: k^ and
// v^ are stored in the gauge of their sequence's origin (k^_t = P_t^T k_t), so
// they never change as the sequence grows and a fork shares its parent's pages.
//
// Bookkeeping (int32, on the device):
//   table (S, W)   page ids of each row (sequence) in order, -1 beyond its last
//   lens  (S)      tokens of each row; row s uses ceil(lens[s] / page) entries
//   refs  (n_pages) rows that hold each page; a page is free when refs == 0
// Every operation reads one state and writes the next one to other buffers, so
// the caller's old state stays valid; payload moves only into pages that are
// free in the old state.  Free pages are taken lowest index first and ranks
// follow the order of the request list, so results do not depend on timing.
//
// One cluster of 8 CTAs does the bookkeeping of an operation in one launch: the
// state is small (four bytes a page and a table entry) and its phases (count,
// rank, assign) depend on one another, so what bounds it is the latency of two
// or three cluster barriers, not bytes.  The payload is copied by a second
// launch over (pair of pages, pool, 32 KB chunk) units, bound by HBM.
#include <cooperative_groups.h>

#include "hoa_common.cuh"

namespace hoa {
namespace cg = cooperative_groups;

// (64 forks over a table of 25600 entries / 4 over 64: 128 threads a CTA 21.2 / 7.3 us, 256 18.5 / 7.6, 512 18.6 / 9.0, each
// with the payload; one CTA of 1024 instead of the cluster 24.0 / 8.5)
constexpr int kPgCluster = 8, kPgThreads = 256, kPgWarps = kPgThreads / 32;
constexpr int kPgMaxRows = 65536;          // rows of a table (a bitmap of them is 8 KB)

struct PgState {                           // one bookkeeping state
  const int* table; const int* lens; const int* refs;
  int* table_out; int* lens_out; int* refs_out;
  int S, W, n_pages, page;
};

HOA_DEVICE void pg_fail(int* status) {
  if (status != nullptr) *reinterpret_cast<volatile int*>(status) = HOA_ERR_PAGES;
}

HOA_DEVICE int pg_used(int len, int page) { return (int)(((long long)len + page - 1) / page); }

// dst[i] = src[i], i < n, by all threads of the cluster; 16 bytes at a time where both allow it
HOA_DEVICE void pg_copy(const int* __restrict__ src, int* __restrict__ dst, long long n, int gt) {
  constexpr int NT = kPgCluster * kPgThreads;
  if (((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) & 15) == 0) {
    const long long n4 = n >> 2;
    const int4* s4 = reinterpret_cast<const int4*>(src);
    int4* d4 = reinterpret_cast<int4*>(dst);
#pragma unroll 4
    for (long long i = gt; i < n4; i += NT) d4[i] = s4[i];
    for (long long i = (n4 << 2) + gt; i < n; i += NT) dst[i] = src[i];
  } else {
    for (long long i = gt; i < n; i += NT) dst[i] = src[i];
  }
}

// Exclusive rank of `flag` (0 / 1 or a count) among the block's threads and the block's total.
HOA_DEVICE int pg_block_rank(int v, int* total, int* s_warp) {
  const int lid = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lid >= o) x += y;
  }
  if (lid == 31) s_warp[w] = x;
  __syncthreads();
  int base = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kPgWarps; ++i) {
    const int c = s_warp[i];
    base += i < w ? c : 0;
    sum += c;
  }
  __syncthreads();
  *total = sum;
  return base + x - v;
}

// This CTA's slice of the pages.
struct PgSlice { int lo, hi; };
HOA_DEVICE PgSlice pg_slice(int n_pages, int rank) {
  const int per = (n_pages + kPgCluster - 1) / kPgCluster;
  return {min(rank * per, n_pages), min((rank + 1) * per, n_pages)};
}

// Pages of the slice for which pred(page) holds, counted.
template <class Pred>
HOA_DEVICE int pg_count(PgSlice s, Pred pred) {
  int c = 0;
  for (int i0 = s.lo; i0 < s.hi; i0 += kPgThreads) {
    const int i = i0 + (int)threadIdx.x;
    c += __syncthreads_count(i < s.hi && pred(i));
  }
  return c;
}

// The same pages written to out[base ..] in ascending order, up to out[limit - 1].
template <class Pred>
HOA_DEVICE void pg_list(PgSlice s, Pred pred, int base, int limit, int* out, int* s_warp) {
  for (int i0 = s.lo; i0 < s.hi && base < limit; i0 += kPgThreads) {
    const int i = i0 + (int)threadIdx.x;
    const bool on = i < s.hi && pred(i);
    int total;
    const int r = base + pg_block_rank(on ? 1 : 0, &total, s_warp);
    if (on && r < limit) out[r] = i;
    base += total;
  }
}

// ---------------------------------------------------------------------------
// payload: page to[i] of every pool = page from[i]
// ---------------------------------------------------------------------------
constexpr int kCpThreads = 256, kCpVecs = 8;       // 16-byte vectors a thread has in flight
constexpr int kMaxPools = 32;

struct PgCopyArgs {
  uint8_t* base[kMaxPools];
  long long stride[kMaxPools];   // bytes between pages
  long long bytes[kMaxPools];    // bytes of a page
  const int* from; const int* to;
  const int* count;              // device count of pairs (nullptr: n)
  int n, n_pages, pools, chunks; // chunks: of the largest page
  int* status;
};

// One unit: kThreads * kCpVecs vectors of one page of one pool, by kThreads threads of which this is number t.
template <class V, int kThreads>
HOA_DEVICE void pg_copy_unit(const PgCopyArgs& p, long long u, int t) {
  const int c = (int)(u % p.chunks);
  const long long r = u / p.chunks;
  const int pool = (int)(r % p.pools), i = (int)(r / p.pools);
  const int a = p.from[i], b = p.to[i];
  if (a < 0 && b < 0) return;                      // no copy for this pair
  if (a < 0 || b < 0 || a >= p.n_pages || b >= p.n_pages) {
    if (t == 0) pg_fail(p.status);
    return;
  }
  const V* src = reinterpret_cast<const V*>(p.base[pool] + a * p.stride[pool]);
  V* dst = reinterpret_cast<V*>(p.base[pool] + b * p.stride[pool]);
  const long long nv = p.bytes[pool] / (long long)sizeof(V);
  const long long v0 = (long long)c * (kThreads * kCpVecs) + t;
  V buf[kCpVecs];
#pragma unroll
  for (int k = 0; k < kCpVecs; ++k)
    if (v0 + k * kThreads < nv) buf[k] = src[v0 + k * kThreads];
#pragma unroll
  for (int k = 0; k < kCpVecs; ++k)
    if (v0 + k * kThreads < nv) dst[v0 + k * kThreads] = buf[k];
}

// A payload of up to kCpInline bytes is copied by the bookkeeping cluster itself (16-byte vectors, a warp a 4 KB
// unit), which spares the second launch: a fork with four pages of 12 KB in two pools takes 20 us with its host side
// against 23.  Beyond a megabyte eight CTAs take longer than the launch that they spare.
constexpr long long kCpInline = 1 << 20;
HOA_DEVICE void pg_copy_inline(const PgCopyArgs& p, int n, int warp, int warps) {
  const long long units = (long long)n * p.pools * p.chunks;
  for (long long u = warp; u < units; u += warps) pg_copy_unit<uint4, 32>(p, u, threadIdx.x & 31);
}

// ---------------------------------------------------------------------------
// reserve: row s grows by counts[s] tokens (new pages where they cross one);
// fork: row dst[i] becomes a copy of row src[i] that shares its full pages and
// has its own copy of a last page that is not full.
// All or nothing: without enough free pages, or with an invalid request, the
// new state equals the old one and the status word says so.
// ---------------------------------------------------------------------------
struct PgTakeArgs {
  PgState st;
  const int* a;          // reserve: counts (S); fork: src (n)
  const int* b;          // fork: dst (n)
  int n;                 // requests (reserve: S)
  int* rank;             // (n) scratch: first fresh page of a request
  int* fresh;            // (n_pages) scratch: the free pages taken, in order
  int* from; int* to;    // (n) fork: the page copies (-1: none)
  int* status;
};

template <bool kFork>
__global__ void __launch_bounds__(kPgThreads)
pages_take_kernel(PgTakeArgs p, const __grid_constant__ PgCopyArgs cp) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ int s_warp[kPgWarps];
  __shared__ int s_free, s_need, s_bad;
  __shared__ unsigned s_seen[kFork ? kPgMaxRows / 32 : 1];
  const int rank = (int)cl.block_rank(), tid = threadIdx.x, gt = rank * kPgThreads + tid;
  wait_previous();
  let_next_start();                        // (the payload's launch, which waits for this one to complete)
  const PgState& st = p.st;
  const int page = st.page, W = st.W, S = st.S;
  pg_copy(st.table, st.table_out, (long long)S * W, gt);
  pg_copy(st.lens, st.lens_out, S, gt);
  pg_copy(st.refs, st.refs_out, st.n_pages, gt);
  const PgSlice sl = pg_slice(st.n_pages, rank);
  const int* refs = st.refs;
  auto is_free = [refs](int i) { return refs[i] == 0; };
  const int mine = pg_count(sl, is_free);
  if (tid == 0) { s_free = mine; s_need = 0; s_bad = 0; }
  __syncthreads();
  if (rank == kPgCluster - 1) {            // (the last slice is the shortest)
    if (kFork) {
      for (int i = tid; i < kPgMaxRows / 32; i += kPgThreads) s_seen[i] = 0;
      __syncthreads();
    }
    int base = 0;
    for (int i0 = 0; i0 < p.n; i0 += kPgThreads) {
      const int i = i0 + tid;
      int need = 0;
      bool bad = false;
      if (i < p.n) {
        if (kFork) {
          const int a = p.a[i], b = p.b[i];
          bad = a < 0 || a >= S || b < 0 || b >= S || a == b;
          if (!bad) {
            const int len = st.lens[a];
            bad = len < 0 || (long long)len > (long long)W * page || st.lens[b] != 0 ||
                  (atomicOr(&s_seen[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1u;
            need = !bad && len % page != 0 ? 1 : 0;
          }
        } else {
          const int len = st.lens[i], c = p.a[i];
          // (lengths are ints: a row may have room for more tokens than one counts)
          bad = len < 0 || c < 0 || (long long)len + c > min((long long)W * page, 0x7fffffffll);
          if (!bad) need = pg_used(len + c, page) - pg_used(len, page);
        }
      }
      int total;
      const int r = base + pg_block_rank(need, &total, s_warp);
      if (i < p.n) p.rank[i] = r;
      if (__syncthreads_or(bad) && tid == 0) s_bad = 1;
      // (a sum beyond the pool fails below; it is held at the pool's size + 1)
      base = min(base + min(total, st.n_pages + 1), st.n_pages + 1);
    }
    if (tid == 0) s_need = base;
  }
  cl.sync();
  int before = 0, all = 0;
#pragma unroll
  for (int r = 0; r < kPgCluster; ++r) {
    const int c = *cl.map_shared_rank(&s_free, r);
    before += r < rank ? c : 0;
    all += c;
  }
  const int need = *cl.map_shared_rank(&s_need, kPgCluster - 1);
  const bool fail = *cl.map_shared_rank(&s_bad, kPgCluster - 1) != 0 || need > all;
  if (!fail) pg_list(sl, is_free, before, need, p.fresh, s_warp);
  cl.sync();                               // fresh, rank and the copies are visible; no CTA leaves before its shared memory was read
  const int lid = tid & 31;
  if (fail) {
    if (gt == 0) pg_fail(p.status);
    if (kFork)
      for (int i = gt; i < p.n; i += kPgCluster * kPgThreads) { p.from[i] = -1; p.to[i] = -1; }
    return;
  }
  for (int i = gt >> 5; i < p.n; i += kPgCluster * kPgWarps) {     // a warp per request
    if (kFork) {
      const int a = p.a[i], b = p.b[i], len = st.lens[a], full = len / page;
      const int* src = st.table + (long long)a * W;
      int* dst = st.table_out + (long long)b * W;
      const bool part = len % page != 0;
      bool bad = false;
      for (int j = lid; j < W; j += 32) {
        int id = -1;
        if (j < full) {
          id = src[j];
          if (id >= 0 && id < st.n_pages) atomicAdd(&st.refs_out[id], 1);
          else bad = true;
        } else if (j == full && part) {
          id = p.fresh[p.rank[i]];
          st.refs_out[id] = 1;
          const int old = src[j];
          const bool ok = old >= 0 && old < st.n_pages;
          p.from[i] = ok ? old : -1;
          p.to[i] = ok ? id : -1;
          bad |= !ok;
        }
        dst[j] = id;
      }
      if (bad) pg_fail(p.status);
      if (lid == 0) {
        st.lens_out[b] = len;
        if (!part) { p.from[i] = -1; p.to[i] = -1; }
      }
    } else {
      const int len = st.lens[i], c = p.a[i], u0 = pg_used(len, page), u1 = pg_used(len + c, page);
      int* dst = st.table_out + (long long)i * W;
      for (int j = u0 + lid; j < u1; j += 32) {
        const int id = p.fresh[p.rank[i] + j - u0];
        st.refs_out[id] = 1;
        dst[j] = id;
      }
      if (lid == 0) st.lens_out[i] = len + c;
    }
  }
  if (kFork && cp.n > 0) {                 // a small payload
    cl.sync();
    pg_copy_inline(cp, cp.n, gt >> 5, kPgCluster * kPgWarps);
  }
}

// ---------------------------------------------------------------------------
// free: the rows end; a page that no row holds any more becomes free
// ---------------------------------------------------------------------------
struct PgFreeArgs { PgState st; const int* rows; int n; int* status; };

__global__ void __launch_bounds__(kPgThreads) pages_free_kernel(PgFreeArgs p) {
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, gt = (int)cl.block_rank() * kPgThreads + tid, lid = tid & 31;
  wait_previous();
  const PgState& st = p.st;
  const int W = st.W;
  pg_copy(st.table, st.table_out, (long long)st.S * W, gt);
  pg_copy(st.lens, st.lens_out, st.S, gt);
  pg_copy(st.refs, st.refs_out, st.n_pages, gt);
  cl.sync();
  for (int i = gt >> 5; i < p.n; i += kPgCluster * kPgWarps) {
    const int row = p.rows[i];
    if (row < 0 || row >= st.S) {
      if (lid == 0) pg_fail(p.status);
      continue;
    }
    // a row that is listed twice is freed once: the first to come takes its length
    int len = 0;
    if (lid == 0) len = atomicExch(&st.lens_out[row], 0);
    len = __shfl_sync(0xffffffffu, len, 0);
    const int used = min(len > 0 ? pg_used(len, st.page) : 0, W);
    const int* src = st.table + (long long)row * W;
    int* dst = st.table_out + (long long)row * W;
    for (int j = lid; j < W; j += 32) {
      if (j < used) {
        const int id = src[j];
        if (id < 0 || id >= st.n_pages) {
          pg_fail(p.status);
        } else if (atomicSub(&st.refs_out[id], 1) <= 0) {
          // a page that its row does not own, by a table that was made wrongly: it stays as it was, at 0 (each of those that
          // come too late adds what it took, so the sum does not depend on their order)
          atomicAdd(&st.refs_out[id], 1);
          pg_fail(p.status);
        }
      }
      dst[j] = -1;
    }
  }
}

// ---------------------------------------------------------------------------
// compact: the L live pages move to 0 .. L-1 (the i-th hole below L takes the
// i-th live page at or above L, both ascending), the table follows
// ---------------------------------------------------------------------------
struct PgCompactArgs {
  PgState st;            // lens unused
  int* live;             // L
  int* remap;            // (n_pages) scratch: new place of a page that moves
  int* from; int* to;    // (n_pages) scratch, the moves
  int* moves;            // their number
  int* status;
};

__global__ void __launch_bounds__(kPgThreads)
pages_compact_kernel(PgCompactArgs p, const __grid_constant__ PgCopyArgs cp) {
  cg::cluster_group cl = cg::this_cluster();
  __shared__ int s_warp[kPgWarps];
  __shared__ int s_live, s_hole, s_move;
  const int rank = (int)cl.block_rank(), tid = threadIdx.x, gt = rank * kPgThreads + tid;
  wait_previous();
  let_next_start();                        // (the payload's launch, which waits for this one to complete)
  constexpr int NT = kPgCluster * kPgThreads;
  const PgState& st = p.st;
  const int* refs = st.refs;
  const PgSlice sl = pg_slice(st.n_pages, rank);
  const int mine = pg_count(sl, [refs](int i) { return refs[i] > 0; });
  if (tid == 0) s_live = mine;
  cl.sync();
  int live = 0;
#pragma unroll
  for (int r = 0; r < kPgCluster; ++r) live += *cl.map_shared_rank(&s_live, r);
  auto hole = [refs, live](int i) { return i < live && refs[i] <= 0; };
  auto mover = [refs, live](int i) { return i >= live && refs[i] > 0; };
  const int holes = pg_count(sl, hole), movers = pg_count(sl, mover);
  if (tid == 0) { s_hole = holes; s_move = movers; }
  cl.sync();
  int hb = 0, mb = 0, moves = 0;
#pragma unroll
  for (int r = 0; r < kPgCluster; ++r) {
    const int h = *cl.map_shared_rank(&s_hole, r), m = *cl.map_shared_rank(&s_move, r);
    hb += r < rank ? h : 0;
    mb += r < rank ? m : 0;
    moves += m;
  }
  pg_list(sl, hole, hb, st.n_pages, p.to, s_warp);
  pg_list(sl, mover, mb, st.n_pages, p.from, s_warp);
  if (gt == 0) { *p.live = live; *p.moves = moves; }
  cl.sync();                               // the lists are visible; shared memory has been read
  for (int i = gt; i < moves; i += NT) {
    const int a = p.from[i], b = p.to[i];
    p.remap[a] = b;
    st.refs_out[b] = refs[a];
  }
  for (int i = gt; i < st.n_pages; i += NT)
    if (i >= live || refs[i] > 0) st.refs_out[i] = i < live ? refs[i] : 0;
  cl.sync();
  const long long n = (long long)st.S * st.W;
  for (long long i = gt; i < n; i += NT) {
    int id = st.table[i];
    if (id >= live) {
      // an entry that no row counts, or outside the pool: a table that was made wrongly
      if (id < st.n_pages && refs[id] > 0) id = p.remap[id];
      else { pg_fail(p.status); id = -1; }
    }
    st.table_out[i] = id;
  }
  if (cp.n > 0) pg_copy_inline(cp, min(moves, cp.n), gt >> 5, kPgCluster * kPgWarps);   // a small payload
}

// The copy as a launch of its own, bound by HBM: 894 pages of 196 KB in each of two pools (703 MB read and written) 110 us,
// 6.4 TB/s, the rate of a plain copy.
template <class V>
__global__ void __launch_bounds__(kCpThreads) pages_copy_kernel(const __grid_constant__ PgCopyArgs p) {
  wait_previous();
  const int n = p.count != nullptr ? min(*p.count, p.n) : p.n;
  const long long units = (long long)n * p.pools * p.chunks;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) pg_copy_unit<V, kCpThreads>(p, u, threadIdx.x);
}

template <class V>
static int launch_copy(PgCopyArgs a, long long most, cudaStream_t s) {
  a.chunks = (int)((most / (long long)sizeof(V) + kCpThreads * kCpVecs - 1) / (kCpThreads * kCpVecs));
  if (a.chunks < 1) a.chunks = 1;
  const long long units = (long long)a.n * a.pools * a.chunks;
  return launch_early(pages_copy_kernel<V>, (unsigned)(units < 148 * 8 ? units : 148 * 8), 1, kCpThreads, 0, s, a);
}

struct PgPools { void* const* base; const long long* stride; const long long* bytes; int n; };

// The copy of up to kMaxPools pools from number k0 on; `bits`: alignment of everything it touches, `most`: bytes of its
// largest page.
static PgCopyArgs copy_args(const PgPools& q, int k0, const int* from, const int* to, const int* count, int n, int n_pages,
                            int* status, unsigned long long* bits, long long* most) {
  PgCopyArgs a{};
  a.pools = q.n - k0 < kMaxPools ? q.n - k0 : kMaxPools;
  a.from = from; a.to = to; a.count = count; a.n = n; a.n_pages = n_pages; a.status = status;
  *bits = 0;
  *most = 0;
  for (int k = 0; k < a.pools; ++k) {
    a.base[k] = static_cast<uint8_t*>(q.base[k0 + k]);
    a.stride[k] = q.stride[k0 + k];
    a.bytes[k] = q.bytes[k0 + k];
    *bits |= (unsigned long long)reinterpret_cast<uintptr_t>(a.base[k]) | (unsigned long long)a.stride[k] |
             (unsigned long long)a.bytes[k];
    if (a.bytes[k] > *most) *most = a.bytes[k];
  }
  return a;
}

// The copy for the bookkeeping kernel itself, or one with n = 0: small, in 16-byte vectors, one set of pools.
static PgCopyArgs inline_copy(const PgPools& q, const int* from, const int* to, int n, int n_pages, int* status) {
  unsigned long long bits;
  long long most, all = 0;
  if (q.n == 0 || q.n > kMaxPools || n == 0) return PgCopyArgs{};
  PgCopyArgs a = copy_args(q, 0, from, to, nullptr, n, n_pages, status, &bits, &most);
  for (int k = 0; k < a.pools; ++k) all += a.bytes[k] * n;
  if ((bits & 15) != 0 || all > kCpInline) return PgCopyArgs{};
  a.chunks = (int)((most / 16 + 32 * kCpVecs - 1) / (32 * kCpVecs));
  return a;
}

static int copy_pools(const PgPools& q, const int* from, const int* to, const int* count, int n, int n_pages, int* status,
                      cudaStream_t s) {
  if (n == 0) return HOA_OK;
  for (int k0 = 0; k0 < q.n; k0 += kMaxPools) {
    unsigned long long bits;
    long long most;
    const PgCopyArgs a = copy_args(q, k0, from, to, count, n, n_pages, status, &bits, &most);
    const int st = (bits & 15) == 0 ? launch_copy<uint4>(a, most, s)
                 : (bits & 3) == 0 ? launch_copy<uint32_t>(a, most, s)
                 : (bits & 1) == 0 ? launch_copy<uint16_t>(a, most, s) : launch_copy<uint8_t>(a, most, s);
    if (st != HOA_OK) return st;
  }
  return HOA_OK;
}

// ---------------------------------------------------------------------------
// write: the last T tokens of each row, k and v (B, T, H, d), into their slots
// ---------------------------------------------------------------------------
struct PgWriteArgs {
  const void* k; const void* v;
  long long ksb, kst, ksh, vsb, vst, vsh;          // element strides of row, token, head
  void* kp; void* vp;
  long long ps, hs, ts;                            // element strides of page, head, token (both pools)
  const int* table; long long tw; const int* lens;
  int B, T, H, d, page, W, n_pages, src_dtype, dtype;
  int* status;
};

__global__ void __launch_bounds__(256) pages_write_kernel(PgWriteArgs p) {
  wait_previous();
  const long long rows = (long long)p.B * p.T * p.H;
  const int lid = threadIdx.x & 31;
  for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (long long)gridDim.x * 8) {
    const int h = (int)(r % p.H), t = (int)((r / p.H) % p.T), b = (int)(r / ((long long)p.H * p.T));
    const int pos = p.lens[b] - p.T + t;
    if (pos < 0) continue;                         // a row shorter than T tokens: the first ones are not its
    const int j = pos / p.page;
    const int id = j < p.W ? p.table[(long long)b * p.tw + j] : -1;
    if (id < 0 || id >= p.n_pages) {
      if (lid == 0) pg_fail(p.status);
      continue;
    }
    const long long o = id * p.ps + h * p.hs + (long long)(pos % p.page) * p.ts;
    const long long ko = b * p.ksb + t * p.kst + h * p.ksh, vo = b * p.vsb + t * p.vst + h * p.vsh;
    for (int e = lid; e < p.d; e += 32) {
      store_elem(p.kp, o + e, p.dtype, load_elem(p.k, ko + e, p.src_dtype));
      store_elem(p.vp, o + e, p.dtype, load_elem(p.v, vo + e, p.src_dtype));
    }
  }
}

// The loops over pages and requests count past the last one, by up to a cluster's threads, with an int.
constexpr int kPgMost = 0x7fff0000;

static bool pg_state_ok(const int* table, const int* lens, const int* refs, const int* t2, const int* l2,
                        const int* r2, int S, int W, int n_pages, int page) {
  return table && lens && refs && t2 && l2 && r2 && table != t2 && lens != l2 && refs != r2 && S >= 1 && W >= 1 &&
         n_pages >= 1 && page >= 1 && (long long)S * W < 0x7fffffffll;
}

}  // namespace hoa

using namespace hoa;

extern "C" size_t hoa_pages_workspace_bytes(int n, int n_pages) {
  if (n < 0 || n_pages < 1) return 0;
  // requests: rank, from, to; pages: fresh (take) or remap, from, to (compact); one count
  const size_t take = 3 * (size_t)n + (size_t)n_pages, comp = 3 * (size_t)n_pages;
  return 4 * ((take > comp ? take : comp) + 4);
}

extern "C" int hoa_pages_reserve(const int* table, const int* lens, const int* refs, const int* counts, int* table_out,
                                 int* lens_out, int* refs_out, int S, int W, int n_pages, int page, void* workspace,
                                 size_t workspace_bytes, int* status, void* stream) {
  if (!pg_state_ok(table, lens, refs, table_out, lens_out, refs_out, S, W, n_pages, page) || !counts || !workspace)
    return HOA_ERR_INVALID_ARG;
  if (S > kPgMaxRows || n_pages > kPgMost) return HOA_ERR_UNSUPPORTED;
  if (workspace_bytes < hoa_pages_workspace_bytes(S, n_pages)) return HOA_ERR_WORKSPACE;
  int* ws = static_cast<int*>(workspace);
  PgTakeArgs a{{table, lens, refs, table_out, lens_out, refs_out, S, W, n_pages, page},
               counts, nullptr, S, ws, ws + S, nullptr, nullptr, status};
  return launch_early(pages_take_kernel<false>, kPgCluster, kPgCluster, kPgThreads, 0, reinterpret_cast<cudaStream_t>(stream), a,
                      PgCopyArgs{});
}

extern "C" int hoa_pages_fork(const int* table, const int* lens, const int* refs, const int* src, const int* dst, int n,
                              int* table_out, int* lens_out, int* refs_out, int S, int W, int n_pages, int page,
                              void* const* pools, const long long* strides, const long long* bytes, int n_pools,
                              void* workspace, size_t workspace_bytes, int* status, void* stream) {
  if (!pg_state_ok(table, lens, refs, table_out, lens_out, refs_out, S, W, n_pages, page) || n < 0 || n_pools < 0 ||
      (n > 0 && (!src || !dst)) || (n_pools > 0 && (!pools || !strides || !bytes)) || !workspace)
    return HOA_ERR_INVALID_ARG;
  if (S > kPgMaxRows || n > S || n_pages > kPgMost) return HOA_ERR_UNSUPPORTED;
  if (workspace_bytes < hoa_pages_workspace_bytes(n, n_pages)) return HOA_ERR_WORKSPACE;
  int* ws = static_cast<int*>(workspace);
  int *from = ws + n, *to = ws + 2 * (size_t)n;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  PgTakeArgs a{{table, lens, refs, table_out, lens_out, refs_out, S, W, n_pages, page},
               src, dst, n, ws, ws + 3 * (size_t)n, from, to, status};
  const PgPools q{pools, strides, bytes, n_pools};
  const PgCopyArgs cp = inline_copy(q, from, to, n, n_pages, status);
  const int st = launch_early(pages_take_kernel<true>, kPgCluster, kPgCluster, kPgThreads, 0, s, a, cp);
  if (st != HOA_OK || cp.n > 0) return st;
  return copy_pools(q, from, to, nullptr, n, n_pages, status, s);
}

extern "C" int hoa_pages_free(const int* table, const int* lens, const int* refs, const int* rows, int n, int* table_out,
                              int* lens_out, int* refs_out, int S, int W, int n_pages, int page, int* status,
                              void* stream) {
  if (!pg_state_ok(table, lens, refs, table_out, lens_out, refs_out, S, W, n_pages, page) || n < 0 || (n > 0 && !rows))
    return HOA_ERR_INVALID_ARG;
  if (S > kPgMaxRows || n > kPgMost || n_pages > kPgMost) return HOA_ERR_UNSUPPORTED;
  PgFreeArgs a{{table, lens, refs, table_out, lens_out, refs_out, S, W, n_pages, page}, rows, n, status};
  return launch_early(pages_free_kernel, kPgCluster, kPgCluster, kPgThreads, 0, reinterpret_cast<cudaStream_t>(stream), a);
}

extern "C" int hoa_pages_compact(const int* table, const int* refs, int* table_out, int* refs_out, int* live, int S, int W,
                                 int n_pages, void* const* pools, const long long* strides, const long long* bytes,
                                 int n_pools, void* workspace, size_t workspace_bytes, int* status, void* stream) {
  if (!pg_state_ok(table, table, refs, table_out, table_out, refs_out, S, W, n_pages, 1) || !live || n_pools < 0 ||
      (n_pools > 0 && (!pools || !strides || !bytes)) || !workspace)
    return HOA_ERR_INVALID_ARG;
  if (S > kPgMaxRows || n_pages > kPgMost) return HOA_ERR_UNSUPPORTED;
  if (workspace_bytes < hoa_pages_workspace_bytes(0, n_pages)) return HOA_ERR_WORKSPACE;
  int* ws = static_cast<int*>(workspace);
  int *from = ws, *to = ws + n_pages, *remap = ws + 2 * (size_t)n_pages, *moves = ws + 3 * (size_t)n_pages;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  PgCompactArgs a{{table, nullptr, refs, table_out, nullptr, refs_out, S, W, n_pages, 1}, live, remap, from, to, moves, status};
  // at most half of the pages move: a mover needs a hole below it
  const PgPools q{pools, strides, bytes, n_pools};
  const PgCopyArgs cp = inline_copy(q, from, to, n_pages / 2, n_pages, status);
  const int st = launch_early(pages_compact_kernel, kPgCluster, kPgCluster, kPgThreads, 0, s, a, cp);
  if (st != HOA_OK || cp.n > 0) return st;
  return copy_pools(q, from, to, moves, n_pages / 2, n_pages, status, s);
}

extern "C" int hoa_pages_copy(void* const* pools, const long long* strides, const long long* bytes, int n_pools,
                              const int* from, const int* to, int n, int n_pages, int* status, void* stream) {
  if (n < 0 || n_pools < 0 || n_pages < 1 || (n > 0 && (!from || !to)) || (n_pools > 0 && (!pools || !strides || !bytes)))
    return HOA_ERR_INVALID_ARG;
  return copy_pools(PgPools{pools, strides, bytes, n_pools}, from, to, nullptr, n, n_pages, status,
                    reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int hoa_pages_write(const void* k, const void* v, int src_dtype, const long long* k_strides,
                               const long long* v_strides, void* k_pages, void* v_pages, int dtype,
                               const long long* page_strides, const int* table, long long table_stride, const int* lens,
                               int B, int T, int H, int d, int page, int W, int n_pages, int* status, void* stream) {
  if (!k || !v || !k_strides || !v_strides || !k_pages || !v_pages || !page_strides || !table || !lens || B < 1 ||
      T < 1 || H < 1 || d < 1 || page < 1 || W < 1 || n_pages < 1)
    return HOA_ERR_INVALID_ARG;
  if ((src_dtype != HOA_F32 && src_dtype != HOA_BF16) || (dtype != HOA_F32 && dtype != HOA_BF16)) return HOA_ERR_UNSUPPORTED;
  PgWriteArgs a{k, v, k_strides[0], k_strides[1], k_strides[2], v_strides[0], v_strides[1], v_strides[2],
                k_pages, v_pages, page_strides[0], page_strides[1], page_strides[2], table, table_stride, lens,
                B, T, H, d, page, W, n_pages, src_dtype, dtype, status};
  const long long blocks = ((long long)B * T * H + 7) / 8;
  return launch_early(pages_write_kernel, (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 1, 256, 0,
                      reinterpret_cast<cudaStream_t>(stream), a);
}
