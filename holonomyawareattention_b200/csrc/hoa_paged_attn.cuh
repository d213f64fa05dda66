// Work items of the paged attention, shared by its kernels.
//
// An item is (part, kv head, tile of query rows, split of the keys).  Part 1: the
// shared pages; its rows are (b, t, g) over the whole batch, g the query heads of
// the kv head.  Part 2: a row's own pages; its rows are (t, g) of that row.
#pragma once

#include "hoa_common.cuh"

namespace hoa {

struct PaArgs {
  const void* q; long long qsb, qst, qsh;          // element strides of row, token, head
  const void* kp; const void* vp; long long ps, hs, ts;   // element strides of page, head, token
  const int* shared; int n_shared;
  const int* table; long long tstride; int W;
  const int* lens;
  const float* paths;                              // (B, H, d, d) or nullptr
  void* out; int out_dtype; float* lse;            // (B, Tq, H, d), (B, Tq, H)
  float* part_o; float2* part_ml;                  // (slots, rows, d) unnormalised; (slots, rows) (m, l), l = 0: no key
  float* o;                                        // (rows, d) fp32: o before its transport (Tq = 1)
  long long rows;                                  // B * Tq * H
  float scale_log2;
  int dtype, B, Tq, H, Hk, G, d, page, n_pages;
  unsigned page_mul; int page_shift;               // j / page = umulhi(j, page_mul) >> page_shift for 0 <= j < 2^31 (page > 1)
  int tiles1, ns1, tiles2, ns2;
  int leads, more;                                 // this launch is the first of the call; the join: the transport follows
  int* status;
};

struct PaItem {
  int part, kvh, b, row0, slot;
  int k0, k1;                                      // keys of this part [k0, k1)
  int key_base;                                    // position of the part's key 0
};

struct PaRow { bool ok; int b, t, h, seen; long long grow; };

HOA_DEVICE float pa_ex2(float x) {     // 2^x, results below 2^-126 flushed to 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

HOA_DEVICE void pa_fail(int* status) {
  if (status != nullptr) *reinterpret_cast<volatile int*>(status) = HOA_ERR_PAGES;
}

// Keys of a tensor-core tile: whole pages, or whole tiles of a page, of at most 128 keys in
// multiples of 16 (a product's k-step); 0 where no such tile exists (pages of 25, say).
inline int pa_tile_keys(int page) {
  if (page % 8 != 0) return 0;                     // the swizzle pattern repeats every 8 rows
  if (page <= 128) {
    int kt = 128 / page * page;
    while (kt > 0 && kt % 16 != 0) kt -= page;
    return kt;
  }
  for (int kt = 128; kt > 0; kt -= 16)
    if (page % kt == 0) return kt;
  return 0;
}

// Which kernel takes a part.
//   vec:  fp32 with 16-byte rows, up to 4 rows a head (1, 2 or 4 a tile).
//   simt: fp32, head dims or strides that the copies do not take; 16 rows a tile, 32 where there are more.
//   mma:  bf16, 16 rows a tile, any page size.
//   tc:   bf16, pages that tile (pa_tile_keys); 256 rows a tile, or 128 where a head has no more.
enum PaKind { kPaVec1, kPaVec2, kPaVec4, kPaSimt, kPaSimt32, kPaMma, kPaTc128, kPaTc };
inline bool pa_is_tc(int kind) { return kind >= kPaTc128; }
inline int pa_tile_rows(int kind) {
  const int rows[] = {1, 2, 4, 16, 32, 16, 128, 256};
  return rows[kind];
}

// Rows of a head from which tcgen05 takes a part: up to 16 one mma item reads the keys once.
constexpr int kPaTcRows = 17;

struct PaPlan { int kind1, tiles1, ns1, kind2, tiles2, ns2; };

// `vec`: fp32 with d % 4 == 0 and 16-byte strides, `tensor`: bf16 with d % 8 == 0 and 16-byte strides, `tc`: tcgen05
// takes the call (tensor, scale > 0).
inline PaPlan pa_plan(int B, int Tq, int H, int Hk, int d, int page, int n_shared, int W, int num_sms, bool vec, bool tensor,
                      bool tc) {
  PaPlan pl{};
  const long long G = H / Hk, keys1 = (long long)n_shared * page, keys2 = (long long)W * page;
  const long long rows1 = B * (long long)Tq * G, rows2 = Tq * G;
  const int kt = pa_tile_keys(page);
  tc = tc && kt > 0;
  auto kind_of = [&](long long rows) -> int {
    if (vec && rows <= 4) return rows == 1 ? kPaVec1 : rows == 2 ? kPaVec2 : kPaVec4;
    return tc && rows >= kPaTcRows ? (rows <= 128 ? kPaTc128 : kPaTc) : tensor ? kPaMma : rows > 16 ? kPaSimt32 : kPaSimt;
  };
  pl.kind1 = kind_of(rows1);
  pl.kind2 = kind_of(rows2);
  if (pa_is_tc(pl.kind1) && pa_is_tc(pl.kind2) && keys1 > 0 && keys2 > 0 && pl.kind1 != pl.kind2)
    pl.kind1 = pl.kind2 = kPaTc;                   // one launch for both parts
  const long long r1 = pa_tile_rows(pl.kind1), r2 = pa_tile_rows(pl.kind2);
  const long long t1 = keys1 > 0 ? (rows1 + r1 - 1) / r1 : 0, t2 = keys2 > 0 ? (rows2 + r2 - 1) / r2 : 0;
  const long long u1 = t1 * Hk, u2 = t2 * Hk * B;
  // An item's range of keys: all the keys that the launch reads, over 4 CTAs an SM - one wave of equal items, whatever
  // their part (of the room that the rows have: shorter rows split what they have as finely).  Measured at 65536
  // shared tokens and 8 rows: one wave 96 us, two 103, three 107.  A simt item spends about four times as long on a key
  // as the others, which only read it.  At least 64 keys: there an item's time is its latency.
  // Simt items get 3 CTAs an SM, what their shared memory holds, or 4 with 16 rows and a head dim of up to 88.  Measured
  // for 3 and for 4 at 8 rows of 32 queries: 88 us and 110; 64 such rows: 71 and 79; bf16, d = 20: 86 and 69.
  auto range_of = [&](int kind, long long cost) -> long long {
    const long long slots = (kind == kPaSimt32 || (kind == kPaSimt && d > 88) ? 3ll : 4ll) * num_sms;
    const long long r = (cost + slots - 1) / slots;
    return r < 64 ? 64 : r;
  };
  auto weight = [](int kind) -> long long { return kind == kPaSimt || kind == kPaSimt32 ? 4 : 1; };
  const long long cost1 = u1 * keys1 * weight(pl.kind1), cost2 = u2 * keys2 * weight(pl.kind2);
  auto splits = [&](int kind, long long units, long long keys, long long cost) -> int {
    if (units == 0) return 0;
    long long ns, most;
    if (pa_is_tc(kind)) {                         // one CTA an SM: split only what leaves SMs without one
      ns = num_sms / units;
      most = (keys + kt - 1) / kt;
    } else {
      ns = (keys * weight(kind) + range_of(kind, cost) - 1) / range_of(kind, cost);
      most = (keys + 63) / 64;
    }
    ns = ns > most ? most : ns;
    return (int)(ns < 1 ? 1 : ns > 4096 ? 4096 : ns);
  };
  const bool same = pl.kind1 == pl.kind2;          // one launch
  pl.ns1 = splits(pl.kind1, u1, keys1, cost1 + (same ? cost2 : 0));
  pl.ns2 = splits(pl.kind2, u2, keys2, cost2 + (same ? cost1 : 0));
  pl.tiles1 = (int)t1;
  pl.tiles2 = (int)t2;
  return pl;
}

// keys of row b beyond the shared ones (a length beyond the table's room is an error and held at it)
HOA_DEVICE int pa_own_keys(const PaArgs& p, int b) {
  const int own = p.lens[b] - p.n_shared * p.page, room = p.W * p.page;
  if (own > room) pa_fail(p.status);
  return max(0, min(own, room));
}

HOA_DEVICE PaItem pa_item(const PaArgs& p, unsigned idx, int tile_rows, int tile_keys) {
  PaItem it;
  const unsigned n1 = (unsigned)p.tiles1 * p.Hk * p.ns1;
  int split, ns, keys;
  if (idx < n1) {
    it.part = 1;
    it.b = 0;
    it.row0 = (int)(idx % p.tiles1) * tile_rows;   // neighbours read the same keys
    idx /= p.tiles1;
    it.kvh = (int)(idx % p.Hk);
    split = (int)(idx / p.Hk);
    ns = p.ns1;
    it.slot = split;
    keys = p.n_shared * p.page;
    it.key_base = 0;
  } else {
    idx -= n1;
    it.part = 2;
    it.row0 = (int)(idx % p.tiles2) * tile_rows;
    idx /= p.tiles2;
    it.kvh = (int)(idx % p.Hk);
    idx /= p.Hk;
    split = (int)(idx % p.ns2);
    it.b = (int)(idx / p.ns2);
    ns = p.ns2;
    it.slot = p.ns1 + split;
    keys = pa_own_keys(p, it.b);
    it.key_base = p.n_shared * p.page;
  }
  const int tiles = (keys + tile_keys - 1) / tile_keys, per = (tiles + ns - 1) / ns;
  it.k0 = min(keys, split * per * tile_keys);
  it.k1 = min(keys, it.k0 + per * tile_keys);
  return it;
}

HOA_DEVICE PaRow pa_row(const PaArgs& p, const PaItem& it, int r) {
  PaRow w;
  const int per = p.Tq * p.G;
  const int rr = it.part == 1 ? r % per : r;
  w.b = it.part == 1 ? r / per : it.b;
  w.ok = w.b < p.B && rr < per;
  if (!w.ok) w.b = 0;
  w.t = w.ok ? rr / p.G : 0;
  w.h = it.kvh * p.G + (w.ok ? rr % p.G : 0);
  w.seen = w.ok ? p.lens[w.b] - p.Tq + w.t + 1 : 0;
  w.grow = ((long long)w.b * p.Tq + w.t) * p.H + w.h;
  return w;
}

HOA_DEVICE int pa_page(const PaArgs& p, int j) { return p.page > 1 ? (int)(__umulhi((unsigned)j, p.page_mul) >> p.page_shift) : j; }

// element offset of key j of the item's part in k_pages / v_pages, or -1 for a page outside the pool
HOA_DEVICE long long pa_key(const PaArgs& p, const PaItem& it, int j) {
  const int pg = pa_page(p, j);
  const int id = it.part == 1 ? p.shared[pg] : p.table[it.b * p.tstride + pg];
  if (id < 0 || id >= p.n_pages) {
    pa_fail(p.status);
    return -1;
  }
  return id * p.ps + it.kvh * p.hs + (long long)(j - pg * p.page) * p.ts;
}

// The launches of a call overlap (launch_early).  The first one waits for the work before the call and then lets the
// next start; the items of part 2 may so run beside those of part 1, and the join comes up while the last items run.
// Each later launch waits for the one before it at its own end at the latest, so that a kernel has completed only
// after all before it have: the join's wait covers both.  `leads`: the first launch of a call.
HOA_DEVICE void pa_begin(bool leads) {
  if (leads) wait_previous();
  let_next_start();
}

// items first .. first + items - 1
int paged_attn_mma(const PaArgs& a, unsigned first, unsigned items, cudaStream_t s);
int paged_attn_tc(const PaArgs& a, bool dup, unsigned first, unsigned items, cudaStream_t s);

}  // namespace hoa
