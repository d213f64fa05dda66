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
  long long rows;                                  // B * Tq * H
  float scale_log2;
  int dtype, B, Tq, H, Hk, G, d, page, n_pages;
  int tiles1, ns1, tiles2, ns2;
  int* status;
};

struct PaItem {
  int part, kvh, b, row0, slot;
  int k0, k1;                                      // keys of this part [k0, k1)
  int key_base;                                    // position of the part's key 0
};

struct PaRow { bool ok; int b, t, h, seen; long long grow; };

struct PaPlan { int tiles1, ns1, tiles2, ns2; };

HOA_DEVICE void pa_fail(int* status) {
  if (status != nullptr) *reinterpret_cast<volatile int*>(status) = HOA_ERR_PAGES;
}

// rows of a tile: see paged_attn_simt_kernel
inline PaPlan pa_plan(int B, int Tq, int H, int Hk, int page, int n_shared, int W, int num_sms) {
  PaPlan pl{};
  const int G = H / Hk;
  if (n_shared > 0) {
    pl.tiles1 = ceil_div((long long)B * Tq * G, 16);
    const long long units = (long long)pl.tiles1 * Hk, tiles = ceil_div((long long)n_shared * page, 64);
    long long ns = (2 * num_sms + units - 1) / units;
    if (ns > tiles) ns = tiles;
    pl.ns1 = (int)(ns < 1 ? 1 : ns);
  }
  if (W > 0) {
    pl.tiles2 = ceil_div((long long)Tq * G, 16);
    const long long units = (long long)B * Hk * pl.tiles2, tiles = ceil_div((long long)W * page, 64);
    long long ns = (2 * num_sms + units - 1) / units;
    if (ns > tiles) ns = tiles;
    pl.ns2 = (int)(ns < 1 ? 1 : ns);
  }
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

// element offset of key j of the item's part in k_pages / v_pages, or -1 for a page outside the pool
HOA_DEVICE long long pa_key(const PaArgs& p, const PaItem& it, int j) {
  const int pg = j / p.page;
  const int id = it.part == 1 ? p.shared[pg] : p.table[it.b * p.tstride + pg];
  if (id < 0 || id >= p.n_pages) {
    pa_fail(p.status);
    return -1;
  }
  return id * p.ps + it.kvh * p.hs + (long long)(j - pg * p.page) * p.ts;
}

}  // namespace hoa
