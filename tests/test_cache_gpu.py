"""Generation operators against plain float64 / Python restatements: the cache's pages, paged
attention with shared pages, the path step.

Tolerances.  fp32 results: 1e-5 rel-L2, the library's fp32 bar (a score's rounding error, about
sqrt(d) 2^-24 |s|, is below 1e-5 for the scores here, and the softmax passes it on as a relative
error of the weights).  bf16 results: 5e-3 rel-L2, from one rounding of the output (2^-9 at most)
and one of the softmax weights (2^-9 at most, averaged).  lse comes from exact products of the bf16
inputs: 1e-5 of max(1, |lse|).  Bookkeeping and moved payload: exact.
"""
import math

import numpy as np
import pytest
import torch

from holonomyawareattention_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
TOL = {F32: 1e-5, BF: 5e-3}


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def rel(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    n = float(b.norm())
    return float((a - b).norm()) / n if n else float((a - b).norm())


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
class Books:
    """The bookkeeping restated with Python lists."""

    def __init__(self, S, W, n_pages, page):
        self.S, self.W, self.page = S, W, page
        self.rows = [[] for _ in range(S)]
        self.lens = [0] * S
        self.refs = [0] * n_pages

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, counts):
        for s, c in enumerate(counts):
            self.lens[s] += c
            while len(self.rows[s]) * self.page < self.lens[s]:
                self.rows[s].append(self.take())

    def fork(self, src, dst):
        moves = []
        shared = []                               # references are added after the fresh pages are taken
        for a, b in zip(src, dst):
            full, part = divmod(self.lens[a], self.page)
            row = self.rows[a][:full]
            shared += row
            if part:
                new = self.take()
                moves.append((self.rows[a][full], new))
                row = row + [new]
            self.rows[b], self.lens[b] = row, self.lens[a]
        for p in shared:
            self.refs[p] += 1
        return moves

    def free(self, rows):
        for r in set(rows):
            for p in self.rows[r]:
                self.refs[p] -= 1
            self.rows[r], self.lens[r] = [], 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if self.refs[i] == 0]
        movers = [i for i in range(live, len(self.refs)) if self.refs[i] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return list(to.items()), live

    def tensors(self):
        table = np.full((self.S, self.W), -1)
        for s, r in enumerate(self.rows):
            table[s, :len(r)] = r
        return i32(table), i32(self.lens), i32(self.refs)


def same(got, books):
    for a, b in zip(got, books.tensors()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("S,W,n_pages,page,shape,dtype", [
    (1, 1, 1, 1, (1, 1, 1), F32),
    (5, 7, 40, 4, (2, 4, 8), BF),
    (9, 6, 64, 3, (1, 3, 5), BF),                 # pages of 30 bytes: two-byte copies
    (33, 20, 700, 16, (4, 16, 48), F32),
    (300, 5, 1500, 2, (2, 2, 6), F32),            # more rows than warps of the cluster
    (700, 3, 5000, 8, (1, 8, 4), BF),             # more forks than threads of a block
])
def test_pages_life(S, W, n_pages, page, shape, dtype):
    """reserve, fork, grow, free and compact in turn, the state and the payload after each."""
    r = np.random.RandomState(S + W)
    bk = Books(S, W, n_pages, page)
    pools = [torch.randn(n_pages, *shape, device=DEV).to(dtype) for _ in range(3)]
    wide = torch.randn(n_pages, 2, *shape, device=DEV).to(dtype)
    pools.append(wide[:, 1])                      # a view: pages further apart than their size
    want = [p.clone() for p in pools]
    state = bk.tensors()

    def move(pairs):
        for w in want:
            src = w.clone()
            for a, b in pairs:
                w[b] = src[a]
        for p, w in zip(pools, want):
            assert torch.equal(p, w)

    first = max(1, S // 3)
    counts = [int(r.randint(0, W * page + 1)) if s < first else 0 for s in range(S)]
    room = n_pages - (S - first)                  # leave a page for every fork
    while sum(-(-c // page) for c in counts) > room:
        counts = [c // 2 for c in counts]
    bk.reserve(counts)
    state = ops.pages_reserve(*state, i32(counts), page)
    same(state, bk)
    dst = list(r.permutation(np.arange(first, S)))
    src = [int(x) for x in r.randint(0, first, size=len(dst))]
    old = [t.clone() for t in state]
    moves = bk.fork(src, dst)
    new = ops.pages_fork(pools, *state, i32(src), i32(dst), page)
    assert all(torch.equal(a, b) for a, b in zip(state, old))       # the old state is left as it was
    state = new
    same(state, bk)
    move(moves)
    gone = [int(x) for x in r.permutation(S)[:S // 2]]
    bk.free(gone)
    state = ops.pages_free(*state, i32(gone + gone[:1]), page)      # (a row listed twice is freed once)
    same(state, bk)
    moves, live = bk.compact()
    table, refs, n = ops.pages_compact(pools, state[0], state[2])
    state = (table, state[1], refs)
    same(state, bk)
    assert n.tolist() == [live]
    move(moves)
    ops.check_status()


def test_pages_out_of_pages_changes_nothing():
    """Too few free pages, a row beyond its table, a dst that is taken or listed twice: the state
    comes back as it was, no payload moves, and the status word says so."""
    bk = Books(4, 4, 6, 4)
    bk.reserve([9, 5, 0, 0])                      # 3 + 2 pages, one free
    state = bk.tensors()
    pool = torch.randn(6, 8, device=DEV)
    want = pool.clone()

    def refused(call):
        out = call()
        torch.cuda.synchronize()
        with pytest.raises(_lib.HoaError) as e:
            ops.check_status()
        assert e.value.status == _lib.HOA_ERR_PAGES
        assert all(torch.equal(a, b) for a, b in zip(out, state)) and torch.equal(pool, want)

    refused(lambda: ops.pages_reserve(*state, i32([0, 0, 4, 4]), 4))
    refused(lambda: ops.pages_reserve(*state, i32([9, 0, 0, 0]), 4))
    refused(lambda: ops.pages_reserve(*state, i32([0, -1, 0, 0]), 4))
    refused(lambda: ops.pages_fork([pool], *state, i32([0, 1]), i32([2, 3]), 4))
    refused(lambda: ops.pages_fork([pool], *state, i32([0]), i32([1]), 4))
    refused(lambda: ops.pages_fork([pool], *state, i32([0, 0]), i32([2, 2]), 4))
    refused(lambda: ops.pages_fork([pool], *state, i32([0]), i32([4]), 4))
    refused(lambda: ops.pages_free(*state, i32([-1]), 4))
    ops.check_status()                            # reported once


def test_pages_copy_and_write():
    page, H, d, n_pages = 5, 3, 7, 12
    kp, vp = (torch.randn(n_pages, H, page, d, device=DEV).to(BF) for _ in range(2))
    want = [kp.clone(), vp.clone()]
    src, dst = [3, -1, 0], [7, -1, 9]
    ops.pages_copy([kp, vp], i32(src), i32(dst))
    for w in want:
        w[7], w[9] = w[3], w[0]
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    table = i32([[1, 4, 10], [2, 6, -1], [5, -1, -1], [-1, -1, -1]])
    lens, T = [12, 9, 2, 0], 4
    k = torch.randn(4, T, 2 * H, d, device=DEV)[:, :, ::2]          # strided heads, fp32 into bf16 pages
    v = torch.randn(H, 4, T, d, device=DEV).permute(1, 2, 0, 3)
    ops.pages_write(k, v, kp, vp, table, i32(lens))
    for b in range(4):
        for t in range(T):
            pos = lens[b] - T + t
            if pos >= 0:
                want[0][table[b, pos // page], :, pos % page] = k[b, t].to(BF)
                want[1][table[b, pos // page], :, pos % page] = v[b, t].to(BF)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])
    ops.check_status()
    with pytest.raises(_lib.HoaError):            # a row without the page: reported, not written
        ops.pages_write(k, v, kp, vp, table, i32([12, 9, 2, 3]))
        torch.cuda.synchronize()
        ops.check_status()
    with pytest.raises(_lib.HoaError):
        ops.pages_copy([kp], i32([n_pages]), i32([0]))
        torch.cuda.synchronize()
        ops.check_status()


# ---------------------------------------------------------------------------
# paged attention
# ---------------------------------------------------------------------------
def make_cache(seed, lens, n_shared, W, page, Hk, d, dtype, spread=1.0):
    """Pools with NaN in every slot no token was written to, table, shared, and each row's k, v."""
    r = np.random.RandomState(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, Ls = len(lens), n_shared * page
    need = [max(0, -(-(n - Ls) // page)) for n in lens]
    n_pages = n_shared + sum(need) + 2
    order = r.permutation(n_pages)
    kp, vp = (torch.full((n_pages, Hk, page, d), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
    shared = order[:n_shared]
    sk, sv = (spread * torch.randn(Ls, Hk, d, device=DEV, generator=g).to(dtype) for _ in range(2))
    for j in range(n_shared):
        for pool, x in ((kp, sk), (vp, sv)):
            pool[shared[j]] = x[j * page:(j + 1) * page].permute(1, 0, 2)
    table = np.full((B, W), -1)
    rows, at = [], n_shared
    for b, n in enumerate(lens):
        own = max(0, n - Ls)
        k, v = (spread * torch.randn(own, Hk, d, device=DEV, generator=g).to(dtype) for _ in range(2))
        for j in range(need[b]):
            table[b, j] = order[at + j]
            part = k[j * page:(j + 1) * page]
            kp[table[b, j], :, :len(part)] = part.permute(1, 0, 2)
            vp[table[b, j], :, :len(part)] = v[j * page:(j + 1) * page].permute(1, 0, 2)
        at += need[b]
        rows.append((torch.cat([sk, k])[:n], torch.cat([sv, v])[:n]))
    return kp, vp, i32(table), i32(shared), rows


def attn_ref(q, rows, lens, scale):
    B, Tq, H, d = q.shape
    out = torch.zeros(B, Tq, H, d, dtype=torch.float64)
    lse = torch.full((B, Tq, H), float("-inf"), dtype=torch.float64)
    for b in range(B):
        k, v = (x.double().cpu() for x in rows[b])
        G = H // k.shape[1]
        for t in range(Tq):
            n = lens[b] - Tq + t + 1
            if n <= 0:
                continue
            for h in range(H):
                s = k[:n, h // G] @ q[b, t, h].double().cpu() * scale
                lse[b, t, h] = torch.logsumexp(s, 0)
                out[b, t, h] = torch.softmax(s, 0) @ v[:n, h // G]
    return out, lse


def check_attn(got, want, dtype):
    (out, lse), (ro, rl) = got, want
    torch.cuda.synchronize()
    ops.check_status()
    empty = torch.isinf(rl)
    lse = lse.double().cpu()
    assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all())
    assert bool(((lse - rl)[~empty].abs() <= 1e-5 * rl[~empty].abs().clamp(min=1)).all())
    assert torch.isfinite(out.float()).all()
    assert bool((out.float().cpu()[empty] == 0).all())
    assert rel(out, ro) <= TOL[dtype], rel(out, ro)


ATTN = [
    # lens, n_shared, W, page, H, Hk, d, Tq
    ([1], 0, 1, 16, 1, 1, 8, 1),
    ([0], 0, 1, 16, 2, 1, 16, 1),                                    # no key at all
    ([0, 0], 0, 0, 4, 1, 1, 8, 2),                                   # no page at all
    ([37, 0, 16, 17, 1], 0, 3, 16, 4, 2, 48, 1),
    ([64, 64, 70, 128, 3, 0], 2, 4, 32, 3, 3, 64, 1),                # rows that end at, in and after the shared pages
    ([130, 200, 129], 2, 5, 64, 16, 16, 96, 1),
    ([300, 257, 260, 0, 100], 4, 2, 64, 6, 6, 120, 1),
    ([77, 90, 78], 3, 3, 25, 2, 1, 20, 1),                           # rows of 40 bytes, pages of 25
    ([50, 41], 1, 4, 13, 3, 1, 33, 2),                               # odd head dim
    ([130, 66, 65, 2, 0, 200], 1, 9, 64, 4, 4, 96, 5),               # queries that reach into the shared pages; fewer keys than queries
    ([300, 290, 128], 1, 3, 128, 8, 2, 128, 40),                     # grouped heads, many queries
    ([500], 0, 8, 64, 2, 2, 48, 500),                                # a whole prompt
    ([140, 9, 260], 0, 17, 16, 4, 1, 64, 137),                       # prompts of other lengths
    ([700, 650, 641] * 20, 10, 2, 64, 2, 2, 96, 1),                  # many rows over a prefix
    ([4096 + 9, 4096 + 300], 64, 5, 64, 1, 1, 96, 1),                # splits along the keys
    ([2100] * 3, 16, 9, 128, 2, 2, 104, 3),
    ([520, 531] * 70, 8, 1, 64, 1, 1, 40, 2),                        # more than one tile of rows
    ([5], 0, 1, 16, 1, 1, 33, 1),                                    # odd counts of floats before the (m, l) pairs
    ([7], 0, 1, 16, 1, 1, 35, 3),
]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_paged_attn(case, dtype):
    lens, n_shared, W, page, H, Hk, d, Tq = ATTN[case]
    kp, vp, table, shared, rows = make_cache(case, lens, n_shared, W, page, Hk, d, dtype)
    q = torch.randn(len(lens), Tq, H, d, device=DEV).to(dtype)
    got = ops.paged_attn_fwd(q, kp, vp, table, i32(lens), 1 / math.sqrt(d), shared=shared)
    check_attn(got, attn_ref(q, rows, lens, 1 / math.sqrt(d)), dtype)
    again = ops.paged_attn_fwd(q, kp, vp, table, i32(lens), 1 / math.sqrt(d), shared=shared)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d,page", [(96, 64), (48, 16), (120, 64), (50, 24)])
def test_paged_attn_paths_strides_streams(d, page, dtype):
    """out = P o; q and the pools as views of wider tensors, the table's rows strided, another
    stream than the one the inputs were made on; fp32 output of bf16 inputs."""
    lens, n_shared, H = [page * 3 + 5, page * 2, page * 2 + 1, 0, 7], 2, 4
    kp, vp, table, shared, rows = make_cache(d, lens, n_shared, 3, page, H, d, dtype)
    pools = torch.zeros(2, kp.shape[0], 2, H, page, d, device=DEV, dtype=dtype)
    pools[0, :, 1], pools[1, :, 1] = kp, vp
    qkv = torch.randn(len(lens), 1, H, 3 * d, device=DEV).to(dtype)
    q = qkv[..., d:2 * d]
    wide = torch.cat([torch.full((len(lens), 2), 10 ** 6, device=DEV, dtype=torch.int32), table], 1)
    P = torch.randn(len(lens), H, d, d, device=DEV)
    ro, rl = attn_ref(q, rows, lens, 0.2)
    ro = torch.einsum("bhij,bthj->bthi", P.double().cpu(), ro)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        out, lse = ops.paged_attn_fwd(q, pools[0, :, 1], pools[1, :, 1], wide[:, 2:], i32(lens), 0.2, shared=shared, paths=P,
                                      out_dtype=F32)
        torch.cuda.current_stream().synchronize()
    assert out.dtype == F32
    check_attn((out, lse), (ro, rl), dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,H,d", [(400, 3, 24), (150, 8, 50), (1190, 1, 120)])
def test_paged_attn_paths_many_rows(B, H, d, dtype):
    """More rows than the join takes P for itself: the transport in a launch of its own."""
    page, n_shared = 16, 1
    r = np.random.RandomState(B)
    lens = [int(x) for x in r.randint(0, 60, size=B)]
    kp, vp, table, shared, rows = make_cache(B, lens, n_shared, 3, page, H, d, dtype)
    q = torch.randn(B, 1, H, d, device=DEV).to(dtype)
    P = torch.randn(B, H, d, d, device=DEV)
    out, lse = ops.paged_attn_fwd(q, kp, vp, table, i32(lens), 0.2, shared=shared, paths=P)
    plain, lse2 = ops.paged_attn_fwd(q, kp, vp, table, i32(lens), 0.2, shared=shared, out_dtype=F32)
    torch.cuda.synchronize()
    ops.check_status()
    assert torch.equal(lse, lse2)
    want = torch.einsum("bhij,bthj->bthi", P.double(), plain.double())
    assert rel(out, want) <= TOL[dtype]
    some = [0, 1, B // 2, B - 1]
    ro, _ = attn_ref(q[some], [rows[b] for b in some], [lens[b] for b in some], 0.2)
    assert rel(plain[some], ro) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,Tq", [(3, 1), (40, 1), (2, 70)])
def test_paged_attn_peaked(B, Tq, dtype):
    """Scores of hundreds: the running maximum moves, weights underflow to 0."""
    n_shared, page, H, d = 6, 64, 2, 96
    lens = [n_shared * page + 100 + b for b in range(B)]
    kp, vp, table, shared, rows = make_cache(3, lens, n_shared, 3, page, H, d, dtype, spread=6.0)
    q = (6 * torch.randn(B, Tq, H, d, device=DEV)).to(dtype)
    got = ops.paged_attn_fwd(q, kp, vp, table, i32(lens), 1 / math.sqrt(d), shared=shared)
    ro, rl = attn_ref(q, rows, lens, 1 / math.sqrt(d))
    # a score of size s carries an error of about s 2^-22, here up to 1e-4 in the weights
    assert rel(got[0], ro) <= TOL[dtype] + 1e-4
    assert bool(((got[1].double().cpu() - rl).abs() <= 1e-5 * rl.abs().clamp(min=1)).all())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lens,n_shared,Tq,H,Hk,d", [
    ([300, 257, 0], 2, 1, 2, 2, 96),              # one row a head of its own, three of the shared part
    ([300, 257], 0, 1, 8, 2, 50),                 # a head dim that no copy takes
    ([300, 280], 2, 3, 4, 2, 96),
    ([300, 280], 2, 40, 4, 2, 64),                # 80 rows a head
    ([400, 380, 390], 3, 130, 2, 2, 96),          # more than one tile of rows
])
def test_paged_attn_nan_and_inf_in_what_is_seen(lens, n_shared, Tq, H, Hk, d, dtype):
    """A query of NaN, a key of +inf: NaN in the rows that see them, nothing in the others."""
    page, W = 64, 6
    kp, vp, table, shared, rows = make_cache(d, lens, n_shared, W, page, Hk, d, dtype)
    q = torch.randn(len(lens), Tq, H, d, device=DEV).to(dtype)
    args = (vp, table, i32(lens), 0.1)
    clean, lse0 = ops.paged_attn_fwd(q, kp, *args, shared=shared)
    bad = q.clone()
    bad[0, Tq - 1, 1, 3] = float("nan")
    out, lse = ops.paged_attn_fwd(bad, kp, *args, shared=shared)
    torch.cuda.synchronize()
    hit = torch.zeros(len(lens), Tq, H, dtype=torch.bool, device=DEV)
    hit[0, Tq - 1, 1] = True
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], lse0[~hit])
    # the last key of sequence 0, seen by its last query alone; 0 * inf in no other score
    k2 = kp.clone()
    k2[table[0, (lens[0] - 1) // page - n_shared].item(), 0, (lens[0] - 1) % page] = float("inf")
    q2 = q.clone()
    q2[0, Tq - 1] = 1.0                           # a score of +inf
    out, lse = ops.paged_attn_fwd(q2, k2, *args, shared=shared)
    torch.cuda.synchronize()
    ops.check_status()
    hit[:] = False
    hit[0, Tq - 1, :H // Hk] = True
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    rest = ~hit
    rest[0, Tq - 1] = False
    assert torch.equal(out[rest], clean[rest]) and torch.equal(lse[rest], lse0[rest])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,Tq,H,Hk,d,page", [
    (1, 1, 2, 2, 96, 64), (3, 1, 2, 2, 48, 16), (3, 1, 4, 2, 50, 32), (9, 2, 2, 1, 64, 24),
    (40, 1, 2, 2, 96, 64), (3, 50, 2, 2, 120, 32), (2, 150, 2, 2, 64, 128), (5, 30, 1, 1, 33, 13),
])
def test_paged_attn_rows_that_end_in_the_shared_pages(B, Tq, H, Hk, d, page, dtype):
    """No row fills the shared pages: what lies after the longest one is NaN, and is in no result."""
    n_shared = 6 if page >= 64 else 12
    room = n_shared * page
    lens = [room // 2 - 5 + (7 * b) % (room // 3) for b in range(B)]
    kp, vp, table, shared, rows = make_cache(page, lens, n_shared, 1, page, Hk, d, dtype)
    for x in range(max(lens), room):
        for pool in (kp, vp):
            pool[shared[x // page].item(), :, x % page] = float("nan")
    q = torch.randn(B, Tq, H, d, device=DEV).to(dtype)
    got = ops.paged_attn_fwd(q, kp, vp, table, i32(lens), 1 / math.sqrt(d), shared=shared)
    check_attn(got, attn_ref(q, rows, lens, 1 / math.sqrt(d)), dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_offsets_past_32_bits(dtype):
    """Pages at the far end of a pool of more than 2^31 elements: the same bits as from a small one."""
    page, H, d, W, B = 64, 8, 96, 4, 3
    n_pages = 2 ** 31 // (H * page * d) + 64
    lens = [page * 3 + 9, page * 2, 70]
    kp, vp, table, shared, rows = make_cache(5, lens, 2, W, page, H, d, dtype)
    small = kp.shape[0]
    kp, vp = kp.nan_to_num(0.0), vp.nan_to_num(0.0)
    far = n_pages - small
    K, V = (torch.empty(n_pages, H, page, d, device=DEV, dtype=dtype) for _ in range(2))
    K[far:], V[far:] = kp, vp
    T = torch.where(table >= 0, table + far, table)
    for Tq in (1, 5, 60):
        q = torch.randn(B, Tq, H, d, device=DEV).to(dtype)
        want = ops.paged_attn_fwd(q, kp, vp, table, i32(lens), 0.1, shared=shared)
        got = ops.paged_attn_fwd(q, K, V, T, i32(lens), 0.1, shared=shared + far)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    k, v = (torch.randn(B, 3, H, d, device=DEV).to(dtype) for _ in range(2))
    a, qkv = torch.randn(B, H * d * (d - 1) // 2, device=DEV), torch.randn(B, 3 * H * d, device=DEV).to(dtype)
    P = torch.eye(d, device=DEV).repeat(B, H, 1, 1)
    own = i32([page * 2 + 1, page, 70])
    step = []
    for x, y, t, at in ((kp, vp, table, 0), (K, V, T, far)):
        full = torch.cat([(shared + at).repeat(B, 1), t], 1)
        ops.pages_write(k, v, x, y, full, own)
        step.append(ops.path_step(a, P, qkv, H, 0.1, x, y, full, own + 2 * (own < 70).int()))
        ops.pages_copy([x, y], i32([at + 1]), i32([at + small - 1]))
    torch.cuda.synchronize()
    ops.check_status()
    assert torch.equal(step[0][0], step[1][0]) and torch.equal(step[0][1], step[1][1])
    assert torch.equal(K[far:], kp) and torch.equal(V[far:], vp)


def test_paged_attn_bad_page_is_reported():
    lens = [100, 90]
    kp, vp, table, shared, rows = make_cache(1, lens, 0, 7, 16, 2, 48, BF)
    q = torch.randn(2, 1, 2, 48, device=DEV).to(BF)
    for bad in (-1, kp.shape[0], 2 ** 30):
        t = table.clone()
        t[1, 2] = bad
        ops.paged_attn_fwd(q, kp, vp, t, i32(lens), 0.1)
        torch.cuda.synchronize()
        with pytest.raises(_lib.HoaError) as e:
            ops.check_status()
        assert e.value.status == _lib.HOA_ERR_PAGES
    ops.paged_attn_fwd(q, kp, vp, table, i32([100, 200]), 0.1)        # longer than its pages
    torch.cuda.synchronize()
    with pytest.raises(_lib.HoaError):
        ops.check_status()
    check_attn(ops.paged_attn_fwd(q, kp, vp, table, i32(lens), 0.1), attn_ref(q, rows, lens, 0.1), BF)


# ---------------------------------------------------------------------------
# path step
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [2, 3, 8, 20, 32, 48, 63, 64, 80, 96, 104, 119, 120])
@pytest.mark.parametrize("es", [0.05, 1.5])
def test_path_step(d, es, dtype):
    torch.manual_seed(d)
    B, H, page, W = 5, 3, 4, 3
    lens = [7, 0, 1, 12, 5]
    m = d * (d - 1) // 2
    a = 0.3 * torch.randn(B, H * m, device=DEV)
    P = torch.linalg.qr(torch.randn(B, H, d, d, device=DEV))[0].contiguous()
    qkv = torch.randn(B, 3 * H * d + 8, device=DEV).to(dtype)[:, :3 * H * d]     # strided rows
    table = i32(np.random.RandomState(d).permutation(B * W).reshape(B, W))
    kp, vp = (torch.randn(B * W, H, page, d, device=DEV).to(dtype) for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    P2, qh = ops.path_step(a, P, qkv, H, es, kp, vp, table, i32(lens))
    torch.cuda.synchronize()
    ops.check_status()
    i, j = torch.triu_indices(d, d, 1)
    A = torch.zeros(B, H, d, d, dtype=torch.float64)
    A[:, :, i, j] = es * a.double().cpu().view(B, H, m)
    A = A - A.transpose(2, 3)
    want = torch.linalg.matrix_exp(A) @ P.double().cpu()
    want[1] = P[1].double().cpu()
    want[2] = torch.eye(d, dtype=torch.float64)
    assert rel(P2, want) <= 1e-5
    x = torch.einsum("bhij,bhni->bhnj", want, qkv.double().cpu().view(B, H, 3, d))
    x[1, :, 0] = 0
    assert rel(qh, x[:, :, 0]) <= TOL[dtype]
    assert bool((qh[1] == 0).all()) and torch.equal(P2[1], P[1])
    for pool, old, n in ((kp, k0, 1), (vp, v0, 2)):
        for b in range(B):
            if lens[b]:
                at, slot = int(table[b, (lens[b] - 1) // page]), (lens[b] - 1) % page
                assert rel(pool[at, :, slot], x[b, :, n]) <= TOL[dtype]
                old[at, :, slot] = pool[at, :, slot]
        assert torch.equal(pool, old)                                 # nothing else was written
    # in place, with a bias, in the banked layout where the head dim has it
    bias = 0.1 * torch.randn(H * m, device=DEV)
    plain = ops.path_step(a + bias, P, qkv, H, es, kp, vp, table, i32(lens))[0]
    Q = P.clone()
    got, _ = ops.path_step(a, Q, qkv, H, es, kp, vp, table, i32(lens), a_bias=bias, P_out=Q)
    assert got is Q and rel(Q, plain) <= 1e-5
    if d % 32 == 0:
        Q2, _ = ops.path_step(ops.gen_to_banked(a, H, d), P, qkv, H, es, kp, vp, table, i32(lens),
                              a_bias=ops.gen_to_banked(bias, H, d), gen_layout="banked")
        assert torch.equal(Q2, Q)


@pytest.mark.parametrize("d", [32, 63, 80, 120])
@pytest.mark.parametrize("es", [0.02, 0.1, 0.5, 1.5])
def test_path_step_as_exact_as_fp32(d, es):
    """Within twice the error of fp32's own matrix exponential and product, from no squaring to six (2e-7: products of
    factors and sums with 2^-23 each, where fp32 is nearly exact)."""
    torch.manual_seed(d)
    B, H = 6, 2
    a = 0.3 * torch.randn(B, H * d * (d - 1) // 2, device=DEV)
    P = torch.linalg.qr(torch.randn(B, H, d, d, device=DEV, dtype=torch.float64))[0].float().contiguous()
    kp, vp = (torch.zeros(B, H, 4, d, device=DEV) for _ in range(2))
    got, _ = ops.path_step(a, P, torch.randn(B, 3 * H * d, device=DEV), H, es, kp, vp, i32([[b] for b in range(B)]), i32([2] * B))
    torch.cuda.synchronize()
    ops.check_status()
    i, j = torch.triu_indices(d, d, 1)
    A = torch.zeros(B, H, d, d, device=DEV)
    A[:, :, i, j] = es * a.view(B, H, -1)
    A = A - A.transpose(2, 3)
    want = torch.linalg.matrix_exp(A.double().cpu()) @ P.double().cpu()
    fp32 = torch.linalg.matrix_exp(A.cpu()) @ P.cpu()
    assert rel(got, want) <= 2 * rel(fp32, want) + 2e-7, (rel(got, want), rel(fp32, want))


def test_path_step_keeps_rotations():
    """A thousand steps: P stays orthogonal to fp32 accuracy (the errors of the steps add like a
    random walk at worst linearly: 1000 x 1e-7)."""
    torch.manual_seed(0)
    B, H, d = 2, 2, 96
    P = torch.eye(d, device=DEV).expand(B, H, d, d).contiguous()
    kp = torch.zeros(B, H, 16, d, device=DEV)
    table, lens = i32([[0], [1]]), i32([2, 2])
    for _ in range(1000):
        a = 0.3 * torch.randn(B, H * d * (d - 1) // 2, device=DEV)
        P, _ = ops.path_step(a, P, torch.zeros(B, 3 * H * d, device=DEV), H, 0.05, kp, kp.clone(), table, lens)
    err = (P.double().transpose(2, 3) @ P.double() - torch.eye(d, device=DEV, dtype=torch.float64)).abs().max()
    assert float(err) <= 1e-4


def test_path_step_bad_page_is_reported():
    B, H, d = 2, 1, 16
    P = torch.eye(d, device=DEV).expand(B, H, d, d).contiguous()
    kp = torch.zeros(3, H, 4, d, device=DEV)
    vp = kp.clone()
    a, qkv = torch.zeros(B, d * (d - 1) // 2, device=DEV), torch.ones(B, 3 * d, device=DEV)
    for table, lens in (([[0, -1], [1, 2]], [5, 5]), ([[0, 3], [1, 2]], [5, 5]), ([[0, 1], [1, 2]], [9, 5])):
        ops.path_step(a, P, qkv, H, 0.1, kp, vp, i32(table), i32(lens))
        torch.cuda.synchronize()
        with pytest.raises(_lib.HoaError) as e:
            ops.check_status()
        assert e.value.status == _lib.HOA_ERR_PAGES
        assert bool((kp[0] == 0).all())


# ---------------------------------------------------------------------------
# the two host sides of a call
# ---------------------------------------------------------------------------
def test_both_host_sides_give_the_same(monkeypatch):
    """The ordinary calls' C++ side against the Python functions behind it, bit for bit; a call that the
    C++ side does not take (here: another pool stride, an integer scale) reaches them by itself."""
    class Declines:
        def __getattr__(self, name):
            return lambda *a: None

    d, H, page = 48, 2, 16
    bk = Books(6, 4, 40, page)
    bk.reserve([50, 20, 0, 7, 0, 0])
    state = bk.tensors()
    pools = [torch.randn(40, H, page, d, device=DEV) for _ in range(2)]
    q = torch.randn(6, 1, H, d, device=DEV)
    P = torch.linalg.qr(torch.randn(6, H, d, d, device=DEV))[0].contiguous()
    a, qkv = torch.randn(6, H * d * (d - 1) // 2, device=DEV), torch.randn(6, 3 * H * d, device=DEV)

    def all_calls():
        kp, vp = (p.clone() for p in pools)
        out = list(ops.pages_reserve(*state, i32([3, 0, 0, 20, 0, 1]), page))
        out += ops.pages_fork([kp, vp], *state, i32([0, 1]), i32([2, 4]), page)
        out += ops.pages_free(*state, i32([0]), page)
        out += ops.pages_compact([kp, vp], state[0], state[2])
        out += ops.paged_attn_fwd(q, kp, vp, state[0], state[1], 0.25, paths=P)
        out += ops.path_step(a, P, qkv, H, 0.05, kp, vp, state[0], state[1])
        torch.cuda.synchronize()
        ops.check_status()
        return out + [kp, vp]

    fast = all_calls()
    monkeypatch.setattr(ops, "_HOST", Declines())
    slow = all_calls()
    monkeypatch.undo()
    assert len(fast) == len(slow) and all(torch.equal(x, y) for x, y in zip(fast, slow))
    wide = torch.randn(40, 2, H, page, d, device=DEV)
    assert ops.paged_attn_fwd(q, wide[:, 0], wide[:, 1], state[0], state[1], 1)[0].shape == q.shape
    with pytest.raises(ValueError, match="must be"):
        ops.paged_attn_fwd(q, pools[0], pools[1], state[0].long(), state[1], 0.25)
    with pytest.raises(ValueError, match="contiguous int32"):
        ops.pages_free(state[0], state[1][::2], state[2], i32([0]), page)
    with pytest.raises(NotImplementedError, match="CUDA"):
        ops.paged_attn_fwd(q, pools[0], pools[1], state[0].cpu(), state[1], 0.25)


def test_calls_under_graph_capture():
    """A decode step (reserve apart) captured once and replayed on new inputs."""
    d, H, page, B = 96, 4, 64, 3
    table = i32([[0, 1], [2, 3], [4, 5]])
    lens = i32([70, 100, 1])
    kp, vp = (torch.randn(6, H, page, d, device=DEV).to(BF) for _ in range(2))
    P = torch.linalg.qr(torch.randn(B, H, d, d, device=DEV))[0].contiguous()
    a, qkv = 0.3 * torch.randn(B, H * d * (d - 1) // 2, device=DEV), torch.randn(B, 3 * H * d, device=DEV).to(BF)

    def step():
        P2, qh = ops.path_step(a, P, qkv, H, 0.05, kp, vp, table, lens)
        return ops.paged_attn_fwd(qh.view(B, 1, H, d), kp, vp, table, lens, 0.1, paths=P2)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = step()
    for seed in (1, 2):
        torch.manual_seed(seed)
        a.normal_(0, 0.3)
        qkv.normal_()
        g.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    ops.check_status()
