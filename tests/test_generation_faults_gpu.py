"""Generation when something goes wrong around a call: threads, errors in the middle of a step, lists and
modes that are out of the ordinary.  What a call reports, and what it leaves behind.
"""
import threading

import pytest
import torch

from holonomyawareattention_b200 import PathCache, PathOrderedGeometricMHA, _lib, decode, ops, prefill  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def clean_status():
    """No status of one test is left for the next."""
    yield
    torch.cuda.synchronize()
    try:
        ops.check_status()
    except _lib.HoaError:
        pass


def pages(n, H=2, page=16, d=48, dtype=BF, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(n, H, page, d, device=DEV, generator=g).to(dtype) for _ in range(2)]


def module(D=64, H=2, dtype=F32):
    torch.manual_seed(D)
    return PathOrderedGeometricMHA(D, n_heads=H, edge_scale=0.05).to(DEV, dtype).eval()


def state_of(cache):
    live = [r for r in range(cache.rows) if cache.tokens[r]]
    return ([t.clone() for t in (cache.table, cache.lens, cache.refs, cache.P[live], cache.last[live])],
            (list(cache.tokens), [list(h) for h in cache._held], dict(cache._count), cache.n_shared))


def same_state(a, b):
    return all(torch.equal(x, y) for x, y in zip(a[0], b[0])) and a[1] == b[1]


# ---------------------------------------------------------------------------
# host threads
# ---------------------------------------------------------------------------
def attn_args(seed, B=6, H=2, d=48, W=24, page=16):
    kp, vp = pages(B * W, H, page, d, seed=seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(B, 1, H, d, device=DEV, generator=g).to(BF)
    table = i32([[b * W + j for j in range(W)] for b in range(B)])
    return q, kp, vp, table, i32([W * page - 3 * b for b in range(B)]), 0.2


def test_calls_in_progress_share_no_scratch(monkeypatch):
    """A call that begins while another one on the same stream has not returned (two threads: the library is
    called without the interpreter's lock) hands its parts over in memory of its own."""
    a, b = attn_args(1), attn_args(2)
    ops.paged_attn_fwd(*a, out_dtype=F32)         # (what is looked up once is known)
    real, seen = ops._fn, []

    def fn(name):
        f = real(name)

        def call(*args):
            if name == "hoa_paged_attn_fwd":
                seen.append(args[-4])             # the workspace
                if len(seen) == 1:
                    ops.paged_attn_fwd(*b, out_dtype=F32)
            return f(*args)
        return call

    monkeypatch.setattr(ops, "_fn", fn)
    ops.paged_attn_fwd(*a, out_dtype=F32)
    torch.cuda.synchronize()
    assert len(seen) == 2 and seen[0] != seen[1]


def test_two_threads_on_one_stream():
    """Attention, fork and prefill from two threads on the default stream: each result as in one thread alone."""
    attn = module(192, 4, BF)
    prompts = [torch.randn(2, 90, 192, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)).to(BF) for i in range(2)]
    args = [attn_args(i) for i in range(2)]

    def work(i, n):
        out = []
        with torch.no_grad():
            for k in range(n):
                out += ops.paged_attn_fwd(*args[i], out_dtype=F32)
                if k % 10 == 0:
                    cache = PathCache(attn, rows=4, max_tokens=128, page=16)
                    y = prefill(attn, prompts[i], cache, [0, 1])
                    # pools as a tuple: the Python side of the call
                    st = ops.pages_fork((cache.k_pages, cache.v_pages), cache.table, cache.lens, cache.refs, i32([0, 1]), i32([2, 3]), 16)
                    new = st[0][2:, 5].long()
                    out += [y, *st, cache.k_pages[new], cache.v_pages[new]]
        torch.cuda.current_stream().synchronize()
        return out

    want = [work(i, 10) for i in range(2)]
    got = [None, None]

    def run(i):
        got[i] = work(i, 200)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    per = len(want[0])
    for i in range(2):
        assert len(got[i]) == 20 * per
        # slots that no token was written to are whatever the pool's memory held: compare the written ones
        for k, x in enumerate(got[i]):
            w = want[i][k % per]
            if x.dim() == 4 and x.shape[0] == 2 and x.dtype == BF and x.shape[2] == 16:
                x, w = x[:, :, :90 % 16], w[:, :, :90 % 16]
            assert torch.equal(x, w), (i, k)
    ops.check_status()


# ---------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------
def test_reserve_of_more_tokens_than_an_int_counts():
    """Pages so large that W of them hold 2^31 tokens and more: a row that would pass an int is refused, one that comes
    just up to it is not."""
    page, W = 2 ** 30, 4
    state = i32([[0, 1, -1, -1], [-1] * 4]), i32([2 ** 31 - 10, 0]), i32([1, 1, 0, 0, 0, 0])
    for counts in ([10, 5], [2 ** 31 - 1, 2 ** 31 - 1]):
        out = ops.pages_reserve(*state, i32(counts), page)
        torch.cuda.synchronize()
        with pytest.raises(_lib.HoaError) as e:
            ops.check_status()
        assert e.value.status == _lib.HOA_ERR_PAGES
        assert all(torch.equal(a, b) for a, b in zip(out, state))
    t, n, r = ops.pages_reserve(*state, i32([9, 2 ** 30 + 1]), page)
    torch.cuda.synchronize()
    ops.check_status()
    assert t.tolist() == [[0, 1, -1, -1], [2, 3, -1, -1]] and n.tolist() == [2 ** 31 - 1, 2 ** 30 + 1] and r.tolist() == [1, 1, 1, 1, 0, 0]


# ---------------------------------------------------------------------------
# what check_status waits for
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("side", [False, True])
def test_check_status_waits_for_the_cache_kernels(side):
    """A page outside the pool, in a call that is still queued behind other work (on any stream)."""
    q, kp, vp, table, lens, scale = attn_args(3)
    bad = table.clone()
    bad[1, 2] = kp.shape[0]
    ops.paged_attn_fwd(q, kp, vp, table, lens, scale)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.current_stream()):
        torch.cuda._sleep(200_000_000)
        ops.paged_attn_fwd(q, kp, vp, bad, lens, scale)
    with pytest.raises(_lib.HoaError) as e:
        ops.check_status()
    assert e.value.status == _lib.HOA_ERR_PAGES
    ops.check_status()


def test_status_outlives_its_watch():
    """The word that the kernels set stays the one that is read when the watch of a device is made anew."""
    q, kp, vp, table, lens, scale = attn_args(3)
    ops.paged_attn_fwd(q, kp, vp, table, lens, scale)
    torch.cuda.synchronize()
    ops._WATCH.clear()
    bad = table.clone()
    bad[0, 0] = -1
    ops.paged_attn_fwd(q, kp, vp, bad, lens, scale)
    torch.cuda.synchronize()
    with pytest.raises(_lib.HoaError) as e:
        ops.check_status()
    assert e.value.status == _lib.HOA_ERR_PAGES


def test_cache_across_inference_mode():
    """Made and fed in inference mode, then outside it, and the other way round."""
    attn = module(96, 2)
    x = torch.randn(2, 10, 96, device=DEV)
    outs = []
    for modes in ((torch.inference_mode, torch.no_grad), (torch.no_grad, torch.inference_mode), (torch.no_grad, torch.no_grad)):
        got = []
        with modes[0]():
            cache = PathCache(attn, rows=3, max_tokens=60, page=16)
            got.append(prefill(attn, x, cache, [0, 1]))
            got.append(decode(attn, torch.ones(3, 96, device=DEV), cache))
        with modes[1]():
            got.append(prefill(attn, x + 1, cache, [0, 1]))
            cache.fork([0], [2])
            got.append(decode(attn, torch.ones(3, 96, device=DEV), cache))
            cache.share(0, 0)
        with modes[0]():
            got.append(prefill(attn, x - 1, cache, [2, 1]))
            got.append(decode(attn, torch.ones(3, 96, device=DEV), cache))
        outs.append(got)
    for got in outs[:2]:
        assert all(torch.equal(a, b) for a, b in zip(got, outs[2]))
    ops.check_status()


# ---------------------------------------------------------------------------
# an error in the middle of an operation
# ---------------------------------------------------------------------------
class Boom(Exception):
    pass


def failing(real, after=0):
    """``real``, but the call after ``after`` good ones raises."""
    left = [after]

    def call(*a, **k):
        if left[0] == 0:
            raise Boom
        left[0] -= 1
        return real(*a, **k)
    return call


def test_fork_after_transposed_hidden_states():
    """decode with hidden states of other strides (a transposed view), then a fork, with and without idle rows."""
    attn = module(96, 2)
    x = torch.randn(96, 3, device=DEV)
    with torch.no_grad():
        caches = [PathCache(attn, rows=3, max_tokens=60, page=16) for _ in range(2)]
        for cache, y in zip(caches, (x.t(), x.t().contiguous())):
            prefill(attn, torch.ones(1, 20, 96, device=DEV), cache, [0])
            decode(attn, y, cache)
            cache.fork([0], [2])
            decode(attn, y, cache)
            cache.fork([2], [1])
            decode(attn, y, cache)                                # every row has tokens
            cache.free([0])
            cache.fork([1], [0])
        assert same_state(state_of(caches[0]), state_of(caches[1]))
        for cache in caches:                                      # (k^ and v^: GEMMs of other layouts round otherwise)
            assert torch.equal(cache.P[0], cache.P[1]) and torch.equal(cache.last[0], cache.last[1])
        ops.check_status()


@pytest.mark.parametrize("where", ["pages_fork", "pages_copy", "_ints"])
def test_fork_that_fails_changes_nothing(monkeypatch, where):
    attn = module(96, 2)
    with torch.no_grad():
        cache = PathCache(attn, rows=3, max_tokens=60, page=16)
        prefill(attn, torch.randn(1, 20, 96, device=DEV), cache, [0])
        before = state_of(cache)
        with monkeypatch.context() as m:
            owner = cache if where == "_ints" else ops
            m.setattr(owner, where, failing(getattr(owner, where), after=1 if where == "_ints" else 0))
            with pytest.raises(Boom):
                cache.fork([0, 0], [1, 2])
        assert same_state(state_of(cache), before)
        cache.fork([0, 0], [1, 2])
        assert cache.tokens == [20] * 3 and cache.lens.tolist() == [20] * 3
        assert torch.equal(cache.P[1], cache.P[0]) and torch.equal(cache.last[2], cache.last[0])
        ops.check_status()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("where,after", [("paged_attn_fwd", 0), ("compose_paths", 0), ("paged_attn_fwd", 1), ("compose_paths", 1)])
def test_prefill_that_fails_changes_nothing(monkeypatch, where, after, dtype):
    """In the first or the second piece of rows, for new rows and for rows that go on: the cache is as it was,
    and the same prompt then gives what a cache that never failed gives."""
    attn = module(96, 2, dtype)
    monkeypatch.setattr(attn, "PIECE_TOKENS", 50)                 # a row a piece
    x = [torch.randn(3, 40, 96, device=DEV).to(dtype) for _ in range(2)]
    with torch.no_grad():
        good, cache = (PathCache(attn, rows=4, max_tokens=100, page=16) for _ in range(2))
        for c in (good, cache):
            prefill(attn, x[0][:1, :7], c, [3])
        for step in range(2):
            before = state_of(cache)
            with monkeypatch.context() as m:
                m.setattr(ops, where, failing(getattr(ops, where), after))
                with pytest.raises(Boom):
                    prefill(attn, x[step], cache, [2, 0, 1])
            assert same_state(state_of(cache), before)
            want, got = (prefill(attn, x[step], c, [2, 0, 1]) for c in (good, cache))
            assert torch.equal(want, got) and same_state(state_of(good), state_of(cache))
        ops.check_status()


@pytest.mark.parametrize("where", ["path_step", "paged_attn_fwd", "out", "qkv"])
@pytest.mark.parametrize("idle", [False, True])
def test_decode_that_fails_changes_nothing(monkeypatch, where, idle):
    attn = module(96, 2)
    rows = 3
    x = torch.randn(2, rows, 96, device=DEV)
    with torch.no_grad():
        good, cache = (PathCache(attn, rows=rows + idle, max_tokens=100, page=16) for _ in range(2))
        xs = torch.cat([x, torch.zeros(2, idle, 96, device=DEV)], 1)
        for c in (good, cache):
            prefill(attn, torch.randn(rows, 16, 96, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)), c, range(rows))
        for step in range(2):
            before = state_of(cache)
            with monkeypatch.context() as m:
                if where in ("out", "qkv"):
                    m.setattr(getattr(attn, where), "forward", failing(None))
                else:
                    m.setattr(ops, where, failing(getattr(ops, where)))
                with pytest.raises(Boom):
                    decode(attn, xs[step], cache)
            assert same_state(state_of(cache), before)
            want, got = (decode(attn, xs[step], c) for c in (good, cache))
            assert torch.equal(want, got) and same_state(state_of(good), state_of(cache))
        ops.check_status()


def test_compact_that_fails_changes_nothing(monkeypatch):
    """The copy of the shared pages' ids fails after the pages were moved: the old state still holds."""
    attn = module(96, 2)
    with torch.no_grad():
        cache = PathCache(attn, rows=4, max_tokens=60, page=16)
        prefill(attn, torch.randn(2, 40, 96, device=DEV), cache, [0, 3])
        cache.free([0])                           # row 3's pages lie behind row 0's
        cache.fork([3], [1])
        cache.share(3)
        before, shared = state_of(cache), cache.shared.clone()
        with monkeypatch.context() as m:
            m.setattr(torch.Tensor, "clone", failing(None), raising=False)
            with pytest.raises(Boom):
                cache.compact()
        assert same_state(state_of(cache), before) and torch.equal(cache.shared, shared)
        live = cache.compact()
        assert int(live) == len(cache._count) and torch.equal(cache.shared, cache.table[3, :2])
        y = decode(attn, torch.ones(4, 96, device=DEV), cache)
        assert torch.isfinite(y).all() and torch.equal(y[3], y[1])
        ops.check_status()


# ---------------------------------------------------------------------------
def test_share_refuses_a_negative_length():
    attn = module()
    with torch.no_grad():
        cache = PathCache(attn, rows=2, max_tokens=80, page=16)
        prefill(attn, torch.randn(1, 50, 64, device=DEV), cache, [0])
        cache.fork([0], [1])
        for tokens in (-1, -16, -40):
            with pytest.raises(ValueError, match="tokens"):
                cache.share(0, tokens)
            assert cache.n_shared == 0 and cache.shared is None
        assert cache.share(0, 47) == 32 and cache.share(0, 0) == 0


def test_reserve_refuses_an_empty_row_while_pages_are_shared():
    """Attention reads the shared pages as every row's first ones: a row that begins with others cannot start."""
    attn = module()
    with torch.no_grad():
        cache = PathCache(attn, rows=3, max_tokens=80, page=16)
        prefill(attn, torch.randn(1, 40, 64, device=DEV), cache, [0])
        cache.share(0)
        before = state_of(cache)
        with pytest.raises(ValueError, match="shared pages"):
            cache.reserve([1, 0, 5])
        assert same_state(state_of(cache), before)
        cache.reserve([1, 0, 0])
        cache.share(0, 0)
        cache.reserve([0, 0, 5])
        assert cache.tokens == [41, 0, 5] and cache.lens.tolist() == [41, 0, 5]
        ops.check_status()


def test_free_of_a_page_that_nobody_counts():
    """A table that holds pages with refs 0 (or fewer references than rows): reported, refs stay at 0, and the pages can be
    taken again."""
    table, lens, refs = i32([[0, 1, -1], [1, 2, -1], [1, -1, -1]]), i32([8, 7, 3]), i32([1, 1, 0, 0])
    t, n, r = ops.pages_free(table, lens, refs, i32([0, 1, 2]), 4)
    with pytest.raises(_lib.HoaError) as e:
        torch.cuda.synchronize()
        ops.check_status()
    assert e.value.status == _lib.HOA_ERR_PAGES
    assert r.tolist() == [0, 0, 0, 0] and n.tolist() == [0, 0, 0] and bool((t == -1).all())
    t, n, r = ops.pages_reserve(t, n, r, i32([8, 8, 0]), 4)
    assert t.tolist() == [[0, 1, -1], [2, 3, -1], [-1, -1, -1]] and r.tolist() == [1, 1, 1, 1]
    torch.cuda.synchronize()
    ops.check_status()


# ---------------------------------------------------------------------------
# rows that are idle
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,H,d", [(5, 2, 96), (4, 3, 50), (700, 2, 48), (400, 3, 25)])
def test_an_idle_row_gives_zeros_whatever_its_path_holds(B, H, d, dtype):
    """out is 0 where a query sees no key: NaN and infinities in that row's P do not reach it (few rows: the join applies
    P; many: a launch of its own)."""
    page, W = 16, 2
    kp, vp = pages(B * W, H, page, d, dtype)
    q = torch.randn(B, 1, H, d, device=DEV).to(dtype)
    lens = [0 if b % 4 == 1 else 1 + (5 * b) % (W * page) for b in range(B)]
    idle = torch.tensor([n == 0 for n in lens], device=DEV)
    P = torch.randn(B, H, d, d, device=DEV)
    args = (q, kp, vp, i32([[b * W, b * W + 1] for b in range(B)]), i32(lens), 0.2)
    want = ops.paged_attn_fwd(*args, paths=P)
    bad = P.clone()
    bad[idle] = float("nan")
    bad[1, 0, 0, 0] = float("inf")
    out, lse = ops.paged_attn_fwd(*args, paths=bad)
    torch.cuda.synchronize()
    ops.check_status()
    assert bool((out[idle] == 0).all()) and bool(torch.isneginf(lse[idle]).all())
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_a_row_freed_after_nan_decodes_to_zero():
    attn = module(96, 2)
    with torch.no_grad():
        cache = PathCache(attn, rows=2, max_tokens=40, page=16)
        x = torch.randn(2, 5, 96, device=DEV)
        x[1] = float("nan")
        prefill(attn, x, cache, [0, 1])
        cache.free([1])
        y = decode(attn, torch.ones(2, 96, device=DEV), cache)
        torch.cuda.synchronize()
        assert torch.isfinite(y[0]).all() and bool((y[1] == 0).all())
        ops.check_status()


# ---------------------------------------------------------------------------
# waits that give up
# ---------------------------------------------------------------------------
def test_path_step_surfaces_a_timed_out_wait():
    """With a short wait bound the step gives up on its products, leaves, and reports it; with the default bound the same
    call then gives the first result.  Seven products a head: the time of a call that gives up is bounded too."""
    B, H, d = 40, 4, 120
    g = torch.Generator(device=DEV).manual_seed(0)
    a = torch.randn(B, H * d * (d - 1) // 2, device=DEV, generator=g)
    P = torch.linalg.qr(torch.randn(B, H, d, d, device=DEV, generator=g))[0].contiguous()
    qkv = torch.randn(B, 3 * H * d, device=DEV, generator=g)
    table, lens = i32([[b] for b in range(B)]), i32([3] * B)

    def step():
        kp = torch.zeros(B, H, 4, d, device=DEV)
        return ops.path_step(a, P, qkv, H, 0.5, kp, kp.clone(), table, lens)

    want = step()
    torch.cuda.synchronize()
    ops.check_status()
    ops.set_wait_bound(1)
    try:
        step()
        torch.cuda.synchronize()
        with pytest.raises(_lib.HoaError) as e:
            ops.check_status()
        assert e.value.status == _lib.HOA_ERR_TIMEOUT
    finally:
        ops.set_wait_bound(0)
    for _ in range(3):
        got = step()
        torch.cuda.synchronize()
        ops.check_status()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("Tq", [30, 200])
def test_paged_attention_surfaces_a_timed_out_wait(Tq):
    """The tcgen05 kernel, one and two tiles of rows."""
    H, d, page, W = 2, 96, 64, 40
    kp, vp = pages(2 * W, H, page, d)
    q = torch.randn(2, Tq, H, d, device=DEV).to(BF)
    table, lens = i32([[b * W + j for j in range(W)] for b in range(2)]), i32([W * page, W * page - 9])
    args = (q, kp, vp, table, lens, 0.1)
    want = ops.paged_attn_fwd(*args)
    torch.cuda.synchronize()
    ops.check_status()
    ops.set_wait_bound(1)
    try:
        ops.paged_attn_fwd(*args)
        torch.cuda.synchronize()
        with pytest.raises(_lib.HoaError) as e:
            ops.check_status()
        assert e.value.status == _lib.HOA_ERR_TIMEOUT
    finally:
        ops.set_wait_bound(0)
    got = ops.paged_attn_fwd(*args)
    torch.cuda.synchronize()
    ops.check_status()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
