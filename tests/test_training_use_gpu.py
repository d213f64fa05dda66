"""The training operators as programs use them: captured into graphs, on other streams, from two threads, at sizes past
32 bits, one after another, and with waits that give up."""
import threading

import pytest
import torch

from holonomyawareattention_b200 import AdamW, PathOrderedGeometricMHA, _lib, ops, train_step, training

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rel(x, y):
    y = y.double()
    return float((x.double() - y).norm() / y.norm().clamp(min=1e-300))


def attn_inputs(dt, BH=3, T=200, d=64, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    q, k, v, do = (torch.randn(BH, T, d, device=DEV, generator=g).to(dt) for _ in range(4))
    return q, k, v, do


def path_inputs(dt, B=1, T=70, H=2, d=48, chunk=16, seed=0):
    """What the framework's own forward leaves."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    a = 0.3 * torch.randn(B, T, H * (d * (d - 1) // 2), device=DEV, generator=g)
    qkv = torch.randn(B, T, 3 * H * d, device=DEV, generator=g).to(dt)
    R, U, M = ops.link_local(a, qkv, H, 0.05, chunk)
    C, _ = ops.carry_scan(M)
    hats = list(ops.carry_apply(U, C, chunk, dt)) + [torch.randn(B * H, T, d, device=DEV, generator=g)]
    dhats = [torch.randn(B * H, T, d, device=DEV, generator=g).to(dt) for _ in range(4)]
    return a, R, C, chunk, H, 0.05, hats, dhats


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_a_training_step_of_the_operators(dt):
    """link, carry, transport, attention; its backward pass, the path's, AdamW: the gradient of the generators and of q, k, v
    against autograd of the float64 formulas, and the step against the formula on that gradient."""
    from oracle import torch_ref
    B, T, H, d, es, chunk = 2, 50, 2, 48, 0.05, 16
    g = torch.Generator(device=DEV).manual_seed(4)
    a = 0.3 * torch.randn(B, T, H * (d * (d - 1) // 2), device=DEV, generator=g)
    qkv = torch.randn(B, T, 3 * H * d, device=DEV, generator=g).to(dt)
    w = torch.randn(B, T, H * d, device=DEV, generator=g).to(dt)
    R, U, M = ops.link_local(a, qkv, H, es, chunk)
    C, _ = ops.carry_scan(M)
    qh, kh, vh = ops.carry_apply(U, C, chunk, dt)
    o, lse = ops.attn_fwd_lse(qh, kh, vh, d ** -0.5)
    heads = ops.out_transport(o, R, C, chunk, B, H, dt)
    dout = w.view(B, T, H, d).permute(0, 2, 1, 3).float().reshape(B * H, T, d).contiguous()
    doh = ops.apply_paths(dout, R, C, chunk, transpose=True).to(dt)
    dqh, dkh, dvh = ops.attn_bwd(qh, kh, vh, o, lse, doh, d ** -0.5)
    da, dqkv = ops.path_bwd(a, R, C, chunk, H, es, (qh, kh, vh, o), (dqh, dkh, dvh, doh))
    ops.check_status()
    ad, qd = a.double().requires_grad_(), qkv.double().requires_grad_()
    q, k, v = qd.view(B, T, H, 3 * d).transpose(1, 2).chunk(3, -1)
    ref = torch_ref.core_forward(ad.view(B, T, H, -1).transpose(1, 2), q, k, v, es, d ** -0.5)
    (ref.transpose(1, 2).reshape(B, T, H * d) * w.double()).sum().backward()
    # fp32: the forward's bar of 1e-5, twice; bf16: the roundings of the hats, P, dS, their gradients and dqkv, half a step (2^-8) each
    tol = 2e-5 if dt is torch.float32 else 6 * 2.0 ** -8
    assert rel(heads, ref.detach().transpose(1, 2).reshape(B, T, H * d)) < tol
    assert rel(da, ad.grad) < tol and rel(dqkv, qd.grad) < tol
    p, m, v2 = a.clone(), torch.zeros_like(a), torch.zeros_like(a)
    ops.adamw_step([p], [da], [m], [v2], torch.ones(1, dtype=torch.int32, device=DEV), lr=1e-2, weight_decay=0.0)
    # (the first step is lr times the gradient's sign, as far as it is not lost in eps)
    gd = da.double()
    assert float((p.double() - (a.double() - 1e-2 * gd / (gd.abs() + 1e-8))).abs().max()) < 1e-6


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(dt):
    """Two graphs, replayed in turn on changed inputs: each has workspaces of its own."""
    ins = attn_inputs(dt)
    pin = path_inputs(dt)
    o, lse = ops.attn_fwd_lse(*ins[:3], 0.125)
    ops.attn_bwd(*ins[:3], o, lse, ins[3], 0.125)            # (the first call asks the driver for shared memory)
    ops.path_bwd(*pin)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o2, lse2 = ops.attn_fwd_lse(*ins[:3], 0.125)
            out = ops.attn_bwd(*ins[:3], o2, lse2, ins[3], 0.125) + ops.path_bwd(*pin)
        graphs.append((g, out))
    for i in range(3):
        for t in (*ins, *pin[6][3:], *pin[7]):
            t.copy_(torch.randn_like(t))
        g, out = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        o, lse = ops.attn_fwd_lse(*ins[:3], 0.125)
        want = ops.attn_bwd(*ins[:3], o, lse, ins[3], 0.125) + ops.path_bwd(*pin)
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    ops.check_status()


def test_adamw_captured():
    """A captured step counts on the device: three replays are three steps."""
    n = 5000
    p, g = torch.randn(n, device=DEV), torch.randn(n, device=DEV)
    twin = p.clone().requires_grad_()
    ref = torch.optim.AdamW([twin], lr=1e-2)
    m, v, step = torch.zeros_like(p), torch.zeros_like(p), torch.zeros(1, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        ops.adamw_step([p], [g], [m], [v], step, lr=1e-2)
    step.zero_()
    for _ in range(3):
        graph.replay()
        twin.grad = g.clone()
        ref.step()
    assert torch.allclose(p, twin.detach(), rtol=1e-6, atol=2e-8)
    q = torch.zeros(8, device=DEV, requires_grad=True)
    q.grad = torch.ones_like(q)
    opt = AdamW([q])
    opt.step()
    torch.cuda.synchronize()
    with pytest.raises(NotImplementedError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()


def test_train_step_refuses_capture():
    """... before it touches anything: the gradients stay, and no mask made during the capture is kept for later steps."""
    m = PathOrderedGeometricMHA(64, n_heads=4).to(DEV)
    opt, x = AdamW(m.parameters()), torch.randn(1, 23, 64, device=DEV)
    m.qkv.weight.grad = g = torch.randn_like(m.qkv.weight)
    held = dict(training._TRIL)
    torch.cuda.synchronize()
    with pytest.raises(NotImplementedError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            train_step(m, x, opt, lambda y: y.square().mean())
    assert m.qkv.weight.grad is g and training._TRIL == held
    a = train_step(m, x, opt, lambda y: y.square().mean())
    assert bool(torch.isfinite(a))


def test_masks_are_of_a_stream():
    m = torch.ones(9, 9, dtype=torch.bool, device=DEV).tril()
    one = training._tril(9, m.device)
    with torch.cuda.stream(torch.cuda.Stream()):
        two = training._tril(9, m.device)
        assert two is training._tril(9, m.device) and two is not one
    torch.cuda.synchronize()
    assert one is training._tril(9, m.device) and torch.equal(one, m) and torch.equal(two, m)


def test_forward_with_gradients_refuses_capture():
    m = PathOrderedGeometricMHA(64, n_heads=4).to(DEV)
    x, mask = torch.randn(1, 20, 64, device=DEV), torch.ones(20, 20, dtype=torch.bool, device=DEV).tril()
    m(x, attn_mask=mask)[0].sum().backward()
    torch.cuda.synchronize()
    with pytest.raises(NotImplementedError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            m(x, attn_mask=mask)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_other_stream_and_two_threads(dt):
    ins, pin = attn_inputs(dt, seed=1), path_inputs(dt, seed=1)
    o, lse = ops.attn_fwd_lse(*ins[:3], 0.125)
    want = ops.attn_bwd(*ins[:3], o, lse, ins[3], 0.125) + ops.path_bwd(*pin)
    torch.cuda.synchronize()
    bad = []

    def work(k):
        s = torch.cuda.Stream() if k else torch.cuda.current_stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = ops.attn_bwd(*ins[:3], o, lse, ins[3], 0.125) + ops.path_bwd(*pin)
                s.synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, want)):
                    bad.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    ops.check_status()


def test_waits_that_give_up():
    """Short bounds make the tensor-core kernels leave early with HOA_ERR_TIMEOUT; the next calls are whole again."""
    ins, pin = attn_inputs(torch.bfloat16, BH=8, T=700, d=96, seed=2), path_inputs(torch.bfloat16, T=64, d=96, seed=2)
    o, lse = ops.attn_fwd_lse(*ins[:3], 0.1)
    calls = (lambda: ops.attn_bwd(*ins[:3], o, lse, ins[3], 0.1), lambda: ops.path_bwd(*pin), lambda: ops.attn_fwd_lse(*ins[:3], 0.1))
    want = [c() for c in calls]
    ops.check_status()
    for c, w in zip(calls, want):
        ops.set_wait_bound(1)
        try:
            c()
            with pytest.raises(_lib.HoaError) as e:
                ops.check_status()
            assert e.value.status == _lib.HOA_ERR_TIMEOUT
        finally:
            ops.set_wait_bound(0)
        got = c()
        ops.check_status()
        assert all(torch.equal(x, y) for x, y in zip(got, w))


def test_path_bwd_past_32_bits():
    """2.4e9 entries of R, several passes of the workspace: the last chain's gradients are those of its own call."""
    B, T, H, d, chunk = 1, 4096, 64, 96, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    m = d * (d - 1) // 2
    a = torch.zeros(B, T, H * m, device=DEV)
    a[..., -m:] = 0.01 * torch.randn(B, T, m, device=DEV, generator=g)       # (small: R = I stays close enough for both calls alike)
    R = torch.eye(d, device=DEV).expand(H, T, d, d).contiguous()
    C = torch.eye(d, device=DEV).expand(H, T // chunk, d, d).contiguous()
    hats = [torch.randn(H, T, d, device=DEV, generator=g).bfloat16() for _ in range(3)] + [torch.randn(H, T, d, device=DEV, generator=g)]
    dhats = [torch.randn(H, T, d, device=DEV, generator=g).bfloat16() for _ in range(4)]
    da, dqkv = ops.path_bwd(a, R, C, chunk, H, 0.05, hats, dhats)
    for c in (0, H - 1):
        one = lambda t: t[c:c + 1].contiguous()  # noqa: E731
        x, y = ops.path_bwd(a[..., c * m:(c + 1) * m].contiguous(), one(R), one(C), chunk, 1, 0.05, [one(t) for t in hats], [one(t) for t in dhats])
        assert torch.equal(da[..., c * m:(c + 1) * m], x) and torch.equal(dqkv[..., 3 * d * c:3 * d * (c + 1)], y)
    ops.check_status()


def test_attn_bwd_past_32_bits():
    BH, T, d = 60000, 373, 96                                                 # 2.15e9 entries
    q = torch.empty(BH, T, d, dtype=torch.bfloat16, device=DEV).normal_()
    k, do = q.flip(0), q.roll(1, 0)
    o, lse = ops.attn_fwd_lse(q, k, q, 0.1)
    got = ops.attn_bwd(q, k, q, o, lse, do, 0.1)
    for c in (0, BH - 1):
        one = [t[c:c + 1].clone() for t in (q, k, q, o, lse, do)]
        want = ops.attn_bwd(*one, 0.1)
        assert all(torch.equal(x[c:c + 1], y) for x, y in zip(got, want))
    ops.check_status()


def test_adamw_past_32_bits():
    n = 2 ** 31 + 777
    p = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device=DEV)
    m, v = (torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    scales = torch.zeros(2, -(-n // 256), device=DEV)
    ops.adamw_step([p], [g], [m], [v], torch.ones(1, dtype=torch.int32, device=DEV), lr=0.25, weight_decay=0.0, scales=[scales])
    for part in (slice(0, 5), slice(n - 800, n)):
        assert bool((p[part].float() == 0.75).all()) and bool((m[part].float() == 448).all()) and bool((v[part].float() == 448).all())
    assert bool((scales[0] == scales[0, 0]).all()) and abs(float(scales[0, 0]) - 0.05 / 448) < 1e-9


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_host_sides_agree(dt, monkeypatch):
    """The C++ host side takes the ordinary calls and gives the Python functions' bits."""
    torch.manual_seed(3)
    B, H, T, d, chunk = 2, 3, 37, 20, 9
    a = 0.3 * torch.randn(B, T, H * (d * (d - 1) // 2), device=DEV)
    qkv = torch.randn(B, T, 3 * H * d, device=DEV).to(dt)

    def calls():
        R, U, M = ops.link_local(a, qkv, H, 0.5, chunk)
        C, _ = ops.carry_scan(M)
        q, k, v = ops.carry_apply(U, C, chunk, dt)
        o, lse = ops.attn_fwd_lse(q[:, 5:].contiguous(), k, v, 0.2, 5)
        do = torch.ones_like(o).to(dt)
        back = ops.attn_bwd(q[:, 5:].contiguous(), k, v, o, lse, do, 0.2, 5)
        oo, _ = ops.attn_fwd_lse(q, k, v, 0.2)
        da, dqkv = ops.path_bwd(a, R, C, chunk, H, 0.5, (q, k, v, oo), (v, q, k, q))
        out = [o, lse, *back, da, dqkv]
        for bits in (32, 8):
            m = torch.float32 if bits == 32 else torch.float8_e4m3fn
            p = [qkv.clone(), qkv[0, :3, :5].clone()]
            st = [[torch.zeros(x.shape, device=DEV).to(m) for x in p] for _ in range(2)]
            sc = [torch.zeros(2, -(-x.numel() // 256), device=DEV) for x in p] if bits == 8 else None
            ms = [x.float() for x in p] if dt is torch.bfloat16 else None
            before = [x._version for x in p]
            for i in range(2):
                ops.adamw_step(p, [torch.cos(x) for x in p], *st, torch.full((1,), i + 1, dtype=torch.int32, device=DEV), 1e-2,
                               weight_decay=0.1, masters=ms, scales=sc)
            assert [x._version for x in p] == [v + 2 for v in before]
            out += p + [x.float() for s in st for x in s] + (ms or [])
        return out

    first = calls()                                       # (introduces the device)
    taken = []
    host = ops._host()

    class Watch:
        def __getattr__(self, name):
            def call(*args):
                r = getattr(host, name)(*args)
                taken.append((name, r is not None))
                return r
            return call

    monkeypatch.setattr(ops, "_HOST", Watch())
    fast = calls()
    assert {n for n, _ in taken} == {"attn_fwd_lse", "attn_bwd", "path_bwd", "adamw_step"} and all(t for _, t in taken)
    monkeypatch.setattr(ops, "_HOST", ops._Declines())
    slow = calls()
    ops.check_status()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(first, fast, slow))


def test_host_side_declines_what_python_refuses():
    x = torch.randn(2, 6, 16, device=DEV)
    o, lse = ops.attn_fwd_lse(x, x, x, 0.2)
    host = ops._host()
    assert host.attn_fwd_lse(x, x, x, 0.2, 0) is not None
    for bad in ((x, x, x, 0.0, 0), (x, x, x, -0.2, 0), (x, x, x, 0.2, 1), (x, x, x, 0.2, -1), (x, x, x[:1], 0.2, 0), (x.half(), x, x, 0.2, 0),
                (x, x, x.bfloat16(), 0.2, 0), (x.cpu(), x, x, 0.2, 0), (x[:, ::2], x, x, 0.2, 0), (x[:, :0], x, x, 0.2, 0), (x, x, None, 0.2, 0)):
        assert host.attn_fwd_lse(*bad) is None
        assert host.attn_bwd(*bad[:3], o, lse, x, *bad[3:]) is None
    assert host.attn_bwd(x, x, x, o, lse[:, :3], x, 0.2, 0) is None and host.attn_bwd(x, x, x, o.bfloat16(), lse, x, 0.2, 0) is None
    p, g = torch.zeros(8, device=DEV), torch.ones(8, device=DEV)
    m, v, n = torch.zeros(8, device=DEV), torch.zeros(8, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    num = (1e-2, 0.9, 0.99, 1e-8, 0.0)
    for bad in (([p, p], [g, g], [m, m], [v, v], n, *num, None, None), ([p], [g, g], [m], [v], n, *num, None, None),
                ([p], [g[:4]], [m], [v], n, *num, None, None), ([p], [g], [m], [v], n.long(), *num, None, None),
                ([p], [g], [m], [v], n, 1e-2, 1.0, 0.99, 1e-8, 0.0, None, None), ([p], [g], [m], [v], n, *num, [m.bfloat16()], None),
                ([p], [g], [m], [v], n, *num, None, [torch.zeros(2, 1, device=DEV)]), ([p], [None], [m], [v], n, *num, None, None)):
        assert host.adamw_step(*bad) is None
    assert not p.any() and not m.any()
