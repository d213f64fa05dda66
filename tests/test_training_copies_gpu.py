"""The copies of weights that the module lays out for its kernels, in training and between training steps: each forward sees
the weights that are there."""
import pytest
import torch

from holonomyawareattention_b200 import AdamW, PathOrderedGeometricMHA, ops, train_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


def tril(L):
    return torch.ones(L, L, dtype=torch.bool, device=DEV).tril()


def module(D, H, dtype=torch.bfloat16, es=0.05, seed=0):
    torch.manual_seed(seed)
    return PathOrderedGeometricMHA(D, n_heads=H, edge_scale=es).to(DEV, dtype)


def grads_of(m, x):
    m.zero_grad()
    m(x, attn_mask=tril(x.shape[1]))[0].float().square().sum().backward()
    return {k: p.grad for k, p in m.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("D,H", [(192, 4), (128, 4)])                 # packed and banked generators
@pytest.mark.parametrize("mode", ["auto", "split", "split8"])
def test_evaluated_in_inference_mode_between_steps(D, H, mode):
    x = torch.randn(2, 48, D, device=DEV).to(torch.bfloat16)
    seen = []
    for evaluate in (False, True):
        m = module(D, H, seed=1)
        m.generator_precision = mode
        opt = AdamW(m.parameters(), lr=1e-3)
        for _ in range(2):
            train_step(m, x, opt, lambda y: y.float().square().sum())
            if evaluate:
                with torch.inference_mode():
                    m(x, attn_mask=tril(48))
        if evaluate:
            with torch.inference_mode():
                m(x, attn_mask=tril(48))
        seen.append(grads_of(m, x))
    ops.check_status()
    assert seen[0].keys() == seen[1].keys() and all(torch.equal(seen[0][k], seen[1][k]) for k in seen[0])


def same(m, x):
    """m's forward and gradients are those of a fresh module with its weights."""
    fresh = PathOrderedGeometricMHA(m.h * m.d, n_heads=m.h, edge_scale=m.edge_scale).to(DEV, x.dtype)
    fresh.generator_precision = m.generator_precision
    fresh.load_state_dict(m.state_dict())
    with torch.no_grad():
        if not torch.equal(m(x, attn_mask=tril(x.shape[1]))[0], fresh(x, attn_mask=tril(x.shape[1]))[0]):
            return False
    a, b = grads_of(m, x), grads_of(fresh, x)
    return a.keys() == b.keys() and all(torch.equal(a[k], b[k]) for k in a)


@pytest.mark.parametrize("mode", ["bf16", "split", "split8"])
@pytest.mark.parametrize("D,H,dtype", [(192, 4, torch.bfloat16), (128, 4, torch.bfloat16), (128, 4, torch.float32)])
def test_weights_written_past_torch(D, H, dtype, mode):
    """An optimizer that writes through .data, as many do: no version changes, and each training forward has the new weights,
    and the evaluation after it."""
    m = module(D, H, dtype, seed=2)
    m.generator_precision = mode
    x = torch.randn(2, 32, D, device=DEV).to(dtype)
    assert same(m, x)
    for step in range(3):
        g = grads_of(m, x)
        before = [p._version for p in m.parameters()]
        for k, p in m.named_parameters():
            if k in g:
                p.data.add_(g[k], alpha=-0.02 / float(g[k].float().norm()))
        assert before == [p._version for p in m.parameters()]
        y = m(x, attn_mask=tril(32))[0]                           # (trains: what was kept ends)
        assert y.requires_grad and same(m, x)


def test_written_past_torch_without_training():
    m = module(128, 4, seed=3)
    x = torch.randn(1, 32, 128, device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        old = m(x, attn_mask=tril(32))[0]
        for forget in (m.weights_changed, m.eval, m.train, lambda: m.to("cpu").to(DEV)):
            m.edge_mlp[2].weight.data.mul_(1.5)
            forget()
            new = m(x, attn_mask=tril(32))[0]
            assert not torch.equal(new, old)
            old = new
        m.edge_mlp[2].weight.mul_(0.5)                            # (counted)
        assert not torch.equal(m(x, attn_mask=tril(32))[0], old)


@pytest.mark.parametrize("D,H", [(192, 4), (128, 4)])
def test_parametrized_weights(D, H):
    """weight_norm makes a new weight at every access, each at an address that an earlier one may have had."""
    from torch.nn.utils.parametrizations import weight_norm
    m = module(D, H, seed=4)
    weight_norm(m.edge_mlp[2])
    weight_norm(m.edge_mlp[0])
    x = torch.randn(1, 32, D, device=DEV).to(torch.bfloat16)
    opt = torch.optim.SGD(m.parameters(), lr=1e-3)
    for _ in range(4):
        y = m(x, attn_mask=tril(32))[0]
        with torch.no_grad():
            plain = module(D, H, seed=5)
            plain.load_state_dict({**{k: v for k, v in m.state_dict().items() if "edge" not in k},
                                   **{f"edge_mlp.{i}.{n}": getattr(m.edge_mlp[i], n).detach() for i in (0, 2) for n in ("weight", "bias")}})
            want = plain(x, attn_mask=tril(32))[0]
            assert torch.equal(m(x, attn_mask=tril(32))[0], want)
        p = grads_of(plain, x)
        opt.zero_grad()
        y.float().square().sum().backward()
        assert torch.equal(y, plain(x, attn_mask=tril(32))[0])
        assert torch.equal(m.edge_mlp[2].bias.grad, p["edge_mlp.2.bias"]) and torch.equal(m.qkv.weight.grad, p["qkv.weight"])
        assert m.edge_mlp[2].parametrizations.weight.original1.grad.any()
        opt.step()


def test_frozen_layers_keep_their_copies():
    """Training around a frozen edge MLP lays its weights out once."""
    m = module(128, 4, seed=6)
    m.edge_mlp.requires_grad_(False)
    x = torch.randn(4, 32, 128, device=DEV).to(torch.bfloat16)
    m.PIECE_TOKENS = 32
    laid, real = [], m._w2_rows
    m._w2_rows = lambda *a: laid.append(1) or real(*a)
    for _ in range(3):
        m(x, attn_mask=tril(32))[0].float().sum().backward()
    assert len(laid) == 1
    m.edge_mlp.requires_grad_(True)
    m(x, attn_mask=tril(32))[0].float().sum().backward()
    assert len(laid) == 2                                         # (once a forward, not once a piece)


@pytest.mark.parametrize("D,H", [(192, 4), (128, 4)])
def test_captured_forward(D, H):
    """A captured forward goes on with the copies of its capture while eager ones follow the weights; one that is captured
    before the copies were made leaves none that are not there yet (packed: the banked copies' index comes from the host)."""
    m = module(D, H, seed=7)
    x, mask = torch.randn(1, 32, D, device=DEV).to(torch.bfloat16), tril(32)
    with torch.no_grad():
        old = m(x, attn_mask=mask)[0]
        ops.check_status()                                        # (a launch whose status is still to be read cannot be polled in a capture)
        g, cold = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = m(x, attn_mask=mask)[0]
        if D == 192:
            m.weights_changed()
            with torch.cuda.graph(cold):
                z = m(x, attn_mask=mask)[0]
        assert torch.equal(m(x, attn_mask=mask)[0], old)
        m.edge_mlp[2].weight.mul_(0.5)
        new = m(x, attn_mask=mask)[0]
        junk = [torch.full((2 << 20,), 7.0, device=DEV) for _ in range(8)]      # (would take the memory of copies that were let go)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, old) and not torch.equal(new, old)
        if D == 192:
            cold.replay()
            torch.cuda.synchronize()
            assert torch.equal(z, new)
        assert torch.equal(m(x, attn_mask=mask)[0], new)
        del junk


@pytest.mark.parametrize("D,H,dtype", [(192, 4, torch.bfloat16), (128, 4, torch.bfloat16), (128, 4, torch.float32)])
def test_replayed_adamw_steps(D, H, dtype):
    """A captured adamw_step is replayed between forwards: each forward has the weights that it left."""
    m = module(D, H, dtype, seed=8)
    x, mask = torch.randn(1, 32, D, device=DEV).to(dtype), tril(32)
    ps = [m.edge_mlp[0].weight, m.edge_mlp[2].weight]
    gs = [torch.randn_like(p) for p in ps]
    ms, vs = ([torch.zeros(p.shape, device=DEV) for p in ps] for _ in range(2))
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        m(x, attn_mask=mask)
        ops.check_status()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step.add_(1)
            ops.adamw_step([p.detach() for p in ps], gs, ms, vs, step, lr=1e-2)
        assert all(ops.written_by_graphs(p) for p in ps) and not ops.written_by_graphs(m.qkv.weight)
        old = m(x, attn_mask=mask)[0]
        for _ in range(3):
            g.replay()
            fresh = module(D, H, dtype, seed=9)
            fresh.load_state_dict(m.state_dict())
            new = m(x, attn_mask=mask)[0]
            assert torch.equal(new, fresh(x, attn_mask=mask)[0]) and not torch.equal(new, old)
            old = new
        if D == 192 and dtype is torch.bfloat16:                  # (a captured forward lays them out at each replay)
            ops.check_status()
            f = torch.cuda.CUDAGraph()
            with torch.cuda.graph(f):
                y = m(x, attn_mask=mask)[0]
            g.replay()
            f.replay()
            assert torch.equal(m(x, attn_mask=mask)[0], y) and not torch.equal(y, old)


@pytest.mark.parametrize("D,H", [(192, 4), (128, 4)])
@pytest.mark.parametrize("mode,copies", [("bf16", 1), ("split", 1), ("split8", 2)])
def test_one_copy_a_form(D, H, mode, copies):
    """A training forward lays the second layer's weight out once for each type that its products take, however many pieces
    the batch has, and the backward pass reads the forward's copy."""
    m = module(D, H, seed=10)
    m.generator_precision = mode
    m.PIECE_TOKENS = 32
    x = torch.randn(3, 32, D, device=DEV).to(torch.bfloat16)
    laid, real = [], m._w2_rows
    m._w2_rows = lambda *a: laid.append(1) or real(*a)
    for _ in range(2):
        y = m(x, attn_mask=tril(32))[0]
        y.float().square().sum().backward()
        assert len(laid) == copies
        laid.clear()


@pytest.mark.parametrize("dtype,mode", [(torch.float32, "auto"), (torch.bfloat16, "auto"), (torch.bfloat16, "split")])
def test_train_step_waits_for_nothing(dtype, mode):
    m = module(128, 4, dtype, seed=11)
    m.generator_precision = mode
    x = torch.randn(2, 32, 128, device=DEV).to(dtype)
    opt = AdamW(m.parameters(), lr=1e-3, state_bits=8)
    for i in range(3):
        if i:
            torch.cuda.set_sync_debug_mode("error")
        try:
            train_step(m, x, opt, lambda y: y.float().square().sum(), max_grad_norm=1.0)
        finally:
            torch.cuda.set_sync_debug_mode("default")
    ops.check_status()


def test_one_frozen_layer_keeps_its_copies():
    """... and so does training the first layer before a frozen second one; the first one's end with each step."""
    m = module(128, 4, seed=12)
    m.edge_mlp[2].requires_grad_(False)
    x = torch.randn(2, 32, 128, device=DEV).to(torch.bfloat16)
    laid, real = [], m._w2_rows
    m._w2_rows = lambda *a: laid.append(1) or real(*a)
    for _ in range(3):
        m(x, attn_mask=tril(32))[0].float().sum().backward()
        m.edge_mlp[0].weight.data.mul_(1.01)
        with torch.no_grad():
            m(x, attn_mask=tril(32))
    assert len(laid) == 1
    m(x, attn_mask=tril(32))[0].float().sum().backward()
    m.edge_mlp.requires_grad_(True)
    assert same(m, x)


@pytest.mark.parametrize("D,H,dtype,mode", [(192, 4, torch.bfloat16, "bf16"), (128, 4, torch.bfloat16, "split8"), (128, 4, torch.float32, "auto")])
def test_copies_are_waited_for(D, H, dtype, mode):
    """A forward on one stream lays the weights out behind other work; one on another stream, at once, waits for the copies,
    and they stay until it has read them."""
    m = module(D, H, dtype, seed=13)
    m.generator_precision = mode
    x, mask = torch.randn(1, 32, D, device=DEV).to(dtype), tril(32)
    with torch.no_grad():
        want = m(x, attn_mask=mask)[0]
        one, two = torch.cuda.Stream(), torch.cuda.Stream()
        for first, second in ((one, two), (two, one)):
            m.weights_changed()
            torch.cuda.synchronize()
            with torch.cuda.stream(first):
                if mode != "split8":                              # (which reads a number on the host as it lays out)
                    torch.cuda._sleep(50_000_000)
                a = m(x, attn_mask=mask)[0]
            with torch.cuda.stream(second):
                torch.cuda._sleep(5_000_000)
                b = m(x, attn_mask=mask)[0]
            m.weights_changed()
            with torch.cuda.stream(first):
                junk = [torch.full((1 << 18,), 9.0, device=DEV) for _ in range(20)]
            torch.cuda.synchronize()
            assert torch.equal(a, want) and torch.equal(b, want)
            del junk
    ops.check_status()
