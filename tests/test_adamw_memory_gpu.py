"""Buffers of adamw_step that share memory: refused before anything is written, by both host sides."""
import pytest
import torch

from holonomyawareattention_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def buffers(bits, n=3, size=600):
    flat = torch.zeros(2 * n * size, device=DEV)
    cut = lambda t, k: [t[(k * n + i) * size:(k * n + i + 1) * size] for i in range(n)]  # noqa: E731
    m, v = cut(torch.zeros(2 * n * size, device=DEV).to(torch.float8_e4m3fn if bits == 8 else torch.float32), 0), None
    v = [x.clone() for x in m]
    return dict(params=cut(flat, 0), grads=[torch.ones(size, device=DEV) for _ in range(n)], exp_avg=m, exp_avg_sq=v, masters=cut(flat, 1),
                scales=[torch.zeros(2, -(-size // 256), device=DEV) for _ in range(n)] if bits == 8 else None)


@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("bits", [32, 8])
def test_shared_memory(bits, host, monkeypatch):
    step = torch.ones(1, dtype=torch.int32, device=DEV)

    def call(b):
        ops.adamw_step(**b, step=step, lr=1e-2)

    call(buffers(bits))                                           # (neighbours in one buffer, none shared)
    if not host:
        monkeypatch.setattr(ops, "_HOST", ops._Declines())
    call(buffers(bits))
    b = buffers(bits)
    b["masters"] = list(b["params"])                              # (fp32 parameters as their own masters)
    call(b)
    plain = buffers(bits)
    plain["masters"] = None
    call(plain)
    assert all(torch.equal(x, y) for x, y in zip(b["params"], plain["params"]))
    b = buffers(bits)
    b["grads"] = [b["grads"][0]] * 3                              # (grads may share: they are read)
    call(b)

    def over(b, name, i, other, j, shift=0):
        t = b[other][j]
        n = b[name][i].numel()
        whole = t.new_empty(0).set_(t.untyped_storage(), t.storage_offset() + shift, (n,), (1,))
        b[name][i] = whole.view(b[name][i].shape)

    cases = [("exp_avg", 0, "exp_avg", 1, 0), ("exp_avg_sq", 2, "exp_avg", 2, 0), ("exp_avg", 0, "exp_avg", 1, -599), ("params", 0, "params", 1, -1),
             ("masters", 1, "masters", 0, 0), ("masters", 1, "params", 0, 0), ("grads", 1, "params", 1, 0), ("grads", 1, "masters", 2, -300)]
    cases += [("scales", 0, "scales", 1, 0)] if bits == 8 else [("grads", 0, "exp_avg", 0, 0), ("exp_avg_sq", 0, "masters", 1, 5)]
    for c in cases:
        b = buffers(bits)
        over(b, *c)
        before = [b["params"][i].clone() for i in range(3)]
        with pytest.raises(ValueError, match="share no memory|different"):
            call(b)
        assert all(torch.equal(x, y) for x, y in zip(b["params"], before)) and not any(x.float().any() for x in b["exp_avg"] + b["exp_avg_sq"]), c
