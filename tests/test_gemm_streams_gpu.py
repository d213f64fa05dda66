"""The edge MLP's products on several streams at once: each has a workspace of its own."""
import threading

import pytest
import torch

from holonomyawareattention_b200 import PathOrderedGeometricMHA, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_workspace_a_stream():
    dev = torch.device("cuda", torch.cuda.current_device())
    one = ops._gemm_ws(dev)
    assert one is ops._gemm_ws(dev)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        two = ops._gemm_ws(dev)
        assert two is ops._gemm_ws(dev) and two.data_ptr() != one.data_ptr()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        three = ops._gemm_ws(dev)
        assert three.data_ptr() not in (one.data_ptr(), two.data_ptr())
        three.zero_()
    assert ops._gemm_ws(dev) is one


@pytest.mark.parametrize("M,N,K", [(16, 64, 16384), (64, 4512, 768)])      # (few tiles and a long sum: one that may be split)
def test_products_on_two_streams(M, N, K):
    torch.manual_seed(0)
    ins = [(torch.randn(M, K, device=DEV).bfloat16(), torch.randn(K, N, device=DEV).bfloat16(), torch.randn(N, device=DEV)) for _ in range(3)]
    want = [ops.edge_gemm(*i) for i in ins]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        s = torch.cuda.Stream() if k else torch.cuda.current_stream()
        with torch.cuda.stream(s):
            for _ in range(100):
                got = [ops.edge_gemm(*ins[k]) for _ in range(5)]
                s.synchronize()
                if not all(torch.equal(x, want[k]) for x in got):
                    bad.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_modules_trained_on_two_streams():
    """Two modules trained at once, each on a stream and in a thread of its own: the gradients of each alone."""
    torch.manual_seed(1)
    ms = [PathOrderedGeometricMHA(128, n_heads=4, edge_scale=0.1).to(DEV, torch.bfloat16) for _ in range(2)]
    xs = [torch.randn(2, 40, 128, device=DEV).bfloat16() for _ in range(2)]
    mask = torch.ones(40, 40, dtype=torch.bool, device=DEV).tril()

    def grads(k):
        ms[k].zero_grad()
        ms[k](xs[k], attn_mask=mask)[0].float().square().sum().backward()
        return [p.grad for p in ms[k].parameters() if p.grad is not None]

    want = [[g.clone() for g in grads(k)] for k in range(2)]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(10):
                got = grads(k)
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                    bad.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad
    ops.check_status()
