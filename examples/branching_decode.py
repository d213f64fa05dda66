"""One prompt, several continuations: prefill, fork, decode over the shared prompt, retire a branch.

    python examples/branching_decode.py [--d-model 1536 --heads 16 --prompt 4096 --branches 16 --steps 32]

Hidden states are random (the module is one attention layer); the outputs of the first branch are
checked against the module's full forward over the same sequence.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from holonomyawareattention_b200 import PathCache, PathOrderedGeometricMHA, decode, ops, prefill  # noqa: E402


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--d-model", type=int, default=1536)
    ap.add_argument("--heads", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=4096)
    ap.add_argument("--branches", type=int, default=16)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    dev, dt = "cuda", torch.bfloat16
    attn = PathOrderedGeometricMHA(a.d_model, n_heads=a.heads, edge_scale=0.05).to(dev, dt).eval()
    prompt = torch.randn(1, a.prompt, a.d_model, device=dev).to(dt)
    steps = torch.randn(a.steps, a.branches, a.d_model, device=dev).to(dt)
    with torch.no_grad():
        cache = PathCache(attn, rows=a.branches, max_tokens=a.prompt + a.steps)
        prefill(attn, prompt, cache, [0])
        cache.fork([0] * (a.branches - 1), range(1, a.branches))
        shared = cache.share(0)
        ys = []
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        for i in range(a.steps):
            if i == 2:
                ev[0].record()
            ys.append(decode(attn, steps[i], cache)[0])
        ev[1].record()
        ops.check_status()
        torch.cuda.synchronize()
        ms = ev[0].elapsed_time(ev[1]) / max(1, a.steps - 2)
        whole = torch.cat([prompt, steps[:, :1].transpose(0, 1)], 1)
        mask = torch.tril(torch.ones(whole.shape[1], whole.shape[1], dtype=torch.bool, device=dev))
        want = attn(whole, attn_mask=mask)[0][0, a.prompt:]
        err = float((torch.stack(ys).float() - want.float()).norm() / want.float().norm())
        cache.free(range(1, a.branches, 2))
        live = cache.compact()
        ops.check_status()
    print(f"{a.branches} branches over {a.prompt} tokens ({shared} of them read once): {ms:.3f} ms a step, "
          f"rel-L2 against the full forward {err:.2e}; {int(live)} of {cache.n_pages} pages live after retiring half")
    return err


if __name__ == "__main__":
    main()
