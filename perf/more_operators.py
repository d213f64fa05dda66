"""Cases of the training operators: attention's backward pass, the path's backward pass, the AdamW step.

Three operators of one training step of path-ordered attention:

* attn  - gradients of causal attention over transported q^, k^, v^, the probabilities recomputed from
  the forward's log-sum-exp.
* path  - gradients of the generators and of q, k, v through the path products P_t = R_t C_{t / chunk}.
* adamw - one AdamW step over all of a module's tensors, its moments in 32 or in 8 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}
BLOCK = 256                     # elements of a block of 8-bit moments
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the smallest training step: 2 sequences of 128 tokens, 4 heads of 48, fp32
        dict(name="attn_tiny", op="attn", BH=8, Tq=128, Tk=128, off=0, d=48, dtype="f32"),
        # the small model's batch: 64 sequences of 512 tokens, 4 heads of 48, in both types
        dict(name="attn_batch", op="attn", BH=256, Tq=512, Tk=512, off=0, d=48, dtype="bf16"),
        dict(name="attn_batch_f32", op="attn", BH=256, Tq=512, Tk=512, off=0, d=48, dtype="f32"),
        # one sequence of 4096 tokens, 16 heads of 96
        dict(name="attn_long", op="attn", BH=16, Tq=4096, Tk=4096, off=0, d=96, dtype="bf16"),
        # the last shard of a longer sequence, ragged: 1001 queries after 3000 keys
        dict(name="attn_shard", op="attn", BH=16, Tq=1001, Tk=4001, off=3000, d=96, dtype="bf16"),
        # the wide model: 4 sequences of 2048 tokens, 24 heads of 120
        dict(name="attn_wide", op="attn", BH=96, Tq=2048, Tk=2048, off=0, d=120, dtype="bf16"),
        # the smallest training step's path
        dict(name="path_tiny", op="path", B=2, T=128, H=4, d=48, chunk=16, scale=0.05, dtype="f32"),
        # the small model's batch
        dict(name="path_batch", op="path", B=64, T=512, H=4, d=48, chunk=64, scale=0.05, dtype="bf16"),
        # one sequence of 4096 tokens, 16 heads of 96
        dict(name="path_long", op="path", B=1, T=4096, H=16, d=96, chunk=64, scale=0.05, dtype="bf16"),
        # the wide model, 1000 tokens
        dict(name="path_wide", op="path", B=1, T=1000, H=24, d=120, chunk=64, scale=0.05, dtype="bf16"),
        # all trained tensors of the small model (width 192, 4 heads), fp32 throughout
        dict(name="adamw_small", op="adamw", D=192, H=4, shapes=0, dtype="f32", bits=32, step=10, wd=0.01, lr=1e-3),
        # those of the 16-head model (width 1536; its generator layer alone has 448 M weights): bf16, masters, 8-bit moments
        dict(name="adamw_large", op="adamw", D=1536, H=16, shapes=0, dtype="bf16", bits=8, step=100, wd=0.1, lr=3e-4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / (5e14 if case["dtype"] == "bf16" and case["op"] == "attn" else 4e13)


def draw(rng):
    largest = {c["op"]: c for c in sorted(listed(), key=_cost)}
    op = rng.choice(["attn", "attn", "path", "path", "adamw"])
    while True:
        dtype = rng.choice(["bf16", "bf16", "f32"])
        d = rng.choice([5, 8, 16, 20, 24, 32, 40, 48, 50, 56, 64, 72, 80, 96, 96, 104, 112, 120])
        if op == "attn":
            Tq = _log_int(rng, 2, 4096)
            off = 0 if rng.random() < 0.6 else _log_int(rng, 1, 4096)
            Tk = off + Tq + (0 if rng.random() < 0.8 else rng.randint(1, 200))
            c = dict(op=op, BH=_log_int(rng, 1, 256), Tq=Tq, Tk=Tk, off=off, d=d, dtype=dtype)
            fits = c["BH"] * Tq * Tk <= 4.1e8
        elif op == "path":
            T = _log_int(rng, 2, 4096)
            c = dict(op=op, B=_log_int(rng, 1, 64), T=T, H=rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24]), d=d, chunk=min(T, rng.choice([16, 23, 32, 64, 100, 256])),
                     scale=rng.choice([0.05, 0.05, 0.1, 0.5, 1.5]), dtype=dtype)
            fits = c["B"] * T * c["H"] * d * d <= 6.1e8 and c["scale"] * d <= 60
        else:
            c = dict(op=op, D=0, H=0, shapes=rng.randint(1, 10 ** 6), dtype=dtype, bits=rng.choice([8, 32]), step=_log_int(rng, 1, 10000),
                     wd=rng.choice([0.0, 0.01, 0.1]), lr=rng.choice([1e-4, 3e-4, 1e-3]))
            fits = True
        if fits and _cost(c) <= _cost(largest[op]):
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _shapes(case):
    """The tensors of an AdamW case: a module's (width D, H heads), or some of any sizes."""
    if case["shapes"]:
        r = np.random.RandomState(case["shapes"])
        n = int(r.randint(1, 41))
        return [(int(round(math.exp(r.uniform(0, math.log(4e6))))),) for _ in range(n)]
    D, H = case["D"], case["H"]
    d = D // H
    g = H * d * (d - 1) // 2
    return [(3 * D, D), (D, D), (4 * D, 2 * D), (4 * D,), (g, 4 * D), (g,)]


def _seen(case):
    """(Tq, Tk): whether a query sees a key."""
    return torch.arange(case["Tk"], device=DEV)[None, :] <= case["off"] + torch.arange(case["Tq"], device=DEV)[:, None]


def _skew(a, d):
    """(..., d(d-1)/2) -> (..., d, d): the strict upper triangle row by row, and minus it below."""
    i, j = torch.triu_indices(d, d, 1, device=a.device)
    A = torch.zeros(*a.shape[:-1], d, d, dtype=a.dtype, device=a.device)
    A[..., i, j] = a
    return A - A.transpose(-1, -2)


def _expm1(A, squarings):
    """expm(A) - 1 by a Taylor sum of 2^-squarings A and squarings of 1 + E."""
    X = A / 2.0 ** squarings
    E = T = X
    for k in range(2, 10):
        T = torch.matmul(T, X) / k
        E = E + T
    for _ in range(squarings):
        E = 2.0 * E + torch.matmul(E, E)
    return E


def _squarings(case):
    """So many halvings that A, of N(0, 0.3 scale) entries above the diagonal, has a norm below about 0.3."""
    return max(0, math.ceil(math.log2(0.3 * case["scale"] * 2 * math.sqrt(case["d"]) / 0.25)))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if case["op"] == "attn":
        BH, Tq, Tk, d = case["BH"], case["Tq"], case["Tk"], case["d"]
        q, k, v, do = randn(BH, Tq, d).to(dt), randn(BH, Tk, d).to(dt), randn(BH, Tk, d).to(dt), randn(BH, Tq, d).to(dt)
        scale = 1.0 / math.sqrt(d)
        o, lse = torch.empty(BH, Tq, d, device=DEV), torch.empty(BH, Tq, device=DEV)
        seen = _seen(case)
        n = max(1, int(2e8 // (Tq * Tk)))
        for b in range(0, BH, n):                      # what the forward left: o and the log-sum-exp of every row
            s = (torch.matmul(q[b:b + n].float(), k[b:b + n].float().transpose(1, 2)) * scale).masked_fill_(~seen, float("-inf"))
            lse[b:b + n] = torch.logsumexp(s.double() if Tk < 64 else s, -1)
            o[b:b + n] = torch.matmul(torch.softmax(s, -1), v[b:b + n].float())
        return dict(case=case, q=q, k=k, v=v, o=o, lse=lse, do=do, scale=scale)

    if case["op"] == "path":
        B, T, H, d, chunk = case["B"], case["T"], case["H"], case["d"], case["chunk"]
        BH, K = B * H, -(-T // chunk)
        a = 0.3 * randn(B, T, H * (d * (d - 1) // 2))
        # what the forward left: the products R_t within each chunk, and the product C_k in front of each
        R = torch.empty(BH, T, d, d, device=DEV)
        gen = a.view(B, T, H, -1).permute(0, 2, 1, 3).reshape(BH, T, -1)
        at = torch.arange(K, device=DEV) * chunk
        now = torch.eye(d, device=DEV).expand(BH, K, d, d).contiguous()
        sq = _squarings(case)
        for i in range(chunk):
            n = (T - i + chunk - 1) // chunk            # chunks that have an i-th position
            if n <= 0:
                break
            R[:, at[:n] + i] = now[:, :n]
            now[:, :n] += torch.matmul(_expm1(_skew(case["scale"] * gen[:, at[:n] + i], d), sq), now[:, :n])
        C = torch.empty(BH, K, d, d, device=DEV)
        C[:, 0] = torch.eye(d, device=DEV)
        for k in range(1, K):
            C[:, k] = torch.matmul(now[:, k - 1], C[:, k - 1])
        hats = [randn(BH, T, d).to(dt) for _ in range(3)] + [0.3 * randn(BH, T, d)]
        dhats = [(0.05 * randn(BH, T, d)).to(dt) for _ in range(4)]
        return dict(case=case, a=a, R=R, C=C, hats=hats, dhats=dhats)

    shapes = _shapes(case)
    p = [0.02 * randn(*s) for s in shapes]
    grads = [(1e-3 * randn(*s)).to(dt) for s in shapes]
    m = [3e-4 * randn(*s) for s in shapes]
    v = [(1e-3 * randn(*s)).square_() for s in shapes]
    s = dict(case=case, grads=grads, params=p, masters=None, m=m, v=v, scales=None, step=torch.full((1,), case["step"], dtype=torch.int32, device=DEV))
    if case["dtype"] == "bf16":
        s["params"], s["masters"] = [x.to(dt) for x in p], p
    if case["bits"] == 8:
        mq = [_quantise(x, False) for x in m]
        vq = [_quantise(x.sqrt_(), True) for x in v]
        s["m"], s["v"] = [x[0] for x in mq], [x[0] for x in vq]
        s["scales"] = [torch.stack([x[1], y[1]]) for x, y in zip(mq, vq)]
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        from holonomyawareattention_b200 import ops
        if c["op"] == "attn":
            dq, dk, dv = ops.attn_bwd(s["q"], s["k"], s["v"], s["o"], s["lse"], s["do"], s["scale"], q_offset=c["off"])
            return dict(dq=dq, dk=dk, dv=dv)
        if c["op"] == "path":
            da, dqkv = ops.path_bwd(s["a"], s["R"], s["C"], c["chunk"], c["H"], c["scale"], s["hats"], s["dhats"])
            return dict(da=da, dqkv=dqkv)
        ops.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], lr=c["lr"], betas=(0.9, 0.95), eps=1e-8, weight_decay=c["wd"],
                       masters=s["masters"], scales=s["scales"])
        return _adamw_out(s)
    return dict(attn=_plain_attn, path=_plain_path, adamw=_plain_adamw)[c["op"]](s)


def _adamw_out(s):
    some = slice(None) if len(s["params"]) <= 10 else slice(0, 10)     # (of many tensors the first ten)
    keys = ("params", "masters", "m", "v", "scales")
    return {k: s[k][some] for k in keys if s[k] is not None}


def _plain_attn(s):
    c = s["case"]
    q, k, v, do = (s[x].float() for x in ("q", "k", "v", "do"))
    p = torch.matmul(q, k.transpose(1, 2)).mul_(s["scale"]).sub_(s["lse"][..., None]).exp_().masked_fill_(~_seen(c), 0.0)
    dv = torch.matmul(p.transpose(1, 2), do)
    ds = torch.matmul(do, v.transpose(1, 2)).sub_((do * s["o"]).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2), q)
    dt = s["q"].dtype
    return dict(dq=dq.to(dt), dk=dk.to(dt), dv=dv.to(dt))


def _commutator(A, V):
    U = torch.matmul(A, V)
    return U - U.transpose(-1, -2)                     # A V - V A of skew A and V


def _plain_path(s):
    c = s["case"]
    B, T, H, d, chunk = c["B"], c["T"], c["H"], c["d"], c["chunk"]
    BH = B * H
    P = torch.matmul(s["R"], s["C"][:, torch.arange(T, device=DEV) // chunk])
    qh, kh, vh, o = (x.float() for x in s["hats"])
    dqh, dkh, dvh, doh = (x.float() for x in s["dhats"])
    X, Y = torch.stack([qh, kh, vh, doh], 2), torch.stack([dqh, dkh, dvh, o], 2)           # (BH, T, 4, d)
    Z = torch.matmul(X.transpose(2, 3), Y)
    Z = Z - Z.transpose(2, 3)
    # the sums over all later positions, in 64 bits: they run over thousands of terms
    after = Z.sum(1, keepdim=True, dtype=torch.float64) - Z.cumsum(1, dtype=torch.float64)
    W = torch.matmul(torch.matmul(P, after.float()), P.transpose(2, 3))
    del after, Z
    gen = s["a"].view(B, T, H, -1).permute(0, 2, 1, 3).reshape(BH, T, -1)
    n = _squarings(c)
    A = _skew(c["scale"] / 2.0 ** n * gen, d)
    # phi(ad_A) W = sum_k ad_A^k W / (k + 1)! of A / 2^n, doubled n times: phi(2 z) = phi(z) (1 + e^z) / 2
    M, V = W, W
    for k in range(1, 9):
        V = _commutator(A, V) / (k + 1)
        M = M + V
    E = _expm1(A, 0) if n else None
    for _ in range(n):
        U = M + torch.matmul(E, M)                      # G M G^T, G = 1 + E
        M = 0.5 * (M + U + torch.matmul(U, E.transpose(2, 3)))
        E = 2.0 * E + torch.matmul(E, E)
    i, j = torch.triu_indices(d, d, 1, device=DEV)
    da = c["scale"] * M[..., i, j]
    da[:, T - 1] = 0.0                                  # the closing edge is not on any path
    da = da.view(B, H, T, -1).permute(0, 2, 1, 3).reshape(B, T, -1)
    dqkv = torch.matmul(P, torch.stack([dqh, dkh, dvh], 3)).view(B, H, T, d, 3).permute(0, 2, 1, 4, 3).reshape(B, T, 3 * H * d)
    return dict(da=da, dqkv=dqkv.to(s["dhats"][0].dtype))


def _quantise(x, root):
    """(e4m3 values, the scale of each block of 256): the largest magnitude of a block stands at 448.  Roots that are
    not zero stay at least at the smallest e4m3 value, 2^-9."""
    n = x.numel()
    b = torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)
    scale = b.abs().amax(1) / 448.0
    q = torch.where(scale[:, None] > 0, b / scale[:, None], 0.0)
    if root:
        q = torch.where(b > 0, q.clamp(min=2.0 ** -9), q)
    return q.to(E4M3).reshape(-1)[:n].view(x.shape), scale


def _values(q, scale):
    n = q.numel()
    b = torch.nn.functional.pad(q.reshape(-1).float(), (0, -n % BLOCK)).view(-1, BLOCK) * scale[:, None]
    return b.reshape(-1)[:n].view(q.shape)


def _plain_adamw(s):
    [_plain_adamw_one(s, i) for i in range(len(s["params"]))]
    return _adamw_out(s)


def _plain_adamw_one(s, i):
    c = s["case"]
    b1, b2, eps = 0.9, 0.95, 1e-8
    p = s["params"][i] if s["masters"] is None else s["masters"][i]
    g, m, v = s["grads"][i].float(), s["m"][i], s["v"][i]
    step = s["step"].double()
    c1, c2 = 1.0 - b1 ** step, (1.0 - b2 ** step).sqrt()
    if s["scales"] is not None:
        m, v = _values(m, s["scales"][i][0]), _values(v, s["scales"][i][1]).square()
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    r = v.sqrt()
    p.copy_(p * (1.0 - c["lr"] * c["wd"]) - (m / (r / c2.float() + eps)) * (c["lr"] / c1).float())
    if s["masters"] is not None:
        s["params"][i].copy_(p)
    if s["scales"] is None:
        s["m"][i].copy_(m)
        s["v"][i].copy_(v)
        return
    (mq, ms), (vq, vs) = _quantise(m, False), _quantise(r, True)
    s["m"][i].copy_(mq)
    s["v"][i].copy_(vq)
    s["scales"][i][0].copy_(ms)
    s["scales"][i][1].copy_(vs)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "attn":
        BH, Tq, Tk, off, d = case["BH"], case["Tq"], case["Tk"], case["off"], case["d"]
        pairs = BH * (Tq * off + Tq * (Tq + 1) / 2.0)
        # q, do, dq of every query, k, v, dk, dv of every key that a query sees or not, o and the log-sum-exp; five products
        return {"bytes": BH * (3.0 * Tq * d * e + 4.0 * Tk * d * e + Tq * (d + 1) * 4.0), "flops": 10.0 * pairs * d}
    if case["op"] == "path":
        d = case["d"]
        n = float(case["B"]) * case["T"] * case["H"]
        # R, the generators and their gradients in fp32, o in fp32, seven vectors in and three out; two products for W, four for its commutators
        return {"bytes": n * (d * d * 4 + d * (d - 1) * 4 + 4.0 * d + 10.0 * d * e), "flops": n * 12.0 * d ** 3}
    n = float(sum(math.prod(s) for s in _shapes(case)))
    moments = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
    return {"bytes": n * (e + moments + (8.0 if case["dtype"] == "f32" else 10.0)), "flops": 15.0 * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "attn":
        BH, Tq, Tk, d = case["BH"], case["Tq"], case["Tk"], case["d"]
        if float(BH) * Tq * Tk * d > 1e11:
            return None
        s = prepare(case, seed)
        unseen = torch.ones(Tq, Tk, dtype=torch.bool, device=DEV).triu(case["off"] + 1)
        out = [torch.empty(BH, t, d, dtype=torch.float64, device=DEV) for t in (Tq, Tk, Tk)]
        for b in range(BH):
            q, k, v = (s[x][b].double().requires_grad_() for x in ("q", "k", "v"))
            z = (q @ k.t() * s["scale"]).masked_fill(unseen, float("-inf"))
            loss = ((torch.softmax(z, -1) @ v) * s["do"][b].double()).sum()
            for into, g in zip(out, torch.autograd.grad(loss, (q, k, v))):
                into[b] = g
        return dict(dq=out[0], dk=out[1], dv=out[2])
    if case["op"] == "path":
        B, T, H, d, chunk = case["B"], case["T"], case["H"], case["d"], case["chunk"]
        if float(B) * T * H * d ** 3 > 7e10:
            return None
        s = prepare(case, seed)
        m = d * (d - 1) // 2
        rows, cols = (torch.from_numpy(x).to(DEV) for x in np.triu_indices(d, 1))
        da = torch.zeros(B, T, H, m, dtype=torch.float64, device=DEV)
        dqkv = torch.empty(B, T, H, 3, d, dtype=torch.float64, device=DEV)
        step = max(1, int(2e7 // (d * d)))
        for c in range(B * H):
            b, h = divmod(c, H)
            at = s["C"][c].double().repeat_interleave(chunk, 0)[:T]
            vec = [x[c].double() for x in s["hats"]] + [x[c].double() for x in s["dhats"]]
            later = torch.zeros(d, d, dtype=torch.float64, device=DEV)
            for t1 in range(T, 0, -step):
                t0 = max(0, t1 - step)
                P = torch.bmm(s["R"][c, t0:t1].double(), at[t0:t1])
                for w in range(3):
                    dqkv[b, t0:t1, h, w] = torch.einsum("tij,tj->ti", P, vec[4 + w][t0:t1])
                out_grad = torch.einsum("tij,tj->ti", P, vec[7][t0:t1])
                dP = sum(torch.einsum("ti,tj->tij", torch.einsum("tij,tj->ti", P, vec[w][t0:t1]), vec[4 + w][t0:t1]) for w in range(3))
                dP = dP + torch.einsum("ti,tj->tij", out_grad, vec[3][t0:t1])
                own_part = torch.bmm(P.transpose(1, 2), dP)
                total = own_part.flip(0).cumsum(0).flip(0)                 # of this position and those after it, in this range
                Z = torch.cat([total[1:], torch.zeros_like(total[:1])]) + later
                later = later + total[0]
                W = torch.bmm(torch.bmm(P, Z), P.transpose(1, 2))
                A = torch.zeros(t1 - t0, d, d, dtype=torch.float64, device=DEV)
                gen = s["a"].view(B, T, H, m)[b, t0:t1, h].double() * case["scale"]
                A[:, rows, cols], A[:, cols, rows] = gen, -gen
                # expm([[A, W], [0, A]]) has the integral of e^{(1-u) A} W e^{u A} above its diagonal
                big = torch.zeros(t1 - t0, 2 * d, 2 * d, dtype=torch.float64, device=DEV)
                big[:, :d, :d], big[:, d:, d:], big[:, :d, d:] = A, A, W
                big = torch.linalg.matrix_exp(big)
                M = torch.bmm(big[:, :d, d:], big[:, :d, :d].transpose(1, 2))
                da[b, t0:t1, h] = case["scale"] * (M[:, rows, cols] - M[:, cols, rows])
        da[:, T - 1] = 0.0
        return dict(da=da.view(B, T, H * m), dqkv=dqkv.view(B, T, 3 * H * d))
    s = prepare(case, seed)
    out = dict(params=[], masters=[], m=[], v=[], scales=[])
    for i in range(min(10, len(s["params"]))):
        x = (s["params"] if s["masters"] is None else s["masters"])[i].double()
        g = s["grads"][i].double()
        if s["scales"] is None:
            m, v = s["m"][i].double(), s["v"][i].double()
        else:
            n = g.numel()
            m, r = (t[i].double().reshape(-1) * s["scales"][i][w].double().repeat_interleave(BLOCK)[:n] for w, t in enumerate((s["m"], s["v"])))
            m, v = m.view(g.shape), r.square().view(g.shape)
        m = 0.9 * m + (1 - 0.9) * g
        v = 0.95 * v + (1 - 0.95) * g * g
        x = x - case["lr"] * (case["wd"] * x + m / (1 - 0.9 ** case["step"]) / (torch.sqrt(v / (1 - 0.95 ** case["step"])) + 1e-8))
        out["params"].append(x)
        out["masters"].append(x)
        if s["scales"] is None:
            out["m"].append(m)
            out["v"].append(v)
        else:                                                              # (the 8-bit values have no such value; their scales have)
            pad = lambda t: torch.nn.functional.pad(t.reshape(-1), (0, -t.numel() % BLOCK)).view(-1, BLOCK)  # noqa: E731
            out["m"].append(None)
            out["v"].append(None)
            out["scales"].append(torch.stack([pad(m).abs().amax(1), pad(v.sqrt()).amax(1)]) / 448.0)
    return {k: v for k, v in out.items() if s.get(k) is not None}
