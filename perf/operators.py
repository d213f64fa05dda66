"""Cases of the serving operators: pages of the cache, paged attention with a shared prefix, the path step.

Three operators of one decode loop over path-ordered attention:

* pages  - the cache's pages: forking sequences ("fork") and retiring them, i.e. freeing
  rows and compacting the pool ("retire").
* attn   - attention of a batch over a prefix that all rows share and each row's own pages.
* step   - one token's path step: P' = expm(skew(s a)) P, q^ = P'^T q, and k^ = P'^T k,
  v^ = P'^T v written to the row's page.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a small model (4 heads of 48) with short pages: four candidates branch from two sequences
        dict(name="fork_small", op="fork", S=8, W=8, n_pages=64, page=16, H=4, d=48, layers=1, n=4, parents=2, dtype="f32"),
        # 64 candidates branch from 4 long prompts (up to 8192 tokens) of a 16-head model of width 1536
        dict(name="fork_large", op="fork", S=160, W=160, n_pages=1024, page=64, H=16, d=96, layers=2, n=64, parents=4, dtype="bf16"),
        # three of eight short sequences end, the pool closes up
        dict(name="retire_small", op="retire", S=8, W=8, n_pages=64, page=16, H=4, d=48, layers=1, n=3, parents=8, dtype="f32"),
        # half of 128 sequences end; a pool of 262144 tokens closes up so that its tail can be given back
        dict(name="retire_large", op="retire", S=128, W=64, n_pages=4096, page=64, H=16, d=96, layers=1, n=64, parents=128, dtype="bf16"),
        # the smallest decode step: two rows of the small model in fp32, with the inverse transport
        dict(name="attn_tiny", op="attn", B=2, Tq=1, H=4, Hk=4, d=48, page=16, shared=8, W=4, lo=1, hi=64, dtype="f32", paths=True),
        # a decode step of the 16-head model at 4096 shared tokens, 16 rows that have gone on for up to 1024
        dict(name="attn_decode", op="attn", B=16, Tq=1, H=16, Hk=16, d=96, page=64, shared=64, W=16, lo=1, hi=1024, dtype="bf16", paths=True),
        # eight questions about one document of 65536 tokens
        dict(name="attn_long", op="attn", B=8, Tq=1, H=16, Hk=16, d=96, page=64, shared=1024, W=64, lo=1, hi=4096, dtype="bf16", paths=False),
        # the wide model (24 heads of 120), 128 rows over a shared prompt of 2048 tokens
        dict(name="attn_wide", op="attn", B=128, Tq=1, H=24, Hk=24, d=120, page=64, shared=32, W=8, lo=1, hi=512, dtype="bf16", paths=True),
        # prompts of 128 tokens after a shared prefix of 4096, one row shorter than its prompt, one empty
        dict(name="attn_prompt", op="attn", B=16, Tq=128, H=16, Hk=16, d=96, page=64, shared=64, W=10, lo=64, hi=640, dtype="bf16", paths=False),
        # the smallest path step: two rows of the small model in fp32
        dict(name="step_tiny", op="step", B=2, H=4, d=48, page=16, W=4, scale=0.05, dtype="f32"),
        # 16 rows of the 16-head model
        dict(name="step_rows", op="step", B=16, H=16, d=96, page=64, W=4, scale=0.05, dtype="bf16"),
        # 128 rows of the wide model
        dict(name="step_wide", op="step", B=128, H=24, d=120, page=64, W=2, scale=0.05, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """About the seconds of a pass: short head dims are paid for as 64, the softmax has them whole."""
    w = work(case)
    rate = 5e13 if case["op"] == "step" or case["dtype"] == "f32" else 6e14
    return w["bytes"] / 5e12 + w["flops"] * max(1.0, 64 / case["d"]) / rate


def draw(rng):
    largest = {c["op"]: c for c in sorted(listed(), key=_cost)}
    op = rng.choice(["fork", "retire", "attn", "attn", "step", "step"])
    while True:
        dtype = rng.choice(["bf16", "bf16", "f32"])
        page = rng.choice([16, 32, 48, 64, 128])
        d = rng.choice([8, 16, 20, 24, 32, 40, 48, 56, 64, 72, 80, 96, 104, 112, 120])
        H = rng.choice([1, 2, 3, 4, 6, 8, 12, 16, 24])
        if op in ("fork", "retire"):
            S = _log_int(rng, 4, 200)
            W = _log_int(rng, 2, 200)
            n_pages = _log_int(rng, 32, 4096)
            c = dict(op=op, S=S, W=W, n_pages=n_pages, page=page, H=H, d=d, layers=rng.randint(1, 3), n=rng.randint(1, max(1, S // 2)),
                     parents=rng.randint(1, max(1, S // 3)) if op == "fork" else rng.randint(max(1, S // 2), S), dtype=dtype)
            if op == "retire":
                c["n"] = min(c["n"], c["parents"])
        elif op == "attn":
            Hk = rng.choice([h for h in (1, 2, 3, 4, 6, 8, 12, 16, 24) if H % h == 0])
            Tq = 1 if rng.random() < 0.6 else _log_int(rng, 2, 300)
            W = _log_int(rng, 1, max(2, 4096 // page))
            hi = rng.randint(max(1, W * page // 2), W * page)
            shared = 0 if rng.random() < 0.15 else _log_int(rng, 1, 65536 // page)
            c = dict(op=op, B=_log_int(rng, 1, 160), Tq=Tq, H=H, Hk=Hk, d=d, page=page, shared=shared, W=W, lo=rng.randint(0, hi), hi=hi, dtype=dtype,
                     paths=Tq == 1 and rng.random() < 0.5)
        else:
            c = dict(op=op, B=_log_int(rng, 1, 160), H=H, d=d, page=page, W=_log_int(rng, 1, 8), scale=rng.choice([0.05, 0.05, 0.1, 0.5, 1.5]), dtype=dtype)
        pool = c.get("n_pages", 0) * page * H * d * SIZE[dtype] * 2 * c.get("layers", 0)
        if _cost(c) <= _cost(largest[op]) and pool <= 1.7e9:
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _host_lens(case, seed):
    """The attention rows' lengths after the prefix and the whole lengths, as the seed has them."""
    r = np.random.RandomState(seed % (2 ** 31))
    B, Tq = case["B"], case["Tq"]
    own_len = r.randint(case["lo"], case["hi"] + 1, size=B).astype(np.int64)
    total = own_len + case["shared"] * case["page"]
    if B >= 8:
        own_len[B // 2], total[B // 2] = 0, 0           # a row that waits for a request
        if case["shared"]:
            total[B // 3] = max(1, total[B // 3] - own_len[B // 3] - case["page"] // 2)   # a row that ends inside the prefix
            own_len[B // 3] = 0
        if Tq > 1:                                      # a row shorter than its queries
            own_len[0], total[0] = max(1, Tq // 2), case["shared"] * case["page"] + max(1, Tq // 2)
            own_len[0] = min(own_len[0], case["W"] * case["page"])
            total[0] = min(total[0], case["shared"] * case["page"] + own_len[0])
    return own_len, total


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).to(DEV)


def _cache_state(case, seed):
    """Sequences with their pages scattered over the pool: table, lens, refs, as numpy."""
    r = np.random.RandomState(seed % (2 ** 31))
    S, W, n_pages, page = case["S"], case["W"], case["n_pages"], case["page"]
    seqs = case["parents"]
    spare = case["n"] if case["op"] == "fork" else 0
    room = max(seqs, n_pages - spare)
    table = np.full((S, W), -1, np.int64)
    lens = np.zeros(S, np.int64)
    refs = np.zeros(n_pages, np.int64)
    rows = r.permutation(S)
    most = max(1, min(W, room // max(1, seqs)))
    if case["op"] == "fork":                             # few parents, long ones
        most = max(1, min(W, 128, (room // 2) // max(1, seqs)))
    pages = r.permutation(n_pages)
    at = 0
    shared = None
    for i in range(seqs):
        if at >= n_pages - spare:
            seqs = max(1, i)
            break
        used = int(r.randint(max(1, most // 2), most + 1))
        used = min(used, n_pages - spare - at)
        row = rows[i]
        take = pages[at:at + used].copy()
        if case["op"] == "retire" and shared is not None and i % 2 == 1 and used > 1 and len(shared) > 1:
            k = min(used, len(shared)) // 2              # every other row shares the first pages of the one before
            take[:k] = shared[:k]
        table[row, :used] = take
        lens[row] = int(r.randint((used - 1) * page + 1, used * page + 1))
        refs[take] += 1
        shared = take
        at += used
    return table, lens, refs, rows, seqs, r


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[case["dtype"]]
    d, page = case["d"], case["page"]

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    if case["op"] in ("fork", "retire"):
        table, lens, refs, rows, seqs, r = _cache_state(case, seed)
        pools = [randn(case["n_pages"], case["H"], page, d).to(dt) for _ in range(2 * case["layers"])]
        s = dict(case=case, pools=pools, table=_ints(table), lens=_ints(lens), refs=_ints(refs))
        if case["op"] == "fork":
            n = min(case["n"], case["S"] - seqs)
            s["src"] = _ints(rows[:seqs][r.randint(0, seqs, size=n)])
            s["dst"] = _ints(rows[seqs:seqs + n])
        else:
            s["rows"] = _ints(r.permutation(rows[:seqs])[:min(case["n"], seqs)])
        return s

    if case["op"] == "attn":
        B, Tq, H, Hk, W, shared = case["B"], case["Tq"], case["H"], case["Hk"], case["W"], case["shared"]
        own_len, total = _host_lens(case, seed)
        need = -(-own_len // page)
        n_pages = int(shared + need.sum()) + 3
        order = np.random.RandomState((seed + 1) % (2 ** 31)).permutation(n_pages)
        table = np.full((B, W), -1, np.int64)
        at = shared
        for b in range(B):
            table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
        k_pages, v_pages = (randn(n_pages, Hk, page, d).to(dt) for _ in range(2))
        # slots that no token was written to hold whatever was there before: here NaN
        full = np.zeros((n_pages, page), bool)
        full[order[:shared]] = True
        for b in range(B):
            for j in range(int(need[b])):
                full[table[b, j], :max(0, min(page, int(own_len[b]) - j * page))] = True
        empty = torch.from_numpy(~full).to(DEV)[:, None, :, None]
        k_pages.masked_fill_(empty, float("nan"))
        v_pages.masked_fill_(empty, float("nan"))
        s = dict(case=case, q=(1.5 * randn(B, Tq, H, d)).to(dt), k_pages=k_pages, v_pages=v_pages, table=_ints(table), lens=_ints(total),
                 shared=_ints(order[:shared]), scale=1.0 / math.sqrt(d), paths=None)
        if case["paths"]:
            s["paths"] = _rotations(B * H, d, g).view(B, H, d, d)
        return s

    B, H, W = case["B"], case["H"], case["W"]
    r = np.random.RandomState(seed % (2 ** 31))
    lens = r.randint(1, W * page + 1, size=B)
    lens[0] = max(1, W * page - 1)
    if B > 2:
        lens[1], lens[2] = 0, 1                          # a row without a request, and a row at its first token
    table = r.permutation(B * W + 2)[:B * W].reshape(B, W)
    m = d * (d - 1) // 2
    return dict(case=case, a=0.3 * randn(B, H * m), P=_rotations(B * H, d, g).view(B, H, d, d), qkv=randn(B, 3 * H * d).to(dt),
                k_pages=randn(B * W + 2, H, page, d).to(dt), v_pages=randn(B * W + 2, H, page, d).to(dt), table=_ints(table), lens=_ints(lens))


def _rotations(n, d, g):
    """n orthogonal d x d matrices: a few drawn ones, their rows permuted and signs changed."""
    few = min(n, 16)
    q = torch.linalg.qr(torch.randn(few, d, d, device=DEV, generator=g))[0]
    out = q[torch.arange(n, device=DEV) % few]
    order = torch.rand(n, d, device=DEV, generator=g).argsort(1)
    sign = torch.randint(0, 2, (n, d, 1), device=DEV, generator=g).float() * 2 - 1
    return (torch.gather(out, 1, order[:, :, None].expand(n, d, d)) * sign).contiguous()


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        from holonomyawareattention_b200 import ops
        c = s["case"]
        if op == "fork":
            table, lens, refs = ops.pages_fork(s["pools"], s["table"], s["lens"], s["refs"], s["src"], s["dst"], c["page"])
            return dict(table=table, lens=lens, refs=refs, pools=s["pools"])
        if op == "retire":
            table, lens, refs = ops.pages_free(s["table"], s["lens"], s["refs"], s["rows"], c["page"])
            table, refs, live = ops.pages_compact(s["pools"], table, refs)
            return dict(table=table, lens=lens, refs=refs, live=live, pools=s["pools"])
        if op == "attn":
            out, lse = ops.paged_attn_fwd(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["scale"], shared=s["shared"], paths=s["paths"])
            return dict(out=out, lse=lse)
        P, qh = ops.path_step(s["a"], s["P"], s["qkv"], c["H"], c["scale"], s["k_pages"], s["v_pages"], s["table"], s["lens"])
        return dict(P=P, qh=qh, k_pages=s["k_pages"], v_pages=s["v_pages"])
    return dict(fork=_plain_fork, retire=_plain_retire, attn=_plain_attn, step=_plain_step)[op](s)


def _plain_fork(s):
    page, table, lens, refs = s["case"]["page"], s["table"].long(), s["lens"].long(), s["refs"].long()
    src, dst = s["src"].long(), s["dst"].long()
    W = table.shape[1]
    full, part = lens[src] // page, lens[src] % page > 0
    free = torch.argsort((refs > 0).to(torch.int8), stable=True)         # free pages first, in their order
    fresh = free[torch.cumsum(part, 0) - part.long()]
    rows = table[src]
    old = rows.gather(1, (full + part.long() - 1).clamp(min=0)[:, None])[:, 0]      # the last page; one that is full goes onto itself
    into = torch.where(part, fresh, old)
    col = torch.arange(W, device=DEV)[None, :]
    keep = col < full[:, None]
    rows = torch.where((col == full[:, None]) & part[:, None], into[:, None], rows)
    table, lens, refs = table.clone(), lens.clone(), refs.clone()
    lens[dst] = lens[src]
    table[dst] = rows
    refs.index_add_(0, rows.clamp(min=0).reshape(-1), (keep | ((col == full[:, None]) & part[:, None])).long().reshape(-1))
    s["pools"] = [p.index_copy_(0, into, p[old]) for p in s["pools"]]
    return dict(table=table.int(), lens=lens.int(), refs=refs.int(), pools=s["pools"])


def _plain_retire(s):
    page, table, lens, refs, rows = s["case"]["page"], s["table"].long(), s["lens"].long(), s["refs"].long(), s["rows"].long()
    n_pages = refs.numel()
    col = torch.arange(table.shape[1], device=DEV)[None, :]
    used = col * page < lens[rows][:, None]
    refs = refs.index_add(0, table[rows].clamp(min=0).reshape(-1), -used.long().reshape(-1))
    table, lens = table.clone(), lens.clone()
    table[rows], lens[rows] = -1, 0
    live = refs > 0
    count = live.sum()
    idx = torch.arange(n_pages, device=DEV)
    hole, mover = ~live & (idx < count), live & (idx >= count)
    holes = torch.argsort((~hole).to(torch.int8), stable=True)           # the holes first, in their order
    movers = torch.argsort((~mover).to(torch.int8), stable=True)
    moves = mover.sum()
    src, dst = movers[:n_pages // 2 + 1], holes[:n_pages // 2 + 1]
    on = torch.arange(src.numel(), device=DEV) < moves
    src, dst = src[on], dst[on]
    to = idx.clone()
    to[src] = dst
    table = torch.where(table >= 0, to[table.clamp(min=0)], table)
    new_refs = torch.where(idx < count, refs, torch.zeros_like(refs))
    new_refs[dst] = refs[src]
    s["pools"] = [p.index_copy_(0, dst, p[src]) for p in s["pools"]]
    return dict(table=table.int(), lens=lens.int(), refs=new_refs.int(), live=count.int().reshape(1), pools=s["pools"])


def _plain_attn(s):
    q, table, lens, shared = s["q"].float(), s["table"].long(), s["lens"].long(), s["shared"].long()
    B, Tq, H, d = q.shape
    Hk, page = s["k_pages"].shape[1:3]
    G, Ls, W = H // Hk, shared.numel() * page, table.shape[1]
    seen = (lens[:, None] - Tq + 1 + torch.arange(Tq, device=DEV)[None, :]).clamp(min=0)       # (B, Tq): keys that a query sees
    qg = q.view(B, Tq, Hk, G, d)
    kp, vp = (t[shared].float().permute(1, 0, 2, 3).reshape(Hk, Ls, d) for t in (s["k_pages"], s["v_pages"]))
    s1 = torch.matmul(qg.permute(2, 0, 1, 3, 4).reshape(Hk, B * Tq * G, d), kp.transpose(1, 2)) * s["scale"]
    s1 = s1.view(Hk, B, Tq, G, Ls).masked_fill_((torch.arange(Ls, device=DEV) >= seen[:, :, None])[None, :, :, None, :], float("-inf"))
    there = (Ls + torch.arange(W * page, device=DEV) < lens[:, None])[:, None, :, None]
    ks, vs = (t[table.clamp(min=0)].float().permute(0, 2, 1, 3, 4).reshape(B, Hk, W * page, d) for t in (s["k_pages"], s["v_pages"]))
    ks, vs = torch.where(there, ks, 0.0), torch.where(there, vs, 0.0)
    s2 = torch.matmul(qg.permute(0, 2, 1, 3, 4).reshape(B, Hk, Tq * G, d), ks.transpose(2, 3)) * s["scale"]
    s2 = s2.view(B, Hk, Tq, G, W * page).permute(1, 0, 2, 3, 4)
    s2 = s2.masked_fill((Ls + torch.arange(W * page, device=DEV) >= seen[:, :, None])[None, :, :, None, :], float("-inf"))
    top = s2.amax(-1) if Ls == 0 else torch.maximum(s1.amax(-1), s2.amax(-1))                  # (Hk, B, Tq, G)
    m = torch.where(torch.isinf(top), 0.0, top)
    p1, p2 = torch.exp(s1 - m[..., None]), torch.exp(s2 - m[..., None])
    l = p1.sum(-1) + p2.sum(-1)
    o = torch.matmul(p1.reshape(Hk, B * Tq * G, Ls), vp).view(Hk, B, Tq, G, d)
    o = o + torch.matmul(p2.permute(1, 0, 2, 3, 4).reshape(B, Hk, Tq * G, W * page), vs).view(B, Hk, Tq, G, d).permute(1, 0, 2, 3, 4)
    o = torch.where(l[..., None] > 0, o / l[..., None], 0.0)
    out = o.permute(1, 2, 0, 3, 4).reshape(B, Tq, H, d)
    lse = (m + torch.log(l)).permute(1, 2, 0, 3).reshape(B, Tq, H)
    if s["paths"] is not None:
        out = torch.matmul(s["paths"], out.view(B, H, d, 1)).view(B, 1, H, d)
    return dict(out=out.to(s["q"].dtype), lse=lse.contiguous())


def _plain_step(s):
    c = s["case"]
    B, H, d, page = c["B"], c["H"], c["d"], c["page"]
    table, lens = s["table"].long(), s["lens"].long()
    i, j = torch.triu_indices(d, d, 1, device=DEV)
    A = torch.zeros(B, H, d, d, device=DEV)
    A[:, :, i, j] = c["scale"] * s["a"].view(B, H, -1)
    A = A - A.transpose(2, 3)
    # expm by scaling and squaring: 2^-6 of A in a Taylor sum, then the six squarings on E = G - 1
    X = A / 64.0
    E = X
    T = X
    for k in (2, 3, 4, 5, 6, 7, 8):
        T = torch.matmul(T, X) / k
        E = E + T
    for _ in range(6):
        E = 2.0 * E + torch.matmul(E, E)
    P = s["P"] + torch.matmul(E, s["P"])
    P = torch.where((lens == 1)[:, None, None, None], torch.eye(d, device=DEV), P)             # the first token: no edge
    P = torch.where((lens == 0)[:, None, None, None], s["P"], P)                               # no token: unchanged
    q, k, v = s["qkv"].float().view(B, H, 3, d).unbind(2)
    qh, kh, vh = (torch.matmul(P.transpose(2, 3), t[..., None])[..., 0] for t in (q, k, v))
    live = lens > 0
    qh = torch.where(live[:, None, None], qh, 0.0).to(s["qkv"].dtype)
    pos = (lens - 1).clamp(min=0)
    at = table.gather(1, (pos // page)[:, None])[:, 0]
    slot = pos % page
    for pool, x in ((s["k_pages"], kh), (s["v_pages"], vh)):
        pool[at, :, slot] = torch.where(live[:, None, None], x.to(pool.dtype), pool[at, :, slot])
    return dict(P=P, qh=qh, k_pages=s["k_pages"], v_pages=s["v_pages"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = SIZE[case["dtype"]]
    d, page = case["d"], case["page"]
    if case["op"] in ("fork", "retire"):
        table, lens, refs, rows, seqs, r = _cache_state(case, 1)
        payload = case["H"] * page * d * e * 2 * case["layers"]
        books = 8.0 * (table.size + lens.size + refs.size)
        if case["op"] == "fork":
            n = min(case["n"], case["S"] - seqs)
            src = rows[:seqs][r.randint(0, seqs, size=n)]
            moved = int((lens[src] % page > 0).sum())
        else:
            gone = r.permutation(rows[:seqs])[:min(case["n"], seqs)]
            for row in gone:
                used = -(-int(lens[row]) // page)
                np.subtract.at(refs, table[row, :used], 1)
            live = refs > 0
            moved = int(live[int(live.sum()):].sum())
        return {"bytes": books + 2.0 * moved * payload, "flops": 0.0}
    if case["op"] == "attn":
        own_len, total = _host_lens(case, 1)
        B, Tq, H, Hk = case["B"], case["Tq"], case["H"], case["Hk"]
        keys = case["shared"] * page + float(own_len.sum())
        seen = float(np.clip(total[:, None] - Tq + 1 + np.arange(Tq)[None, :], 0, None).sum())
        b = keys * Hk * 2 * d * e + B * Tq * H * (2 * d * e + 4) + (B * H * d * d * 4.0 if case["paths"] else 0.0)
        return {"bytes": b, "flops": 4.0 * seen * H * d + (2.0 * B * H * d * d if case["paths"] else 0.0)}
    units = case["B"] * case["H"]
    # three products for the exponential, one for the composition, three matrix-vector products
    return {"bytes": units * (d * (d - 1) / 2 * 4 + 2 * d * d * 4 + 6.0 * d * e), "flops": units * (8.0 * d ** 3 + 6.0 * d * d)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d, page = case["d"], case["page"]
    if case["op"] in ("fork", "retire"):
        # the payload, page by page, as the bookkeeping on the host says
        table, lens, refs = (s[k].cpu().numpy().copy() for k in ("table", "lens", "refs"))
        pools = s["pools"]
        if case["op"] == "fork":
            free = iter(np.flatnonzero(refs == 0))
            for a in s["src"].cpu().numpy():
                if lens[a] % page:
                    new = int(next(free))
                    for p in pools:
                        p[new] = p[int(table[a, lens[a] // page])]
            return dict(table=None, lens=None, refs=None, pools=[p.double() for p in pools])
        for a in s["rows"].cpu().numpy():
            for j in range(-(-int(lens[a]) // page)):
                refs[table[a, j]] -= 1
        count = int((refs > 0).sum())
        for hole, mover in zip(np.flatnonzero(refs[:count] == 0), count + np.flatnonzero(refs[count:] > 0)):
            for p in pools:
                p[int(hole)] = p[int(mover)]
        return dict(table=None, lens=None, refs=None, live=None, pools=[p.double() for p in pools])
    if case["op"] == "attn":
        B, Tq, H, Hk = case["B"], case["Tq"], case["H"], case["Hk"]
        if float(B) * Tq * H * (case["shared"] + case["W"]) * page * d > 4e12:
            return None
        out = torch.zeros(B, Tq, H, d, dtype=torch.float64, device=DEV)
        lse = torch.full((B, Tq, H), float("-inf"), dtype=torch.float64, device=DEV)
        table, lens, shared = s["table"].cpu().tolist(), s["lens"].cpu().tolist(), s["shared"].cpu().tolist()
        for b in range(B):
            if lens[b] == 0:
                continue
            ids = torch.tensor((shared + [t for t in table[b] if t >= 0])[:-(-lens[b] // page)], device=DEV)
            for h in range(Hk):
                k, v = (t[ids, h].reshape(-1, d)[:lens[b]].double() for t in (s["k_pages"], s["v_pages"]))
                g = slice(h * (H // Hk), (h + 1) * (H // Hk))
                z = torch.einsum("tgd,jd->tgj", s["q"][b, :, g].double(), k) * s["scale"]
                pos = lens[b] - Tq + torch.arange(Tq, device=DEV)
                z[(torch.arange(lens[b], device=DEV)[None, :] > pos[:, None])[:, None, :].expand_as(z)] = float("-inf")
                lse[b, :, g] = torch.logsumexp(z, -1)
                out[b, :, g] = torch.einsum("tgj,jd->tgd", torch.nan_to_num(torch.softmax(z, -1), nan=0.0), v)
        if s["paths"] is not None:
            out = torch.einsum("bhij,bthj->bthi", s["paths"].double(), out)
        return dict(out=out, lse=lse)
    B, H = case["B"], case["H"]
    if float(B) * H * d ** 3 > 3e10:
        return None
    a = s["a"].double().view(B, H, -1) * case["scale"]
    rows, cols = np.triu_indices(d, 1)
    A = torch.zeros(B, H, d * d, dtype=torch.float64, device=DEV)
    A[:, :, torch.from_numpy(rows * d + cols).to(DEV)] = a
    A[:, :, torch.from_numpy(cols * d + rows).to(DEV)] = -a
    P = torch.einsum("bhij,bhjk->bhik", torch.linalg.matrix_exp(A.view(B, H, d, d)), s["P"].double())
    lens, table = s["lens"].cpu().tolist(), s["table"].cpu().tolist()
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    qh = torch.zeros(B, H, d, dtype=torch.float64, device=DEV)
    qkv = s["qkv"].double().view(B, H, 3, d)
    for b in range(B):
        if lens[b] == 0:
            P[b] = s["P"][b].double()
            continue
        if lens[b] == 1:
            P[b] = torch.eye(d, dtype=torch.float64, device=DEV)
        x = torch.einsum("hij,hni->hnj", P[b], qkv[b])
        at, slot = table[b][(lens[b] - 1) // page], (lens[b] - 1) % page
        qh[b], kp[at, :, slot], vp[at, :, slot] = x[:, 0], x[:, 1], x[:, 2]
    return dict(P=P, qh=qh, k_pages=kp, v_pages=vp)
