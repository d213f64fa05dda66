"""Generation with PathOrderedGeometricMHA: a paged cache of k^ and v^, and the steps that fill and read it.

In causal mode k^_t = P_t^T k_t and v^_t = P_t^T v_t do not change as the sequence grows
(core/attention_fast_chunked.py:108-110), so a token is computed from its predecessor's hidden
state, the path product P (d x d a head) and the cache.  A forked sequence shares its parent's
pages as they are.  No counterpart in the reference, which recomputes the whole sequence.

    cache = PathCache(attn, rows=8, max_tokens=4096)
    y = prefill(attn, x, cache, [0])              # x (1, T, D): a prompt into row 0
    cache.fork([0, 0, 0], [1, 2, 3])              # three more candidates
    cache.share(0)                                # what all rows have in common is read once a step
    y = decode(attn, x_next, cache)               # x_next (8, D): one token of every row that has any
    cache.free([2]); cache.compact()

Everything runs on the current stream.  Rows are host integers; the cache keeps the rows' lengths and
which of them hold a page in common on the host too, and refuses what does not fit before anything is
launched.
"""
from __future__ import annotations

import contextlib
from typing import List, Optional, Sequence

import torch

from . import _lib, ops


@contextlib.contextmanager
def _outside_inference_mode():
    with torch.inference_mode(False), torch.no_grad():
        yield


def _plain():
    """Tensors made under this may be updated in place in any mode (those of inference mode only within it)."""
    return _outside_inference_mode() if torch.is_inference_mode_enabled() else contextlib.nullcontext()


class PathCache:
    """Pages of k^ and v^ for ``rows`` sequences of one attention module, each up to ``max_tokens`` long.

    ``n_pages``: pages of the pool (default: enough for every row at its longest).  State, replaced by
    every operation: k_pages / v_pages (n_pages, H, page, d) in the module's type, table (rows, W), lens
    (rows,), refs (n_pages,) int32, P (rows, H, d, d) fp32, last (rows, D) the hidden state of each row's
    newest token; ``tokens``, a host list of the lengths."""

    def __init__(self, attn, rows: int, max_tokens: int, n_pages: Optional[int] = None, page: int = 64):
        if rows < 1 or max_tokens < 1 or page < 1:
            raise ValueError("rows, max_tokens and page must be at least 1")
        if attn.mode != "causal":
            raise NotImplementedError("the cache holds causal transports (mode 'causal')")
        w = attn.qkv.weight
        if not w.is_cuda:
            raise NotImplementedError("the B200 kernels need CUDA tensors (there is no CPU path)")
        self.rows, self.page, self.W = rows, page, -(-max_tokens // page)
        self.max_tokens = max_tokens
        self.n_pages = rows * self.W if n_pages is None else n_pages
        dev, H, d = w.device, attn.h, attn.d
        with _plain():
            self.k_pages = torch.empty(self.n_pages, H, page, d, dtype=w.dtype, device=dev)
            self.v_pages = torch.empty_like(self.k_pages)
            self.table = torch.full((rows, self.W), -1, dtype=torch.int32, device=dev)
            self.lens = torch.zeros(rows, dtype=torch.int32, device=dev)
            self.refs = torch.zeros(self.n_pages, dtype=torch.int32, device=dev)
            self.P = torch.eye(d, device=dev).expand(rows, H, d, d).contiguous()
            self.last = torch.zeros(rows, H * d, dtype=w.dtype, device=dev)
        self.tokens: List[int] = [0] * rows
        # which rows hold a page in common, by serial numbers of their own (not the page ids, which
        # only the device knows): enough to tell what is free and what is shared
        self._held: List[List[int]] = [[] for _ in range(rows)]
        self._count = {}
        self._serial = 0
        self.n_shared = 0
        self.shared: Optional[torch.Tensor] = None
        self._shared_row = -1

    def _rows(self, rows: Sequence[int], what: str) -> List[int]:
        rows = [int(r) for r in rows]
        if any(r < 0 or r >= self.rows for r in rows) or len(set(rows)) != len(rows):
            raise ValueError(f"{what} must be different rows in [0, {self.rows})")
        return rows

    def _take(self, n: int) -> List[int]:
        new = list(range(self._serial, self._serial + n))
        self._serial += n
        self._count.update((i, 1) for i in new)
        return new

    def _need(self, n: int) -> None:
        if n > self.n_pages - len(self._count):
            raise _lib.HoaError("PathCache", _lib.HOA_ERR_PAGES,
                                f"{n} pages are needed, {self.n_pages - len(self._count)} are free")

    def _ints(self, values) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.table.device)

    @contextlib.contextmanager
    def _undo_on_error(self):
        """The rows are as long as before, should the body raise after it has reserved tokens.  (The device's state is replaced,
        not changed, so the old one still holds; P and last are the body's to change once nothing can fail any more.)"""
        state = self.table, self.lens, self.refs, self.tokens
        held, serial = [len(h) for h in self._held], self._serial
        try:
            yield
        except BaseException:
            self.table, self.lens, self.refs, self.tokens = state
            for h, n in zip(self._held, held):
                del h[n:]
            for i in range(serial, self._serial):
                self._count.pop(i, None)
            self._serial = serial
            raise

    def reserve(self, counts: Sequence[int]) -> None:
        """Row s grows by counts[s] tokens.  Without enough free pages: HoaError with HOA_ERR_PAGES,
        nothing changed (fork: likewise).  While pages are shared every row begins with them: an empty
        row cannot grow, it can become a fork."""
        counts = [int(c) for c in counts]
        if len(counts) != self.rows or any(c < 0 for c in counts):
            raise ValueError(f"counts must be {self.rows} numbers of tokens")
        if any(t + c > self.max_tokens for t, c in zip(self.tokens, counts)):
            raise ValueError(f"a row would pass max_tokens = {self.max_tokens}")
        if self.n_shared and any(c and not t for t, c in zip(self.tokens, counts)):
            raise ValueError("a new row does not begin with the shared pages: end the sharing first (share(row, 0))")
        new = [-(-(t + c) // self.page) - len(h) for t, c, h in zip(self.tokens, counts, self._held)]
        self._need(sum(new))
        self.table, self.lens, self.refs = ops.pages_reserve(self.table, self.lens, self.refs, self._ints(counts), self.page)
        self.tokens = [t + c for t, c in zip(self.tokens, counts)]
        for h, n in zip(self._held, new):
            if n:
                h += self._take(n)

    def fork(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Row dst[i], which is empty, becomes a copy of row src[i] (a row may be forked several times)."""
        dst = self._rows(dst, "dst")
        src = [int(r) for r in src]
        if len(src) != len(dst) or any(r < 0 or r >= self.rows or self.tokens[r] == 0 for r in src):
            raise ValueError("src must name a row with tokens for every dst")
        if any(self.tokens[r] for r in dst):
            raise ValueError("dst rows must be empty")
        if not dst:
            return
        self._need(sum(1 for r in src if self.tokens[r] % self.page))
        a, b = self._ints(src), self._ints(dst)
        # (first what writes to the empty rows only, then the state: an error in between leaves it as it was)
        ops.pages_copy([self.P, self.last], a, b)            # a row of these is a page too
        self.table, self.lens, self.refs = ops.pages_fork([self.k_pages, self.v_pages], self.table, self.lens, self.refs, a, b,
                                                          self.page)
        for s, t in zip(src, dst):
            full = self.tokens[s] // self.page
            self._held[t] = self._held[s][:full] + self._take(1 if self.tokens[s] % self.page else 0)
            for i in self._held[s][:full]:
                self._count[i] += 1
            self.tokens[t] = self.tokens[s]

    def free(self, rows: Sequence[int]) -> None:
        """The rows end; pages that no other row holds are free again."""
        rows = self._rows(rows, "rows")
        if not rows:
            return
        self.table, self.lens, self.refs = ops.pages_free(self.table, self.lens, self.refs, self._ints(rows), self.page)
        for r in rows:
            for i in self._held[r]:
                self._count[i] -= 1
                if self._count[i] == 0:
                    del self._count[i]
            self._held[r], self.tokens[r] = [], 0
        if self._shared_row in rows:
            live = [r for r in range(self.rows) if self.tokens[r]]
            self._shared_row = live[0] if live else -1
            if not live:
                self.n_shared, self.shared = 0, None

    def compact(self) -> torch.Tensor:
        """The live pages move to the front of the pools; their number (1,) int32, on the device."""
        # (pages move into free ones only: until the new table is taken, the old one still holds)
        table, refs, live = ops.pages_compact([self.k_pages, self.v_pages], self.table, self.refs)
        shared = table[self._shared_row, :self.n_shared].clone() if self.n_shared else self.shared
        self.table, self.refs, self.shared = table, refs, shared
        return live

    def share(self, row: int, tokens: Optional[int] = None) -> int:
        """Read the first ``tokens`` tokens (default: all that fill whole pages) of ``row`` once for all
        rows from now on: the number of tokens shared, a multiple of the page.  Every row that has
        tokens must begin with the same pages, i.e. be a fork.  share(row, 0) ends it."""
        (row,) = self._rows([row], "row")
        if tokens is not None and tokens < 0:
            raise ValueError(f"tokens must be at least 0, got {tokens}")
        n = (self.tokens[row] if tokens is None else min(tokens, self.tokens[row])) // self.page
        if n:
            if any(self._held[r][:n] != self._held[row][:n] for r in range(self.rows) if self.tokens[r]):
                raise ValueError("every row with tokens must begin with the shared pages (fork them from one row)")
        self.n_shared = n
        self.shared = self.table[row, :n].clone() if n else None
        self._shared_row = row if n else -1
        return n * self.page


def _check(attn, x, cache) -> None:
    if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in attn.parameters())):
        raise NotImplementedError("forward-only kernels: call under torch.no_grad() / torch.inference_mode()")
    if attn.mode != "causal" or (attn.training and attn.dropout.p != 0.0):
        raise NotImplementedError("generation needs mode 'causal' and inactive dropout")
    if x.dtype != cache.k_pages.dtype or x.device != cache.k_pages.device or x.shape[-1] != attn.h * attn.d:
        raise ValueError(f"x must be (..., {attn.h * attn.d}) {cache.k_pages.dtype} on {cache.k_pages.device}")
    ops.poll_status(x.device)


def prefill(attn, x: torch.Tensor, cache: PathCache, rows: Sequence[int]) -> torch.Tensor:
    """x (len(rows), T, D): the next T hidden states of the rows, all of them empty or none; their outputs
    (len(rows), T, D).  The link, carry and transport kernels of the forward, k^ and v^ written to the
    pages, attention over the cache (the shared pages read once).  An error leaves the cache as it was
    (decode: likewise)."""
    rows = cache._rows(rows, "rows")
    if x.dim() != 3 or x.shape[0] != len(rows) or x.shape[1] < 1 or not rows:
        raise ValueError("x must be (len(rows), T, D)")
    _check(attn, x, cache)
    old = [cache.tokens[r] for r in rows]
    go_on = old[0] > 0
    if any((t > 0) != go_on for t in old):
        raise ValueError("the rows must all be empty or all have tokens")
    if not go_on and cache.n_shared:
        raise ValueError("a new row does not begin with the shared pages: end the sharing first (share(row, 0))")
    T = x.shape[1]
    grow = [0] * cache.rows
    for r in rows:
        grow[r] = T
    with cache._undo_on_error():
        cache.reserve(grow)
        y, P = torch.empty_like(x), []
        idx = torch.tensor(rows, device=x.device)
        step = max(1, attn.PIECE_TOKENS // T)
        for i in range(0, len(rows), step):
            y[i:i + step], p = _prefill_rows(attn, x[i:i + step], cache, idx[i:i + step], go_on)
            P.append(p)
        P = P[0] if len(P) == 1 else torch.cat(P)
        cache.P.index_copy_(0, idx, P)
        cache.last.index_copy_(0, idx, x[:, -1])
    return y


def _prefill_rows(attn, x, cache, idx, go_on):
    """Rows ``idx`` (on the device): (outputs, their P after the last token).  The cache's pages are written, its P and last
    are not."""
    B, T, D = x.shape
    H, d = attn.h, attn.d
    # rows that go on: the chain starts at the newest cached token (its P is the carry), whose edge
    # leads to the first new one; `lead` positions are recomputed and left out below
    lead = 1 if go_on else 0
    xs = torch.cat([cache.last[idx].unsqueeze(1), x], 1) if go_on else x
    L = T + lead
    a, bias, layout = attn._edge_generators_nobias(xs, None, cache.max_tokens)
    qkv = attn.qkv(xs).contiguous()
    chunk = attn.chunk or ops.plan_chunk(B, H, L, d, x.device)
    R, U, M = ops.link_local(a, qkv, H, attn.edge_scale, chunk, bias, layout)
    C, _ = ops.carry_scan(M, cache.P[idx].view(B * H, d, d) if go_on else None)
    heads = [t.view(B, H, L, d).permute(0, 2, 1, 3)[:, lead:] for t in ops.carry_apply(U, C, chunk, x.dtype)]
    table, lens = cache.table[idx], cache.lens[idx]
    ops.pages_write(heads[1], heads[2], cache.k_pages, cache.v_pages, table, lens)
    o, _ = ops.paged_attn_fwd(heads[0], cache.k_pages, cache.v_pages, table[:, cache.n_shared:], lens, attn.scale,
                              shared=cache.shared, out_dtype=torch.float32)
    full = torch.zeros(B, H, L, d, dtype=torch.float32, device=x.device)
    full[:, :, lead:] = o.permute(0, 2, 1, 3)
    out = ops.out_transport(full.view(B * H, L, d), R, C, chunk, B, H, x.dtype)[:, lead:]
    P = ops.compose_paths(R[:, -1:].contiguous(), C[:, -1:].contiguous(), 1).view(B, H, d, d)
    return attn.out(out), P


def decode(attn, x: torch.Tensor, cache: PathCache) -> torch.Tensor:
    """x (rows, D): the next hidden state of every row; its output (rows, D).  Rows without tokens are
    idle: their x is not looked at and their output is that of a zero head (0 through attn.out)."""
    if x.dim() != 2 or x.shape[0] != cache.rows:
        raise ValueError(f"x must be ({cache.rows}, D)")
    _check(attn, x, cache)
    H, d, S = attn.h, attn.d, cache.rows
    live = [1 if t else 0 for t in cache.tokens]
    with cache._undo_on_error():
        cache.reserve(live)
        a, bias, layout = attn._edge_generators_nobias(cache.last.unsqueeze(1), x.unsqueeze(1), cache.max_tokens)
        qkv = attn.qkv(x)
        with _plain():
            P = torch.empty_like(cache.P)
            last = x.clone(memory_format=torch.contiguous_format) if all(live) else \
                torch.where(cache.lens.view(-1, 1) > 0, x, cache.last).contiguous()
        _, qh = ops.path_step(a.view(S, -1), cache.P, qkv, H, attn.edge_scale, cache.k_pages, cache.v_pages, cache.table,
                              cache.lens, a_bias=bias, gen_layout=layout, P_out=P)
        o, _ = ops.paged_attn_fwd(qh.view(S, 1, H, d), cache.k_pages, cache.v_pages, cache.table[:, cache.n_shared:], cache.lens,
                                  attn.scale, shared=cache.shared, paths=P)
        y = attn.out(o.view(S, H * d))
    cache.P, cache.last = P, last
    return y
