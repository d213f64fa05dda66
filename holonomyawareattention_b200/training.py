"""Training of PathOrderedGeometricMHA: the module's forward under autograd, AdamW, one training step.

The reference trains its module with autograd (core/attention_fast_chunked.py:98-177 is differentiable; its kernel
drop-in recomputes the forward in the backward pass, kernel/attention_kernel.py:166-187).  Here the core region
between the projections is one autograd node: link rotations, carries, transports and attention forward, and
attn_bwd and path_bwd backward.  The projections are differentiated as the linears they are.

    attn = PathOrderedGeometricMHA(d_model, n_heads=H, edge_scale=0.05).cuda()
    opt = AdamW(attn.parameters(), lr=3e-4, state_bits=8)
    loss = train_step(attn, x, opt, lambda y: ((y - target) ** 2).mean())      # causal, tril mask

or, with any loss around it, `y, _ = attn(x, attn_mask=tril)`, `loss.backward()`, `opt.step()`.
"""
from __future__ import annotations

from typing import Callable, Optional

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import ops


class PathCore(torch.autograd.Function):
    """heads (B,T,D) = core region of (a_all (B,T,H*stride) fp32, qkv (B,T,3D)); a_bias: one generator row or None."""

    @staticmethod
    def forward(ctx, a_all, qkv, a_bias, n_heads, edge_scale, scale, chunk, layout):
        B, T, threeD = qkv.shape
        a_all, qkv = a_all.contiguous(), qkv.contiguous()
        R, U, M = ops.link_local(a_all, qkv, n_heads, edge_scale, chunk, a_bias, layout)
        C, _ = ops.carry_scan(M)
        del M
        qh, kh, vh = ops.carry_apply(U, C, chunk, qkv.dtype)
        del U
        o, lse = ops.attn_fwd_lse(qh, kh, vh, scale)
        ctx.save_for_backward(a_all, a_bias, R, C, qh, kh, vh, o, lse)
        ctx.args = n_heads, edge_scale, scale, chunk, layout
        return ops.out_transport(o, R, C, chunk, B, n_heads, qkv.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dheads):
        a_all, a_bias, R, C, qh, kh, vh, o, lse = ctx.saved_tensors
        H, edge_scale, scale, chunk, layout = ctx.args
        BH, T, d = qh.shape
        dout = dheads.reshape(BH // H, T, H, d).permute(0, 2, 1, 3).float().contiguous().view(BH, T, d)
        doh = ops.apply_paths(dout, R, C, chunk, transpose=True).to(qh.dtype)          # P^T dout
        dqh, dkh, dvh = ops.attn_bwd(qh, kh, vh, o, lse, doh, scale)
        want_a, _, want_bias = ctx.needs_input_grad[:3]
        if not (want_a or want_bias):                                  # (frozen generators: the vectors' gradients alone)
            dqkv = torch.empty(BH // H, T, H, 3, d, dtype=dheads.dtype, device=dheads.device)
            for i, t in enumerate((dqh, dkh, dvh)):
                dqkv[:, :, :, i] = ops.apply_paths(t.float(), R, C, chunk).view(BH // H, H, T, d).transpose(1, 2)
            return None, dqkv.view(BH // H, T, 3 * H * d), None, None, None, None, None, None
        da, dqkv = ops.path_bwd(a_all, R, C, chunk, H, edge_scale, (qh, kh, vh, o), (dqh, dkh, dvh, doh), a_bias, layout)
        return da, dqkv, da.sum((0, 1)) if want_bias else None, None, None, None, None, None


def _weight_grad(dy: torch.Tensor, x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """dy^T x of bf16 factors, in the weight's type (fp32 weights: the product's fp32 sums as they are)."""
    return torch.mm(dy.t(), x) if dtype is torch.bfloat16 else torch.mm(dy.t(), x, out_dtype=torch.float32)


class EdgeLayer0(torch.autograd.Function):
    """The edge MLP's first layer in bf16, fp32 out (hoa_edge_gemm); its weights may be fp32 (autocast).  w1t, b1f: its
    weight transposed in bf16 and its fp32 bias."""

    @staticmethod
    def forward(ctx, pair, weight, bias, w1t, b1f):
        ctx.save_for_backward(pair, weight)
        return ops.edge_gemm(pair, w1t, b1f)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        pair, weight = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        db = dh.sum(0).to(weight.dtype) if want_b else None
        dh = dh.to(torch.bfloat16)
        dx = dh @ weight.to(torch.bfloat16) if want_x else None
        return dx, _weight_grad(dh, pair, weight.dtype) if want_w else None, db, None, None


class EdgeLayer2(torch.autograd.Function):
    """GELU and the edge MLP's second layer: generators (rows, width) fp32 of the hidden layer h (rows, F) fp32.
    ``forward_`` computes them (the module's form for its generator_precision), ``wt`` (F, width) and ``index`` (the
    place of every weight row among the generators, None: in order) say how the weight is laid out."""

    @staticmethod
    def forward(ctx, h, weight, bias, forward_, wt, index):
        ctx.save_for_backward(h, wt, index)
        ctx.dtype = weight.dtype
        return forward_(h)

    @staticmethod
    @once_differentiable
    def backward(ctx, da):
        h, wt, index = ctx.saved_tensors
        want_h, want_w, want_b = ctx.needs_input_grad[:3]
        dh = dw = db = None
        if want_b:
            db = da.sum(0).to(ctx.dtype)
            db = db if index is None else db[index]
        da = da.to(torch.bfloat16)
        if want_w:
            dw = _weight_grad(da, F.gelu(h).to(torch.bfloat16), ctx.dtype)     # (width, F)
            dw = dw if index is None else dw[index]
        if want_h:
            dh = torch.ops.aten.gelu_backward((da @ wt.t()).float(), h)
        return dh, dw, db, None, None, None


class EdgeWeights:
    """The bf16 edge MLP's weights in one forward, as autograd sees them, and the copies that its kernels read.  Those of a
    layer that is trained are made from these very tensors and end with the forward's graph: its weights change at every
    step, by whatever means.  Those of a frozen layer are kept with the module."""

    def __init__(self, attn):
        from .attention import Kept
        own = Kept(streams=False)
        lin0, lin2 = attn.edge_mlp[0], attn.edge_mlp[2]
        self.first, self.second = (
            (w, b, own if w.requires_grad or b.requires_grad else attn._copies) for w, b in ((lin0.weight, lin0.bias), (lin2.weight, lin2.bias)))


def edge_generators(attn, x: torch.Tensor, weights: Optional[EdgeWeights]):
    """(a_all (B, L, H*stride) fp32, layout) of the module's edge MLP, differentiable (attn._edge_generators_nobias)."""
    B, L, D = x.shape
    partner = torch.roll(x, shifts=-1, dims=1)
    if attn.link_mode == "additive":
        return attn.gqproj(x).float() + attn.gkproj(partner).float(), "packed"
    pair = torch.cat([x, partner], dim=-1)
    if weights is None:
        return attn.edge_mlp(pair).float(), "packed"             # (under autocast the linears' results are bf16)
    layout = attn._gen_layout()
    h = EdgeLayer0.apply(pair.reshape(B * L, 2 * D), *weights.first[:2], *attn._w1t(*weights.first))
    mode = attn._precision_for(L, B * L, h.shape[1])
    wt = attn._stacked_w2t(mode == "split", *weights.second)[0][:h.shape[1]]        # (split: the first of its two, for both passes)
    index = ops.banked_index_on(attn.d, attn.h, x.device) if layout == "banked" else None
    a = EdgeLayer2.apply(h, *weights.second[:2], lambda t: attn._generators_of_hidden(t, mode, weights.second), wt, index)
    return a.view(B, L, -1), layout


def forward_rows(attn, x: torch.Tensor, weights: Optional[EdgeWeights]) -> torch.Tensor:
    """The module's causal forward (tril mask) of some batch rows, differentiable."""
    B, L, _ = x.shape
    qkv = attn.qkv(x)
    a, layout = edge_generators(attn, x, weights)
    chunk = attn.chunk or ops.plan_chunk(B, attn.h, L, attn.d, x.device)
    heads = PathCore.apply(a, qkv, None, attn.h, attn.edge_scale, attn.scale, chunk, layout)
    return attn.out(heads)


def forward(attn, x: torch.Tensor, rows: int) -> torch.Tensor:
    """The module's causal forward (tril mask), differentiable, ``rows`` batch rows at a time."""
    for layer in (0, 2):
        if any(p.requires_grad for p in attn.edge_mlp[layer].parameters()):
            attn._copies.clear(layer)                            # (for the forwards without gradients that follow)
    weights = EdgeWeights(attn) if attn.link_mode != "additive" and x.dtype != torch.float32 else None
    pieces = [forward_rows(attn, x[b0:b0 + rows], weights) for b0 in range(0, x.shape[0], rows)]
    return pieces[0] if len(pieces) == 1 else torch.cat(pieces)


_FLOATS = (torch.float32, torch.bfloat16)


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with one launch for all tensors of a type (ops.adamw_step).

    ``state_bits`` 32: fp32 moments; 8: 8-bit ones in blocks of 256 elements (2 bytes an element for both instead of 8): a held
    root is within a factor of about 2 of the fp32 one at betas[1] 0.999, 1.4 up to 0.97.
    bf16 parameters are stepped on fp32 master copies, kept in the state, unless ``masters`` is False; an element of a
    parameter that something else wrote since the last step (load_state_dict, a clamp; not through ``.data``, which torch
    does not count) is taken as it is.  The steps are counted on the host: under graph capture step() raises
    (ops.adamw_step takes a count on the device)."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32, masters: bool = True):
        self._left = {}                                          # parameter -> (address, version) that the last step left
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits, masters=masters))

    def add_param_group(self, param_group):
        g = {**self.defaults, **param_group}
        if not (g["lr"] >= 0.0 and g["eps"] >= 0.0 and g["weight_decay"] >= 0.0 and all(0.0 <= b < 1.0 for b in g["betas"])):
            raise ValueError("lr, eps and weight_decay must be at least 0 and betas in [0, 1)")
        if g["state_bits"] not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        super().add_param_group(param_group)

    def __setstate__(self, state):
        super().__setstate__(state)
        self._left = {}

    def _init(self, p, group):
        s = self.state[p]
        if s:
            if "master" in s and self._left.get(p) != (p.data_ptr(), p._version):
                m = s["master"]                                  # (its low bits stay where the parameter is still its rounding)
                m.copy_(torch.where(m.to(p.dtype) == p, m, p))
            return s
        s["step"] = 0
        moment = torch.float32 if group["state_bits"] == 32 else torch.float8_e4m3fn
        for k in ("exp_avg", "exp_avg_sq"):
            s[k] = torch.zeros(p.shape, dtype=torch.float32, device=p.device).to(moment)
        if group["state_bits"] == 8:
            s["scales"] = torch.zeros(2, -(-p.numel() // ops.ADAMW_BLOCK), dtype=torch.float32, device=p.device)
        if p.dtype == torch.bfloat16 and group["masters"]:
            s["master"] = p.detach().float().contiguous()
        return s

    @torch.no_grad()
    def step(self, closure=None):
        """One step; what is refused is refused before any parameter changes."""
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise NotImplementedError("AdamW.step counts its steps on the host and cannot be captured: capture ops.adamw_step")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        found = [[(p, p.grad) for p in group["params"] if p.grad is not None] for group in self.param_groups]
        for p, g in (x for xs in found for x in xs):
            if not p.is_cuda or g.is_sparse or p.dtype not in _FLOATS or g.dtype not in _FLOATS:
                raise NotImplementedError("AdamW takes dense fp32 or bf16 CUDA parameters and gradients")
            if not p.is_contiguous():
                raise ValueError("parameters must be contiguous")
        for group, xs in zip(self.param_groups, found):
            calls = {}
            for p, g in xs:
                s = self._init(p, group)
                calls.setdefault((p.device, p.dtype, g.dtype, s["step"], "master" in s), []).append((p, g.contiguous(), s))
            for (dev, _, _, n, masters), items in calls.items():
                ps, gs, ss = zip(*items)
                ops.adamw_step(ps, gs, [s["exp_avg"] for s in ss], [s["exp_avg_sq"] for s in ss],
                               torch.full((1,), n + 1, dtype=torch.int32, device=dev), lr=float(group["lr"]), betas=group["betas"],
                               eps=group["eps"], weight_decay=group["weight_decay"], masters=[s["master"] for s in ss] if masters else None,
                               scales=[s["scales"] for s in ss] if group["state_bits"] == 8 else None)
                for p, s in zip(ps, ss):
                    s["step"] = n + 1
                    if masters:
                        self._left[p] = p.data_ptr(), p._version
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch.optim.Optimizer's; the state keeps its types (the base class would make it the parameters')."""
        super().load_state_dict(state_dict)
        old = [i for g in state_dict["param_groups"] for i in g["params"]]
        new = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(old, new):
            for k, v in state_dict["state"].get(i, {}).items():
                self.state[p][k] = v.detach().to(p.device, copy=True) if torch.is_tensor(v) else v


_TRIL = {}


def _tril(L: int, device) -> torch.Tensor:
    """The causal mask, kept for the next step on the same stream (another stream would have to wait for it)."""
    key = device, torch.cuda.current_stream(device).cuda_stream if device.type == "cuda" else 0
    m = _TRIL.get(key)
    if m is None or m.shape[0] != L:
        with torch.inference_mode(False):
            m = _TRIL[key] = torch.ones(L, L, dtype=torch.bool, device=device).tril()
    return m


def train_step(attn, x: torch.Tensor, optimizer, loss: Callable[[torch.Tensor], torch.Tensor], attn_mask: Optional[torch.Tensor] = None,
               max_grad_norm: Optional[float] = None) -> torch.Tensor:
    """One step: y = attn(x) under the causal mask (``attn_mask``, default tril), loss(y), gradients (their norm held to
    ``max_grad_norm``, if given), the optimizer's step.  The optimizer's gradients start and end at None.  Returns the loss,
    detached, on the device.  Nothing waits for the GPU, but where an ``attn_mask`` is given that was not seen before (what it
    holds decides the path) and in the form "split8" of the generators ("auto" beyond 8192 positions: the largest weight
    gives the fp8 product's scale on the host, once a forward while the weights are trained).  Not under graph capture."""
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise NotImplementedError("train_step cannot be captured into a graph")
    L = x.shape[1]
    if attn_mask is None:
        attn_mask = _tril(L, x.device)
    optimizer.zero_grad(set_to_none=True)
    with torch.enable_grad():
        y, _ = attn(x, attn_mask=attn_mask)
        value = loss(y)
        value.backward()
    if max_grad_norm is not None:
        torch.nn.utils.clip_grad_norm_([p for g in optimizer.param_groups for p in g["params"] if p.grad is not None], max_grad_norm)
    optimizer.step()
    optimizer.zero_grad(set_to_none=True)
    return value.detach()
