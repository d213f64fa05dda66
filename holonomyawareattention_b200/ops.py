"""Tensor-level wrappers over the libhoa C ABI (include/hoa.h).

Each function validates shapes/dtypes/devices, allocates outputs and scratch
with PyTorch (the C ABI never allocates), and enqueues the kernels on the
current CUDA stream.  There is no fallback path: a missing library, a CPU
tensor or an unsupported shape raises.
"""
from __future__ import annotations

import collections
import contextlib
import ctypes
import math
import threading
import warnings
from typing import Optional, Tuple

import torch

from . import _lib

_DT = {torch.float32: _lib.HOA_F32, torch.bfloat16: _lib.HOA_BF16}


def _dtype_code(t: torch.dtype) -> int:
    try:
        return _DT[t]
    except KeyError:
        raise NotImplementedError(f"dtype {t} is not supported (float32 or bfloat16)") from None


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise NotImplementedError("the B200 kernels need CUDA tensors (there is no CPU path)")


def _contig(t: torch.Tensor, name: str) -> torch.Tensor:
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


# ---------------------------------------------------------------------------
# device status words.  The tensor-core kernels bound every wait on the GPU; a
# wait that gives up makes its kernel leave early and set HOA_ERR_TIMEOUT in a
# status word, and the output of that launch is not valid.  The word is known
# only once the stream has run, so every op here queues a 4-byte copy of it to
# pinned host memory behind its kernels: poll_status() raises for the copies
# that have landed (the module calls it at every forward), check_status() waits
# for the device first (call it at the end of a run).  The generation kernels set
# a word in mapped host memory instead, which both functions read too.
# ---------------------------------------------------------------------------
# device -> (word, the same as an array): a word in mapped host memory that the generation kernels
# set themselves (no copy to queue behind a call of a few microseconds), 0 until something went
# wrong.  Kept for good: its address is handed out once a device and may be in flight at any time.
_MAPPED = {}


def _mapped_word(dev: torch.device):
    v = _MAPPED.get(dev)
    if v is None:
        with torch.inference_mode(False):
            t = torch.zeros(1, dtype=torch.int32).pin_memory()
        v = _MAPPED.setdefault(dev, (t, t.numpy()))
    return v[1]


class _StatusWatch:
    RING = 256

    def __init__(self, dev: torch.device):
        self.dev = dev
        # normal tensors even when the first call comes under inference mode, so that
        # later calls outside it may update them
        with torch.inference_mode(False):
            # the word the stage entry points share: set by a kernel, cleared here
            self.sticky = torch.zeros(1, dtype=torch.int32, device=dev)
            self.host = torch.zeros(self.RING, dtype=torch.int32).pin_memory()
        self.mapped = _mapped_word(dev)
        self.pending = collections.deque()        # (slot, event, what)
        self.next = 0
        self.lock = threading.Lock()

    def watch(self, word: torch.Tensor, what: str) -> None:
        """Queue a copy of the device int32 ``word`` behind the current stream's work."""
        if torch.cuda.is_current_stream_capturing():
            return
        with self.lock:
            if len(self.pending) == self.RING:
                self.pending[0][1].synchronize()
                self._poll_locked()
            slot = self.next
            self.next = (self.next + 1) % self.RING
            self.host[slot:slot + 1].copy_(word.view(torch.int32)[:1], non_blocking=True)
            ev = torch.cuda.Event()
            ev.record(torch.cuda.current_stream(self.dev))
            self.pending.append((slot, ev, what))

    def _poll_locked(self) -> None:
        st = int(self.mapped[0])
        if st != 0:
            self.mapped[0] = 0
            _lib.check("a cache or training operation", st)
        while self.pending and self.pending[0][1].query():
            slot, _, what = self.pending.popleft()
            st = int(self.host[slot])
            if st != 0:
                # report once: forget the other copies in flight and clear the shared word
                for _, ev, _ in self.pending:
                    ev.synchronize()
                self.pending.clear()
                self.sticky.zero_()
                _lib.check(what, st)

    def poll(self) -> None:
        with self.lock:
            self._poll_locked()

    def check(self) -> None:
        # the whole device: the mapped word has no event behind it, and its kernels run on any stream
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.synchronize(self.dev)
        with self.lock:
            for _, ev, _ in self.pending:
                ev.synchronize()
            self._poll_locked()


_WATCH = {}


def _watch(dev: torch.device) -> _StatusWatch:
    dev = torch.device(dev)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    w = _WATCH.get(dev)
    if w is None:
        w = _WATCH[dev] = _StatusWatch(dev)
    return w


def poll_status(device=None) -> None:
    """Raise HoaError for any finished launch on ``device`` whose device-side wait
    gave up (HOA_ERR_TIMEOUT), or that found a page or row outside its cache
    (HOA_ERR_PAGES).  Does not wait for launches still running."""
    _watch(device if device is not None else "cuda").poll()


def check_status(device=None) -> None:
    """Wait for every launch queued so far on ``device``, on all its streams, and raise
    HoaError if any of them reported HOA_ERR_TIMEOUT or HOA_ERR_PAGES."""
    _watch(device if device is not None else "cuda").check()


def set_wait_bound(max_cycles: int) -> None:
    """Bound (SM cycles) of the device-side waits of the kernels launched from now
    on, process-wide; 0 restores the default.  A diagnostic: a short bound makes
    real kernels give up and report HOA_ERR_TIMEOUT (hoa_set_wait_bound)."""
    _lib.call("hoa_set_wait_bound", int(max_cycles))


def plan_chunk(B: int, H: int, T: int, d: int, device=None) -> int:
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    return int(_lib.load().hoa_plan_chunk(B, H, T, d, sms))


# ---------------------------------------------------------------------------
# generator layouts: "packed" (the reference's upper triangle, d(d-1)/2 floats
# per head) and "banked" (HOA_GEN_BANKED: the same values permuted, and a few
# unused slots, so that the link kernel reads rows without bank conflicts)
# ---------------------------------------------------------------------------
_BANKED_MAPS = {}
_BANKED_INDICES = {}


def gen_stride(d: int, layout: str = "packed") -> int:
    """Floats per head of a generator row in ``layout`` (0: not available for d)."""
    if layout not in ("packed", "banked"):
        raise ValueError("layout must be 'packed' or 'banked'")
    return int(_lib.load().hoa_gen_stride(d, 1 if layout == "banked" else 0))


def gen_banked_map(d: int) -> torch.Tensor:
    """(d(d-1)/2,) int64 on the CPU: the banked slot of every packed (reference-order) entry."""
    if d not in _BANKED_MAPS:
        m = d * (d - 1) // 2
        out = torch.empty(m, dtype=torch.int32)
        _lib.call("hoa_gen_banked_map", d, out.data_ptr())
        _BANKED_MAPS[d] = out.long()
    return _BANKED_MAPS[d]


def gen_banked_index(d: int, n_heads: int, device=None) -> torch.Tensor:
    """(H*m,) int64: the banked position (h*stride + slot) of packed entry h*m + i."""
    S = gen_stride(d, "banked")
    slots = gen_banked_map(d)
    idx = (torch.arange(n_heads).unsqueeze(1) * S + slots.unsqueeze(0)).reshape(-1)
    return idx if device is None else idx.to(device)


def banked_index_on(d: int, n_heads: int, device) -> torch.Tensor:
    """gen_banked_index on a device, kept: not to be written."""
    i = _BANKED_INDICES.get((d, n_heads, device))
    if i is None:
        with torch.inference_mode(False):
            i = _BANKED_INDICES[d, n_heads, device] = gen_banked_index(d, n_heads, device)
    return i


def gen_to_banked(a: torch.Tensor, n_heads: int, d: int) -> torch.Tensor:
    """(..., H*m) packed generators -> (..., H*stride) banked (zeros at unused slots)."""
    S = gen_stride(d, "banked")
    out = a.new_zeros(*a.shape[:-1], n_heads * S)
    out[..., gen_banked_index(d, n_heads, a.device)] = a
    return out


def gen_from_banked(a: torch.Tensor, n_heads: int, d: int) -> torch.Tensor:
    """(..., H*stride) banked generators -> (..., H*m) packed."""
    return a[..., gen_banked_index(d, n_heads, a.device)]


def _gen_code(a_all: torch.Tensor, layout: str) -> int:
    code = _dtype_code(a_all.dtype)
    if layout == "banked":
        if a_all.dtype != torch.float32:
            raise NotImplementedError("banked generators are fp32")
        code |= _lib.HOA_GEN_BANKED
    elif layout != "packed":
        raise ValueError("gen_layout must be 'packed' or 'banked'")
    return code


def _gen_width(n_heads: int, d: int, layout: str) -> int:
    S = gen_stride(d, layout)
    if S == 0:
        raise NotImplementedError(f"the {layout} generator layout needs d % 32 == 0 (d = {d})")
    return n_heads * S


def core_forward(a_all: torch.Tensor, qkv: torch.Tensor, n_heads: int, edge_scale: float,
                 softmax_scale: Optional[float] = None, out_dtype: Optional[torch.dtype] = None,
                 hat_dtype: Optional[torch.dtype] = None, chunk: Optional[int] = None,
                 carry_in: Optional[torch.Tensor] = None,
                 total_out: Optional[torch.Tensor] = None,
                 a_bias: Optional[torch.Tensor] = None,
                 gen_layout: str = "packed") -> torch.Tensor:
    """Core region (kernels 1-4): a_all (B,T,H*m) and qkv (B,T,3D) -> heads (B,T,D).

    ``a_all`` is the raw edge-MLP output (edge_scale is applied in the kernel,
    as core/attention_fast_chunked.py:77 does); ``a_bias`` (one generator row,
    fp32) is the MLP's output bias when the GEMM left it out.  ``gen_layout``
    "banked": a_all (B,T,H*stride) and a_bias in the banked layout
    (gen_to_banked).  ``carry_in`` / ``total_out`` are optional (B*H, d, d) fp32
    tensors (see hoa_core_forward).
    """
    _need_cuda(a_all, qkv, carry_in, total_out, a_bias)
    B, T, threeD = qkv.shape
    D = threeD // 3
    H = n_heads
    d = D // H
    a_code = _gen_code(a_all, gen_layout)
    width = _gen_width(H, d, gen_layout)
    if a_all.shape != (B, T, width):
        raise ValueError(f"a_all must be (B,T,{width}) for the {gen_layout} layout, got {tuple(a_all.shape)}")
    _contig(a_all, "a_all"); _contig(qkv, "qkv")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(d)
    _check_bias(a_bias, width)
    out_dtype = out_dtype or qkv.dtype
    hat_dtype = hat_dtype or qkv.dtype
    if chunk is None:
        chunk = plan_chunk(B, H, T, d, qkv.device)
    for t, nm in ((carry_in, "carry_in"), (total_out, "total_out")):
        if t is not None and (t.dtype != torch.float32 or t.shape != (B * H, d, d) or not t.is_contiguous()):
            raise ValueError(f"{nm} must be a contiguous fp32 ({B * H},{d},{d}) tensor")
    lib = _lib.load()
    hat_code = _dtype_code(hat_dtype)
    ws_bytes = int(lib.hoa_core_workspace_bytes(B, H, T, d, chunk, hat_code))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=qkv.device)
    out = torch.empty(B, T, D, dtype=out_dtype, device=qkv.device)
    _lib.call("hoa_core_forward", _ptr(a_all), a_code, _ptr(a_bias), float(edge_scale),
              _ptr(qkv), _dtype_code(qkv.dtype), _ptr(out), _dtype_code(out_dtype), hat_code,
              float(softmax_scale), _ptr(carry_in), _ptr(total_out), B, H, T, d, int(chunk),
              _ptr(ws), ws_bytes, _stream(qkv.device))
    # the status word is the workspace's first 4 bytes (hoa_core_workspace_bytes)
    _watch(qkv.device).watch(ws[:4], "hoa_core_forward")
    return out


# ---------------------------------------------------------------------------
# individual stages (used by the tests and by the sequence-sharded path)
# ---------------------------------------------------------------------------
def _check_bias(a_bias, n):
    if a_bias is not None and (a_bias.dtype != torch.float32 or a_bias.numel() != n
                               or not a_bias.is_contiguous()):
        raise ValueError(f"a_bias must be a contiguous fp32 tensor of {n} elements")


def link_local(a_all: torch.Tensor, qkv: torch.Tensor, n_heads: int, edge_scale: float,
               chunk: int, a_bias: Optional[torch.Tensor] = None, gen_layout: str = "packed"
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Kernel (1)+(2) local part -> (R (BH,T,d,d), U (BH,T,3,d), M (BH,K,d,d)), all fp32."""
    _need_cuda(a_all, qkv, a_bias)
    B, T, threeD = qkv.shape
    H = n_heads
    d = threeD // 3 // H
    K = (T + chunk - 1) // chunk
    a_code = _gen_code(a_all, gen_layout)
    width = _gen_width(H, d, gen_layout)
    if a_all.shape[-1] != width or a_all.numel() != B * T * width:
        raise ValueError(f"a_all must be (B,T,{width}) for the {gen_layout} layout, got {tuple(a_all.shape)}")
    _contig(a_all, "a_all"); _contig(qkv, "qkv")
    _check_bias(a_bias, width)
    dev = qkv.device
    R = torch.empty(B * H, T, d, d, dtype=torch.float32, device=dev)
    U = torch.empty(B * H, T, 3, d, dtype=torch.float32, device=dev)
    M = torch.empty(B * H, K, d, d, dtype=torch.float32, device=dev)
    w = _watch(dev)
    _lib.call("hoa_link_local", _ptr(a_all), a_code, _ptr(a_bias), float(edge_scale), _ptr(qkv),
              _dtype_code(qkv.dtype), _ptr(R), _ptr(U), _ptr(M), _ptr(w.sticky), B, H, T, d,
              int(chunk), _stream(dev))
    w.watch(w.sticky, "hoa_link_local")
    return R, U, M


def carry_scan(M: torch.Tensor, carry_in: Optional[torch.Tensor] = None,
               want_total: bool = False):
    """C_0 = carry_in (or I), C_{k+1} = M_k C_k -> (C (BH,K,d,d), total (BH,d,d) or None)."""
    _need_cuda(M, carry_in)
    BH, K, d, _ = M.shape
    _contig(M, "M")
    C = torch.empty_like(M)
    total = torch.empty(BH, d, d, dtype=torch.float32, device=M.device) if want_total else None
    _lib.call("hoa_carry_scan", _ptr(M), _ptr(carry_in), _ptr(C), _ptr(total), BH, K, d,
              _stream(M.device))
    return C, total


def vt_stride(T: int) -> int:
    return int(_lib.load().hoa_vt_stride(T))


def carry_apply(U: torch.Tensor, C: torch.Tensor, chunk: int, hat_dtype: torch.dtype,
                v_transposed: bool = False):
    """q^, k^ (BH,T,d) and v^ (BH,T,d), or v^T (BH,d,vt_stride(T)) if v_transposed."""
    _need_cuda(U, C)
    BH, T, _, d = U.shape
    dev = U.device
    qh = torch.empty(BH, T, d, dtype=hat_dtype, device=dev)
    kh = torch.empty(BH, T, d, dtype=hat_dtype, device=dev)
    vs = vt_stride(T) if v_transposed else 0
    vh = (torch.empty(BH, d, vs, dtype=hat_dtype, device=dev) if v_transposed
          else torch.empty(BH, T, d, dtype=hat_dtype, device=dev))
    _lib.call("hoa_carry_apply", _ptr(U), _ptr(C), _ptr(qh), _ptr(kh), _ptr(vh),
              _dtype_code(hat_dtype), vs, BH, T, d, int(chunk), _stream(dev))
    return qh, kh, vh


def attn_fwd(qh: torch.Tensor, kh: torch.Tensor, vh: torch.Tensor,
             softmax_scale: float, q_offset: int = 0) -> torch.Tensor:
    """Kernel (3), fp32 SIMT path: o = softmax(q^ k^T * scale, causal) v^ -> (BH,Tq,d) fp32.

    q^ (BH,Tq,d) holds global positions q_offset.., k^/v^ (BH,Tk,d) positions 0..Tk-1."""
    _need_cuda(qh, kh, vh)
    BH, Tq, d = qh.shape
    Tk = kh.shape[1]
    o = torch.empty(BH, Tq, d, dtype=torch.float32, device=qh.device)
    _lib.call("hoa_attn_fwd", _ptr(qh), _ptr(kh), _ptr(vh), _dtype_code(qh.dtype), _ptr(o),
              float(softmax_scale), BH, Tq, Tk, int(q_offset), d, _stream(qh.device))
    return o


def attn_tc_fwd(qh: torch.Tensor, kh: torch.Tensor, vhT: torch.Tensor, softmax_scale: float,
                status: Optional[torch.Tensor] = None, q_offset: int = 0) -> torch.Tensor:
    """Kernel (3), tcgen05 bf16 path (v^ transposed) -> o (BH,Tq,d) fp32.

    q^ (BH,Tq,d) holds global positions q_offset.., k^ (BH,Tk,d) and
    v^T (BH,d,vt_stride(Tk)) positions 0..Tk-1."""
    _need_cuda(qh, kh, vhT)
    BH, Tq, d = qh.shape
    Tk = kh.shape[1]
    if qh.dtype != torch.bfloat16:
        raise NotImplementedError("the tensor-core attention takes bf16 q^/k^/v^")
    if vhT.shape != (BH, d, vt_stride(Tk)):
        raise ValueError(f"v^T must be (BH, d, vt_stride(Tk)) = ({BH}, {d}, {vt_stride(Tk)})")
    o = torch.empty(BH, Tq, d, dtype=torch.float32, device=qh.device)
    w = _watch(qh.device) if status is None else None
    _lib.call("hoa_attn_tc_fwd", _ptr(qh), _ptr(kh), _ptr(vhT), _ptr(o),
              _ptr(status) if w is None else _ptr(w.sticky),
              float(softmax_scale), BH, Tq, Tk, int(q_offset), d, _stream(qh.device))
    if w is not None:
        w.watch(w.sticky, "hoa_attn_tc_fwd")
    return o


def out_transport(o: torch.Tensor, R: torch.Tensor, C: torch.Tensor, chunk: int, B: int, H: int,
                  out_dtype: torch.dtype) -> torch.Tensor:
    """Kernel (4): out_t = R_t C_k o_t -> (B,T,H*d) in out_dtype."""
    _need_cuda(o, R, C)
    BH, T, d = o.shape
    out = torch.empty(B, T, H * d, dtype=out_dtype, device=o.device)
    _lib.call("hoa_out_transport", _ptr(o), _ptr(R), _ptr(C), int(chunk), _ptr(out),
              _dtype_code(out_dtype), B, H, T, d, _stream(o.device))
    return out


def compose_paths(R: torch.Tensor, C: torch.Tensor, chunk: int, p_dtype: torch.dtype = torch.float32
                  ) -> torch.Tensor:
    """P_t = R_t C_{t/chunk} -> (BH, T, d, d) in p_dtype (the path products of return_geometry)."""
    _need_cuda(R, C)
    BH, T, d, _ = R.shape
    _contig(R, "R"); _contig(C, "C")
    if C.shape != (BH, (T + chunk - 1) // chunk, d, d):
        raise ValueError("C must be (BH, ceil(T/chunk), d, d)")
    P = torch.empty(BH, T, d, d, dtype=p_dtype, device=R.device)
    _lib.call("hoa_compose_paths", _ptr(R), _ptr(C), _ptr(P), _dtype_code(p_dtype), BH, T, d,
              int(chunk), _stream(R.device))
    return P


def core_geometry(a_all, qkv, n_heads, edge_scale, softmax_scale, out_dtype, hat_dtype, chunk,
                  a_bias=None, gen_layout="packed", geo_dtype=None):
    """The core region with the geometry kept: (heads (B,T,D), P (B,H,T,d,d), Hol (B,H,d,d)).

    Same kernels as core_forward, run stage by stage so that the local products
    R and the carries C survive: P_t = R_t C_{t/chunk} (hoa_compose_paths) and
    Hol = the carry scan's total through the closing edge t = T-1
    (core/attention_fast_chunked.py:95, 175-177).  P and Hol come in geo_dtype
    (default: out_dtype), as the reference returns them in x's dtype."""
    B, T, threeD = qkv.shape
    H = n_heads
    d = threeD // 3 // H
    geo_dtype = geo_dtype or out_dtype
    R, U, M = link_local(a_all, qkv, H, edge_scale, chunk, a_bias, gen_layout)
    C, total = carry_scan(M, want_total=True)
    tc = uses_tensor_cores(hat_dtype, d)
    qh, kh, vh = carry_apply(U, C, chunk, hat_dtype, v_transposed=tc)
    o = attn_tc_fwd(qh, kh, vh, softmax_scale) if tc else attn_fwd(qh, kh, vh, softmax_scale)
    heads = out_transport(o, R, C, chunk, B, H, out_dtype)
    del qh, kh, vh, o, U, M
    P = compose_paths(R, C, chunk, geo_dtype).view(B, H, T, d, d)
    return heads, P, total.view(B, H, d, d).to(geo_dtype)


# ---------------------------------------------------------------------------
# the general forms (any mask, wrap pairs, inert ablation), core/attention.py
# ---------------------------------------------------------------------------
def attn_general_fwd(qh: torch.Tensor, kh: torch.Tensor, vh: torch.Tensor, softmax_scale: float,
                     kw: Optional[torch.Tensor] = None, vw: Optional[torch.Tensor] = None,
                     mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention over all keys (fp32, (BH,T,d)): wrap pairs j > i use kw/vw when given;
    mask (T,T) bool/uint8, True = allowed, None = all allowed."""
    _need_cuda(qh, kh, vh, kw, vw, mask)
    BH, T, d = qh.shape
    for t, nm in ((qh, "qh"), (kh, "kh"), (vh, "vh"), (kw, "kw"), (vw, "vw")):
        if t is not None and (t.dtype != torch.float32 or t.shape != (BH, T, d) or not t.is_contiguous()):
            raise ValueError(f"{nm} must be a contiguous fp32 ({BH},{T},{d}) tensor")
    if (kw is None) != (vw is None):
        raise ValueError("kw and vw go together")
    m8 = None
    if mask is not None:
        if tuple(mask.shape) != (T, T):
            raise ValueError(f"mask must be ({T},{T})")
        m8 = mask.to(device=qh.device, dtype=torch.uint8).contiguous()
    o = torch.empty(BH, T, d, dtype=torch.float32, device=qh.device)
    _lib.call("hoa_attn_general_fwd", _ptr(qh), _ptr(kh), _ptr(vh), _ptr(kw), _ptr(vw), _ptr(m8),
              _ptr(o), float(softmax_scale), BH, T, d, _stream(qh.device))
    return o


def chain_matvec(x: torch.Tensor, M: torch.Tensor, transpose: bool = False) -> torch.Tensor:
    """y_t = M x_t (or M^T x_t), x (BH,T,d) fp32, M (BH,d,d) fp32."""
    _need_cuda(x, M)
    BH, T, d = x.shape
    _contig(x, "x"); _contig(M, "M")
    y = torch.empty_like(x)
    _lib.call("hoa_chain_matvec", _ptr(x), _ptr(M), _ptr(y), int(transpose), BH, T, d, _stream(x.device))
    return y


def apply_paths(x: torch.Tensor, R: torch.Tensor, C: torch.Tensor, chunk: int,
                transpose: bool = False) -> torch.Tensor:
    """y_t = P_t x_t (or P_t^T x_t) with P_t = R_t C_{t/chunk}; x (BH,T,d) fp32."""
    _need_cuda(x, R, C)
    BH, T, d = x.shape
    _contig(x, "x")
    y = torch.empty_like(x)
    _lib.call("hoa_apply_paths", _ptr(x), _ptr(R), _ptr(C), int(chunk), _ptr(y), int(transpose),
              BH, T, d, _stream(x.device))
    return y


def core_general(a_all, qkv, n_heads, edge_scale, softmax_scale, out_dtype, chunk, mode="causal",
                 mask=None, a_bias=None, gen_layout="packed", geometry=False, geo_dtype=None):
    """The core region for any mask and both modes of core/attention.py (fp32 throughout).

    "causal": q^ = P^T q etc.; the wrap pairs j > i (live when the mask allows any)
    see Hol k^_j and Hol v^_j (core/attention.py:156-165); out = P o.
    "inert": q~ = P q etc., no wrap pairs, out = P^T o (:166-169).
    Returns heads (B,T,D) in out_dtype, and with ``geometry`` also P (B,H,T,d,d) and
    Hol (B,H,d,d) in geo_dtype (default out_dtype)."""
    B, T, threeD = qkv.shape
    H = n_heads
    D = threeD // 3
    d = D // H
    R, U, M = link_local(a_all, qkv, H, edge_scale, chunk, a_bias, gen_layout)
    C, total = carry_scan(M, want_total=True)
    if mode == "causal":
        qh, kh, vh = carry_apply(U, C, chunk, torch.float32)
        wrap = mask is None or bool(torch.triu(mask.bool(), 1).any())
        kw = chain_matvec(kh, total) if wrap else None
        vw = chain_matvec(vh, total) if wrap else None
        o = attn_general_fwd(qh, kh, vh, softmax_scale, kw, vw, mask)
        heads = out_transport(o, R, C, chunk, B, H, out_dtype)
    elif mode == "inert":
        parts = qkv.view(B, T, H, 3, d).permute(3, 0, 2, 1, 4).float()        # (3,B,H,T,d)
        qt, kt, vt = (apply_paths(parts[i].reshape(B * H, T, d).contiguous(), R, C, chunk)
                      for i in range(3))
        o = attn_general_fwd(qt, kt, vt, softmax_scale, None, None, mask)
        heads = (apply_paths(o, R, C, chunk, transpose=True).view(B, H, T, d).permute(0, 2, 1, 3)
                 .reshape(B, T, D).to(out_dtype))
    else:
        raise ValueError("mode must be 'causal' or 'inert'")
    if not geometry:
        return heads
    geo_dtype = geo_dtype or out_dtype
    P = compose_paths(R, C, chunk, geo_dtype).view(B, H, T, d, d)
    return heads, P, total.view(B, H, d, d).to(geo_dtype)


def edge_gelu_split(h: torch.Tensor, split: bool) -> torch.Tensor:
    """GELU(h) (exact erf) of the fp32 hidden layer as the bf16 GEMM operand:
    (rows, cols) = bf16(g), or with ``split`` (rows, 2 cols) = [bf16(g) | bf16(g - bf16(g))]."""
    _need_cuda(h)
    if h.dtype != torch.float32 or h.dim() != 2 or not h.is_contiguous():
        raise ValueError("h must be a contiguous 2-D fp32 tensor")
    rows, cols = h.shape
    out = torch.empty(rows, (2 if split else 1) * cols, dtype=torch.bfloat16, device=h.device)
    _lib.call("hoa_edge_gelu_split", _ptr(h), _ptr(out), rows, cols, 1 if split else 0, _stream(h.device))
    return out


# fixed scale of the fp8 low half: g - bf16(g) is at most 2^-9 |g|, so 2^12 maps |g| up to 56
# onto e4m3's largest value (448, saturating beyond) and keeps remainders down to 2^-18 normal
SPLIT8_LO_SCALE = 4096.0


def edge_gelu_split8(h: torch.Tensor):
    """GELU(h) (exact erf) of the fp32 hidden layer as (bf16(g), e4m3(SPLIT8_LO_SCALE * (g - bf16(g))))
    (hoa_edge_gelu_split8), both (rows, cols)."""
    _need_cuda(h)
    if h.dtype != torch.float32 or h.dim() != 2 or not h.is_contiguous():
        raise ValueError("h must be a contiguous 2-D fp32 tensor")
    rows, cols = h.shape
    hi = torch.empty(rows, cols, dtype=torch.bfloat16, device=h.device)
    lo = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device=h.device)
    _lib.call("hoa_edge_gelu_split8", _ptr(h), _ptr(hi), _ptr(lo), rows, cols, SPLIT8_LO_SCALE,
              _stream(h.device))
    return hi, lo


_GEMM_WS = {}                   # (device, stream) -> workspace of the products that are queued there, one behind the other
_GEMM_WS_BYTES = 32 << 20


def _gemm_ws(dev, stream=None):
    """The GEMMs' workspace on ``dev``'s current stream.  A product may leave partial sums in it, so products that may run at
    once - on two streams, in a graph beside eager ones - have two; a captured one's is its graph's."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(_GEMM_WS_BYTES, dtype=torch.uint8, device=dev)
    key = dev.index, _stream(dev) if stream is None else stream
    ws = _GEMM_WS.get(key)
    if ws is None:
        with torch.inference_mode(False):
            ws = _GEMM_WS[key] = torch.empty(_GEMM_WS_BYTES, dtype=torch.uint8, device=dev)
    return ws


def edge_gemm_fp8_acc(lo: torch.Tensor, w: torch.Tensor, out: torch.Tensor, alpha: float) -> torch.Tensor:
    """out (M,N) fp32 += alpha * lo (M,K) e4m3 @ w (N,K) e4m3 ^T (hoa_edge_gemm_fp8_acc), in place."""
    _need_cuda(lo, w, out)
    if lo.dtype != torch.float8_e4m3fn or w.dtype != torch.float8_e4m3fn or out.dtype != torch.float32:
        raise ValueError("lo and w must be float8_e4m3fn, out float32")
    lo = _contig(lo, "lo")
    w = _contig(w, "w")
    out = _contig(out, "out")
    M, K = lo.shape
    N = w.shape[0]
    if w.shape[1] != K or out.shape != (M, N):
        raise ValueError(f"shapes: lo {tuple(lo.shape)}, w {tuple(w.shape)}, out {tuple(out.shape)}")
    dev = lo.device
    stream = _stream(dev)
    ws = _gemm_ws(dev, stream)
    _lib.call("hoa_edge_gemm_fp8_acc", _ptr(lo), _ptr(w), _ptr(out), float(alpha), M, N, K, _ptr(ws), _GEMM_WS_BYTES, stream)
    return out


def edge_gemm(hidden: torch.Tensor, wt: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """hidden (M,K) bf16 @ wt (K,N) bf16 + bias (N,) fp32 -> (M,N) fp32 (hoa_edge_gemm: one
    cuBLASLt GEMM with the bias in its epilogue)."""
    _need_cuda(hidden, wt)
    if hidden.dtype != torch.bfloat16 or wt.dtype != torch.bfloat16:
        raise NotImplementedError("hoa_edge_gemm takes bf16 operands")
    hidden = _contig(hidden, "hidden")
    wt = _contig(wt, "wt")
    M, K = hidden.shape
    if wt.shape[0] != K:
        raise ValueError(f"wt must be (K={K}, N), got {tuple(wt.shape)}")
    N = wt.shape[1]
    if bias is not None:
        if bias.dtype != torch.float32 or bias.numel() != N:
            raise ValueError("bias must be float32 with N elements")
        bias = bias.contiguous()
    dev = hidden.device
    stream = _stream(dev)
    ws = _gemm_ws(dev, stream)
    out = torch.empty(M, N, dtype=torch.float32, device=dev)
    try:
        _lib.call("hoa_edge_gemm", _ptr(hidden), _ptr(wt), _ptr(bias), _ptr(out), M, N, K, _ptr(ws),
                  _GEMM_WS_BYTES, stream)
    except _lib.HoaError as e:
        if e.status != _lib.HOA_ERR_UNSUPPORTED:
            raise
        # no cuBLASLt algorithm for this shape (e.g. rows not 16-byte aligned): torch's GEMM
        torch.mm(hidden, wt, out_dtype=torch.float32, out=out)
        if bias is not None:
            out += bias
    return out


def selftest_wait(max_cycles: int, device=None) -> Tuple[int, int, int, int]:
    """Diagnostic of the bounded device-side waits (hoa_selftest_wait): returns
    (status of the bounded wait, 1 if the second waiter left on the abort flag,
    the second waiter's wait in units of 1024 cycles, 1 if both waits gave up)."""
    dev = torch.device(device if device is not None else "cuda")
    out = torch.zeros(4, dtype=torch.int32, device=dev)
    _lib.call("hoa_selftest_wait", _ptr(out), int(max_cycles), _stream(dev))
    r = out.cpu().tolist()
    return r[0], r[1], r[2], r[3]


def uses_tensor_cores(hat_dtype: torch.dtype, d: int) -> bool:
    """Same rule as the library: bf16 hats with d % 8 == 0 and d <= 128."""
    return hat_dtype == torch.bfloat16 and d % 8 == 0 and d <= 128


def core_stages(a_all, qkv, n_heads, edge_scale, softmax_scale, out_dtype, hat_dtype, chunk,
                a_bias=None, gen_layout="packed"):
    """The core region as separate stage calls (same kernels as core_forward)."""
    B, T, threeD = qkv.shape
    H = n_heads
    d = threeD // 3 // H
    R, U, M = link_local(a_all, qkv, H, edge_scale, chunk, a_bias, gen_layout)
    C, _ = carry_scan(M)
    tc = uses_tensor_cores(hat_dtype, d)
    qh, kh, vh = carry_apply(U, C, chunk, hat_dtype, v_transposed=tc)
    o = attn_tc_fwd(qh, kh, vh, softmax_scale) if tc else attn_fwd(qh, kh, vh, softmax_scale)
    return out_transport(o, R, C, chunk, B, H, out_dtype)


# ---------------------------------------------------------------------------
# generation: pages of a cache, attention over them, the path step of one token.
# Page ids and rows that come from device memory are checked by the kernels; what
# they find (HOA_ERR_PAGES) is raised by poll_status() / check_status().
# ---------------------------------------------------------------------------
# These calls take a few microseconds on the GPU, so the host side is kept short: one
# pass of checks by device index, library functions and workspace sizes looked up once.
_INT = torch.int32
_SIZES = {}                     # (op, sizes) -> workspace bytes; the library computes them from the sizes alone
_DEVICES = {}                   # device index -> (SM count, address of the mapped status word)
_FN = {}                        # library functions by name
_ARRAYS = {}                    # ctypes array types by length


def _fn(name: str):
    f = _FN.get(name)
    if f is None:
        f = _FN[name] = getattr(_lib.load(), name)
    return f


# The ordinary case of these functions in C++ (csrc/hoa_torch.cpp): each tries it first; None means that
# the call is not ordinary (another device, an option, a mistake) and that the code below takes it.
_HOST = None
_HOST_FNS = ("hoa_pages_workspace_bytes", "hoa_pages_reserve", "hoa_pages_fork", "hoa_pages_free", "hoa_pages_compact",
             "hoa_paged_attn_workspace_bytes", "hoa_paged_attn_fwd", "hoa_path_step", "hoa_attn_fwd_lse", "hoa_attn_bwd_workspace_bytes",
             "hoa_attn_bwd", "hoa_path_bwd_workspace_bytes", "hoa_path_bwd", "hoa_adamw_step")


class _Declines:
    """Stands in for a C++ side that cannot be loaded: no call is ordinary."""
    def __getattr__(self, name):
        return lambda *a: None


def _host():
    global _HOST
    if _HOST is None:
        try:
            from . import _hoa_torch as m
        except ImportError as e:
            warnings.warn(f"_hoa_torch.so cannot be loaded ({e}): the generation and training operators' host side runs in Python, 10 "
                          "to 30 us a call slower.  Build it with `python -m holonomyawareattention_b200._build`", RuntimeWarning)
            _HOST = _Declines()
            return _HOST
        m.bind(*(ctypes.cast(_fn(n), ctypes.c_void_p).value for n in _HOST_FNS))
        _HOST = m
    return _HOST


def _done(name: str, r):
    """What the C++ side returned: the outputs, or a status to raise."""
    if type(r) is int:
        _lib.check(name, r)
    return r


def _device(idx: int):
    v = _DEVICES.get(idx)
    if v is None:
        v = _DEVICES[idx] = (torch.cuda.get_device_properties(idx).multi_processor_count,
                             _mapped_word(torch.device("cuda", idx)).ctypes.data)
        _host().device(idx, *v)
    return v


def _index(t) -> int:
    i = t.get_device()
    if i < 0:
        raise NotImplementedError("the B200 kernels need CUDA tensors (there is no CPU path)")
    return i


def _bytes_of(fn: str, *sizes) -> int:
    key = (fn, sizes)
    n = _SIZES.get(key)
    if n is None:
        if len(_SIZES) > 4096:
            _SIZES.clear()
        n = _SIZES[key] = int(_fn(fn)(*sizes))
    return n


def _current(idx: int):
    """Device ``idx`` is current inside."""
    return contextlib.nullcontext() if torch.cuda.current_device() == idx else torch.cuda.device(idx)


def _run(idx: int, name: str, *args) -> None:
    """Call ``name`` with device ``idx`` current, its status word and its current stream as the last arguments."""
    if torch.cuda.current_device() == idx:
        st = _fn(name)(*args, _device(idx)[1], torch._C._cuda_getCurrentRawStream(idx))
    else:
        with torch.cuda.device(idx):
            st = _fn(name)(*args, _device(idx)[1], torch._C._cuda_getCurrentRawStream(idx))
    if st != 0:
        _lib.check(name, st)


# Scratch of one call.  The library is called without the interpreter's lock, so the launches of two threads' calls may
# alternate on a stream: each call hands its parts over in memory of its own, which the allocator gives out again in
# stream order once the call has returned.  (The C++ side holds the lock over a call and keeps one buffer a stream.)
def _scratch(idx: int, n: int):
    """(address of n bytes of scratch on device idx's current stream, what keeps them alive)."""
    t = torch.empty(n, dtype=torch.uint8, device=torch.device("cuda", idx))
    return t.data_ptr(), t


def _longs(*values):
    """A host array of 64-bit integers (strides, addresses) for a call."""
    n = len(values)
    t = _ARRAYS.get(n)
    if t is None:
        t = _ARRAYS[n] = ctypes.c_longlong * n
    return t(*values)


def _bad_ints(t, name, shape, idx):
    _index(t)
    raise ValueError(f"{name} must be a contiguous int32 {shape} tensor on cuda:{idx}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _ints(t, name, shape, idx) -> None:
    if t.dtype is not _INT or t.shape != shape or t.get_device() != idx or not t.is_contiguous():
        _bad_ints(t, name, shape, idx)


def _books(table, lens, refs, page):
    """(device index, S, W, n_pages) of a bookkeeping state, checked."""
    idx = _index(table)
    if table.dim() != 2 or refs.dim() != 1 or table.numel() == 0 or refs.numel() == 0:
        raise ValueError("table must be (S, W) and refs (n_pages,), neither empty")
    S, W = table.shape
    n_pages = refs.shape[0]
    _ints(table, "table", (S, W), idx)
    if lens is not None:
        _ints(lens, "lens", (S,), idx)
    _ints(refs, "refs", (n_pages,), idx)
    if page < 1:
        raise ValueError("page must be at least 1")
    if S * W >= 2 ** 31 or n_pages >= 2 ** 31 or page >= 2 ** 31:      # (the library takes them as int)
        raise ValueError("S * W, n_pages and page must be below 2^31")
    return idx, S, W, n_pages


def _pool_args(pools, n_pages, idx):
    """(keep-alive, base pointers, bytes between pages, bytes of a page, count) of a list of pools."""
    n = len(pools)
    base, stride, size = [], [], []
    for t in pools:
        if t.dim() < 2 or t.shape[0] != n_pages or t.get_device() != idx:
            _index(t)
            raise ValueError(f"pools must be ({n_pages}, ...) tensors on cuda:{idx}")
        e = t.element_size()
        st = t.stride(0) * e
        if t.is_contiguous():
            size.append(t.numel() // max(1, n_pages) * e)      # (not st: a pool of one page may have any stride)
        else:
            p = t[0]
            if not p.is_contiguous() or t.stride(0) < p.numel():
                raise ValueError("the pages of a pool must be contiguous, one after another")
            size.append(p.numel() * e)
        base.append(t.data_ptr())
        stride.append(st)
    a = _longs(*base, *stride, *size)
    at = ctypes.addressof(a)
    return a, at, at + 8 * n, at + 16 * n, n


def pages_reserve(table, lens, refs, counts, page: int):
    """Row s grows by counts[s] tokens: (table, lens, refs) with the pages that it takes.

    table (S, W), lens (S,), refs (n_pages,), counts (S,): int32.  Free pages (refs == 0) are taken
    lowest index first, rows in order.  Without enough of them, or where a row would pass W pages, the
    state comes back unchanged and HOA_ERR_PAGES is reported (hoa_pages_reserve)."""
    r = (_HOST or _host()).pages_reserve(table, lens, refs, counts, page)
    if r is not None:
        return _done("hoa_pages_reserve", r)
    idx, S, W, n_pages = _books(table, lens, refs, page)
    _ints(counts, "counts", (S,), idx)
    out = torch.empty_like(table), torch.empty_like(lens), torch.empty_like(refs)
    n = _bytes_of("hoa_pages_workspace_bytes", S, n_pages)
    ws = _scratch(idx, n)
    _run(idx, "hoa_pages_reserve", table.data_ptr(), lens.data_ptr(), refs.data_ptr(), counts.data_ptr(), out[0].data_ptr(),
         out[1].data_ptr(), out[2].data_ptr(), S, W, n_pages, page, ws[0], n)
    return out


def pages_fork(pools, table, lens, refs, src, dst, page: int):
    """Row dst[i] becomes a copy of row src[i]: (table, lens, refs).

    src, dst (n,) int32; the dst rows are empty and differ.  Full pages are shared; a last page that
    is not full is copied, in every pool (n_pages, ...) of ``pools``, to a page of its own.  All or
    nothing, as pages_reserve (hoa_pages_fork)."""
    r = (_HOST or _host()).pages_fork(pools, table, lens, refs, src, dst, page)
    if r is not None:
        return _done("hoa_pages_fork", r)
    idx, S, W, n_pages = _books(table, lens, refs, page)
    n = src.numel()
    _ints(src, "src", (n,), idx)
    _ints(dst, "dst", (n,), idx)
    if n > S:
        raise ValueError("more forks than rows")
    _keep, base, stride, size, np_ = _pool_args(pools, n_pages, idx)
    out = torch.empty_like(table), torch.empty_like(lens), torch.empty_like(refs)
    nb = _bytes_of("hoa_pages_workspace_bytes", n, n_pages)
    ws = _scratch(idx, nb)
    _run(idx, "hoa_pages_fork", table.data_ptr(), lens.data_ptr(), refs.data_ptr(), src.data_ptr(), dst.data_ptr(), n,
         out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), S, W, n_pages, page, base, stride, size, np_, ws[0], nb)
    return out


def pages_free(table, lens, refs, rows, page: int):
    """The rows (n,) int32 end: (table, lens, refs); a page that no row holds any more is free
    (hoa_pages_free)."""
    r = (_HOST or _host()).pages_free(table, lens, refs, rows, page)
    if r is not None:
        return _done("hoa_pages_free", r)
    idx, S, W, n_pages = _books(table, lens, refs, page)
    n = rows.numel()
    _ints(rows, "rows", (n,), idx)
    out = torch.empty_like(table), torch.empty_like(lens), torch.empty_like(refs)
    _run(idx, "hoa_pages_free", table.data_ptr(), lens.data_ptr(), refs.data_ptr(), rows.data_ptr(), n, out[0].data_ptr(),
         out[1].data_ptr(), out[2].data_ptr(), S, W, n_pages, page)
    return out


def pages_compact(pools, table, refs):
    """The live pages move to 0 .. live-1 in every pool: (table, refs, live (1,)).

    The i-th free page below ``live`` receives the i-th live page at or above it (hoa_pages_compact)."""
    r = (_HOST or _host()).pages_compact(pools, table, refs)
    if r is not None:
        return _done("hoa_pages_compact", r)
    idx, S, W, n_pages = _books(table, None, refs, 1)
    _keep, base, stride, size, np_ = _pool_args(pools, n_pages, idx)
    table2, refs2 = torch.empty_like(table), torch.empty_like(refs)
    live = refs.new_empty(1)
    nb = _bytes_of("hoa_pages_workspace_bytes", 0, n_pages)
    ws = _scratch(idx, nb)
    _run(idx, "hoa_pages_compact", table.data_ptr(), refs.data_ptr(), table2.data_ptr(), refs2.data_ptr(), live.data_ptr(),
         S, W, n_pages, base, stride, size, np_, ws[0], nb)
    return table2, refs2, live


def pages_copy(pools, src, dst) -> None:
    """Page dst[i] = page src[i] in every pool (n_pages, ...), in place; no page is both (hoa_pages_copy)."""
    idx = _index(src)
    if not pools:
        return
    n = src.numel()
    _ints(src, "src", (n,), idx)
    _ints(dst, "dst", (n,), idx)
    n_pages = pools[0].shape[0]
    _keep, base, stride, size, np_ = _pool_args(pools, n_pages, idx)
    _run(idx, "hoa_pages_copy", base, stride, size, np_, src.data_ptr(), dst.data_ptr(), n, n_pages)


def _cache(k_pages, v_pages, idx):
    """(n_pages, Hk, page, d, dtype code, strides) of a k and a v pool that go together."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype or k_pages.numel() == 0:
        raise ValueError("k_pages and v_pages must be (n_pages, H, page, d), of one shape and type, not empty")
    st = k_pages.stride()
    if v_pages.stride() != st or (st[3] != 1 and k_pages.shape[3] != 1):
        raise ValueError("k_pages and v_pages must have the same strides, the innermost 1")
    if k_pages.get_device() != idx or v_pages.get_device() != idx:
        _index(k_pages), _index(v_pages)
        raise ValueError(f"k_pages and v_pages must be on cuda:{idx}")
    return (*k_pages.shape, _dtype_code(k_pages.dtype), _longs(*st[:3]))


def _row_table(table, B, idx):
    """(W, row stride) of a (B, W) table; rows may be strided (a view of a wider table)."""
    if table.dtype is not _INT or table.dim() != 2 or table.shape[0] != B or table.get_device() != idx or \
            (table.shape[1] > 1 and table.stride(1) != 1):
        _index(table)
        raise ValueError(f"table must be int32 ({B}, W) on cuda:{idx}, contiguous within a row")
    return table.shape[1], table.stride(0)


def _strides3(t):
    return _longs(*t.stride()[:3])


def pages_write(k, v, k_pages, v_pages, table, lens) -> None:
    """k, v (B, T, H, d) become the last T tokens of each row, in place: token t goes to position
    lens[b] - T + t (lens counts them; the pages are reserved).  hoa_pages_write."""
    idx = _index(k)
    n_pages, H, page, d, code, ps = _cache(k_pages, v_pages, idx)
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.shape[2:] != (H, d) or v.get_device() != idx or \
            (d > 1 and (k.stride(3) != 1 or v.stride(3) != 1)):
        raise ValueError(f"k and v must be (B, T, {H}, {d}) of one type, the innermost stride 1")
    B, T = k.shape[:2]
    if B == 0 or T == 0:
        return
    W, tw = _row_table(table, B, idx)
    _ints(lens, "lens", (B,), idx)
    _run(idx, "hoa_pages_write", k.data_ptr(), v.data_ptr(), _dtype_code(k.dtype), _strides3(k), _strides3(v),
         k_pages.data_ptr(), v_pages.data_ptr(), code, ps, table.data_ptr(), tw, lens.data_ptr(), B, T, H, d, page, W, n_pages)


def paged_attn_fwd(q, k_pages, v_pages, table, lens, softmax_scale: float, shared=None, paths=None, out_dtype=None):
    """Attention of B rows over a paged cache -> (out (B, Tq, H, d), lse (B, Tq, H) fp32).

    q (B, Tq, H, d) in the pools' type, any strides with the innermost 1; k_pages / v_pages
    (n_pages, Hk, page, d), H a multiple of Hk.  ``shared`` (n,) int32: the first pages of every row,
    read once for the batch; ``table`` (B, W) int32: each row's pages after them; ``lens`` (B,) int32:
    all keys of a row, the shared ones and its Tq newest included.  Query t sees the keys at positions
    0 .. lens[b] - Tq + t; one that sees none gives 0 and lse -inf.  ``paths`` (B, H, d, d) fp32 with
    Tq = 1: out = P o.  hoa_paged_attn_fwd."""
    if out_dtype is None or out_dtype is q.dtype:
        r = (_HOST or _host()).paged_attn_fwd(q, k_pages, v_pages, table, lens, softmax_scale, shared, paths)
        if r is not None:
            return _done("hoa_paged_attn_fwd", r)
    idx = _index(q)
    if q.dim() != 4 or q.numel() == 0:
        raise ValueError("q must be (B, Tq, H, d), not empty")
    B, Tq, H, d = q.shape
    n_pages, Hk, page, dk, code, ps = _cache(k_pages, v_pages, idx)
    qs = q.stride()
    if dk != d or q.dtype != k_pages.dtype or H % Hk != 0 or (d > 1 and qs[3] != 1):
        raise ValueError(f"q must be (B, Tq, H, {dk}) {k_pages.dtype} with H a multiple of {Hk}, the innermost stride 1")
    if d > 128:
        raise NotImplementedError(f"head dim {d} > 128")
    W, tw = _row_table(table, B, idx)
    _ints(lens, "lens", (B,), idx)
    n_shared = 0
    if shared is not None:
        n_shared = shared.numel()
        _ints(shared, "shared", (n_shared,), idx)
    if paths is not None:
        if Tq != 1:
            raise ValueError("paths go with one query token a row")
        _path(paths, "paths", (B, H, d, d), idx)
    out_dtype = out_dtype or q.dtype
    sms = _device(idx)[0]
    nb = _bytes_of("hoa_paged_attn_workspace_bytes", B, Tq, H, Hk, d, page, n_shared, W, sms)
    ws = _scratch(idx, nb)
    if out_dtype is q.dtype:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, Tq, H, d))
    else:
        out = q.new_empty((B, Tq, H, d), dtype=out_dtype)
    lse = q.new_empty((B, Tq, H), dtype=torch.float32)
    _run(idx, "hoa_paged_attn_fwd", q.data_ptr(), _longs(*qs[:3]), k_pages.data_ptr(), v_pages.data_ptr(), ps, code,
         shared.data_ptr() if n_shared else None, n_shared, table.data_ptr(), tw, W, lens.data_ptr(),
         paths.data_ptr() if paths is not None else None, out.data_ptr(), _dtype_code(out_dtype), lse.data_ptr(),
         softmax_scale, B, Tq, H, Hk, d, page, n_pages, sms, ws[0], nb)
    return out, lse


def _path(t, name, shape, idx) -> None:
    if t.dtype is not torch.float32 or t.shape != shape or t.get_device() != idx or not t.is_contiguous():
        _index(t)
        raise ValueError(f"{name} must be a contiguous fp32 {shape} tensor on cuda:{idx}")


def path_step(a, P, qkv, n_heads: int, edge_scale: float, k_pages, v_pages, table, lens, a_bias=None,
              gen_layout: str = "packed", P_out=None):
    """One token of every row: (P' (B, H, d, d) fp32, q^ (B, H, d) in the pools' type).

    P' = expm(skew(edge_scale (a + a_bias))) P with a (B, H*stride) fp32 the generators of the edge from
    the row's previous token (``gen_layout`` as core_forward); q^ = P'^T q, and k^, v^ go to slot
    lens[b] - 1 of the row's pages (table (B, W), lens (B,) with the token counted; reserve it first).
    qkv (B, 3D) holds [q | k | v] per head.  lens 1: no edge, P' = I.  lens 0: P' = P, q^ = 0, nothing
    written.  ``P_out`` may be P.  hoa_path_step."""
    if a_bias is None and gen_layout == "packed":
        r = (_HOST or _host()).path_step(a, P, qkv, n_heads, edge_scale, k_pages, v_pages, table, lens, P_out)
        if r is not None:
            return _done("hoa_path_step", r)
    idx = _index(qkv)
    H = n_heads
    n_pages, Hk, page, d, code, ps = _cache(k_pages, v_pages, idx)
    if Hk != H:
        raise ValueError(f"the pools must have n_heads = {H} heads, got {Hk}")
    if qkv.dim() != 2 or qkv.shape[1] != 3 * H * d or qkv.stride(1) != 1 or qkv.shape[0] == 0:
        raise ValueError(f"qkv must be (B, {3 * H * d}), contiguous within a row")
    if d < 2 or d > 120:
        raise NotImplementedError(f"head dim {d} (2 to 120)")
    B = qkv.shape[0]
    if a.dtype is not torch.float32:
        raise NotImplementedError("the path step takes fp32 generators")
    if gen_layout == "packed":
        a_code, width = _lib.HOA_F32, H * (d * (d - 1) // 2)
    else:
        a_code, width = _gen_code(a, gen_layout), _gen_width(H, d, gen_layout)
    if a.shape != (B, width) or not a.is_contiguous() or a.get_device() != idx:
        _index(a)
        raise ValueError(f"a must be a contiguous ({B}, {width}) tensor on cuda:{idx} for the {gen_layout} layout")
    if a_bias is not None:
        _check_bias(a_bias, width)
        if a_bias.get_device() != idx:
            _index(a_bias)
            raise ValueError(f"a_bias must be on cuda:{idx}")
    shape = (B, H, d, d)
    _path(P, "P", shape, idx)
    if P_out is None:
        P_out = torch.empty_like(P)
    else:
        _path(P_out, "P_out", shape, idx)
    W, tw = _row_table(table, B, idx)
    if W == 0:
        raise ValueError("table must have at least one page a row")
    _ints(lens, "lens", (B,), idx)
    qh = k_pages.new_empty((B, H, d))
    _run(idx, "hoa_path_step", a.data_ptr(), a_code, a_bias.data_ptr() if a_bias is not None else None, edge_scale,
         P.data_ptr(), P_out.data_ptr(), qkv.data_ptr(), _dtype_code(qkv.dtype), qkv.stride(0), qh.data_ptr(),
         k_pages.data_ptr(), v_pages.data_ptr(), code, ps, table.data_ptr(), tw, W, lens.data_ptr(), B, H, d, page, n_pages)
    return P_out, qh


# ---------------------------------------------------------------------------
# training: the backward passes of attention and of the path, the AdamW step
# ---------------------------------------------------------------------------
def _like(t, name, shape, dtype, idx) -> None:
    if t.get_device() != idx:
        _index(t)
        raise ValueError(f"{name} must be on cuda:{idx}, got {t.device}")
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} {dtype} tensor, got {tuple(t.shape)} {t.dtype}")


def _attn_shapes(qh, kh, vh, q_offset, softmax_scale):
    """(device index, dtype code, BH, Tq, Tk, d) of causal attention's inputs, checked."""
    idx = _index(qh)
    code = _dtype_code(qh.dtype)
    if qh.dim() != 3 or kh.dim() != 3 or qh.numel() == 0 or kh.numel() == 0:
        raise ValueError("q^ must be (BH, Tq, d) and k^, v^ (BH, Tk, d), none empty")
    BH, Tq, d = qh.shape
    Tk = kh.shape[1]
    _like(qh, "q^", (BH, Tq, d), qh.dtype, idx)
    _like(kh, "k^", (BH, Tk, d), qh.dtype, idx)
    _like(vh, "v^", (BH, Tk, d), qh.dtype, idx)
    if q_offset < 0 or q_offset + Tq > Tk:
        raise ValueError(f"the queries q_offset .. q_offset + Tq = {q_offset} .. {q_offset + Tq} must lie in the {Tk} keys")
    if not 0.0 < softmax_scale < math.inf:
        raise ValueError(f"softmax_scale must be positive and finite, got {softmax_scale}")
    if d > 128:
        raise NotImplementedError(f"head dim {d} (at most 128)")
    if BH > 65535 or Tk >= 2 ** 31 - 256:
        raise NotImplementedError(f"at most 65535 chains and 2^31 - 257 keys, got {BH} and {Tk}")
    return idx, code, BH, Tq, Tk, d


def attn_fwd_lse(qh: torch.Tensor, kh: torch.Tensor, vh: torch.Tensor, softmax_scale: float, q_offset: int = 0):
    """attn_fwd for training: (o (BH,Tq,d) fp32, lse (BH,Tq) fp32), lse the log-sum-exp of each row's scaled
    scores; bf16 (v^ row-major here) runs on the tensor cores where d % 8 == 0.  hoa_attn_fwd_lse."""
    r = (_HOST or _host()).attn_fwd_lse(qh, kh, vh, softmax_scale, q_offset)
    if r is not None:
        return _done("hoa_attn_fwd_lse", r)
    idx, code, BH, Tq, Tk, d = _attn_shapes(qh, kh, vh, q_offset, softmax_scale)
    o = qh.new_empty((BH, Tq, d), dtype=torch.float32)
    lse = qh.new_empty((BH, Tq), dtype=torch.float32)
    _run(idx, "hoa_attn_fwd_lse", qh.data_ptr(), kh.data_ptr(), vh.data_ptr(), code, o.data_ptr(), lse.data_ptr(), softmax_scale,
         BH, Tq, Tk, q_offset, d)
    return o, lse


def attn_bwd(qh: torch.Tensor, kh: torch.Tensor, vh: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, do: torch.Tensor,
             softmax_scale: float, q_offset: int = 0):
    """Gradients (dq^, dk^, dv^) of causal attention for the gradient ``do`` (BH,Tq,d) of its output.

    q^ (BH,Tq,d), k^ and v^ (BH,Tk,d), do and the results share a type (fp32 or bf16); o and lse are what
    attn_fwd_lse gave.  The probabilities are recomputed from lse; sums are fp32 and of a fixed order.
    hoa_attn_bwd."""
    r = (_HOST or _host()).attn_bwd(qh, kh, vh, o, lse, do, softmax_scale, q_offset)
    if r is not None:
        return _done("hoa_attn_bwd", r)
    idx, code, BH, Tq, Tk, d = _attn_shapes(qh, kh, vh, q_offset, softmax_scale)
    _like(o, "o", (BH, Tq, d), torch.float32, idx)
    _like(lse, "lse", (BH, Tq), torch.float32, idx)
    _like(do, "do", (BH, Tq, d), qh.dtype, idx)
    dq, dk, dv = torch.empty_like(qh), torch.empty_like(kh), torch.empty_like(vh)
    at = qh.data_ptr() | kh.data_ptr() | vh.data_ptr() | do.data_ptr() | dq.data_ptr() | dk.data_ptr() | dv.data_ptr()
    nb = _bytes_of("hoa_attn_bwd_workspace_bytes", BH, Tq, Tk, d, code, int(at % 16 == 0))
    ws = _scratch(idx, nb)
    _run(idx, "hoa_attn_bwd", qh.data_ptr(), kh.data_ptr(), vh.data_ptr(), o.data_ptr(), lse.data_ptr(), do.data_ptr(), code,
         dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), softmax_scale, BH, Tq, Tk, q_offset, d, ws[0], nb)
    return dq, dk, dv


def path_bwd(a_all: torch.Tensor, R: torch.Tensor, C: torch.Tensor, chunk: int, n_heads: int, edge_scale: float, hats, dhats,
             a_bias: Optional[torch.Tensor] = None, gen_layout: str = "packed", out_dtype: Optional[torch.dtype] = None):
    """Gradients through the path products: (da (B,T,H*m) fp32 of the raw generators, dqkv (B,T,3D)).

    a_all, a_bias, edge_scale, gen_layout as link_local's (da has a_all's layout), R and C what link_local and
    carry_scan gave for ``chunk``.  hats: (q^, k^, v^, o), each (BH,T,d), o in fp32; dhats: (dq^, dk^, dv^, do^), the
    gradients of the first three and P^T dout (apply_paths with transpose).  q^, k^, v^ and dhats share a type, which
    dqkv has too unless ``out_dtype`` says otherwise.  The gradient of the closing edge (t = T - 1) is 0, as the causal
    forward does not use it.  hoa_path_bwd."""
    if a_bias is None and out_dtype is None and gen_layout == "packed":
        r = (_HOST or _host()).path_bwd(a_all, R, C, chunk, n_heads, edge_scale, hats, dhats)
        if r is not None:
            return _done("hoa_path_bwd", r)
    idx = _index(a_all)
    if a_all.dim() != 3 or R.dim() != 4 or len(hats) != 4 or len(dhats) != 4:
        raise ValueError("a_all must be (B,T,H*stride), R (BH,T,d,d), hats and dhats four tensors each")
    if a_all.dtype is not torch.float32:
        raise NotImplementedError("the path's backward pass takes fp32 generators")
    B, T, H, d = a_all.shape[0], a_all.shape[1], n_heads, R.shape[3]
    if B < 1 or T < 1 or H < 1 or chunk < 1:
        raise ValueError("B, T, n_heads and chunk must be at least 1")
    if d < 2 or d > 120:
        raise NotImplementedError(f"head dim {d} (2 to 120)")
    a_code, width = _gen_code(a_all, gen_layout), _gen_width(H, d, gen_layout)
    dt = hats[0].dtype
    code = _dtype_code(dt)
    out_dtype = out_dtype or dt
    _like(a_all, "a_all", (B, T, width), torch.float32, idx)
    _check_bias(a_bias, width)
    if a_bias is not None and a_bias.get_device() != idx:
        raise ValueError(f"a_bias must be on cuda:{idx}, got {a_bias.device}")
    _like(R, "R", (B * H, T, d, d), torch.float32, idx)
    _like(C, "C", (B * H, (T + chunk - 1) // chunk, d, d), torch.float32, idx)
    for i, name in enumerate(("q^", "k^", "v^", "o")):
        _like(hats[i], name, (B * H, T, d), dt if i < 3 else torch.float32, idx)
    for i, name in enumerate(("dq^", "dk^", "dv^", "do^")):
        _like(dhats[i], name, (B * H, T, d), dt, idx)
    chunk = min(chunk, T)
    with _current(idx):
        nb = _bytes_of("hoa_path_bwd_workspace_bytes", B, H, T, d, chunk)
    if nb == 0:
        raise NotImplementedError(f"B H T = {B} {H} {T} with chunk {chunk} is too large")
    ws = _scratch(idx, nb)
    da = torch.empty_like(a_all)
    dqkv = a_all.new_empty((B, T, 3 * H * d), dtype=out_dtype)
    _run(idx, "hoa_path_bwd", a_all.data_ptr(), a_code, a_bias.data_ptr() if a_bias is not None else None, edge_scale, R.data_ptr(),
         C.data_ptr(), chunk, *(t.data_ptr() for t in hats), *(t.data_ptr() for t in dhats), code, da.data_ptr(), dqkv.data_ptr(),
         _dtype_code(out_dtype), B, H, T, d, ws[0], nb)
    return da, dqkv


ADAMW_BLOCK = 256               # elements of a block of 8-bit moments


_GRAPH_WRITES = [0]


def graph_writes() -> int:
    """How many steps have been captured so far."""
    return _GRAPH_WRITES[0]


def written_by_graphs(t: torch.Tensor) -> bool:
    """Whether a captured adamw_step writes ``t``: its replays change it and no version says so."""
    return getattr(t.untyped_storage(), "_hoa_written_by_graphs", False)


def _pointers(ts):
    return (ctypes.c_void_p * len(ts))(*(None if t is None else t.data_ptr() for t in ts))


def _apart(params, grads, exp_avg, exp_avg_sq, masters, scales) -> None:
    """What a step writes shares no memory with anything else that it writes or reads (an fp32 parameter may be its own master)."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()

    own = [None if p.dtype is not torch.float32 else p.data_ptr() for p in params]
    written = [span(t) for ts in (params, exp_avg, exp_avg_sq, scales or ()) for t in ts if t.numel()]
    written += [span(t) for t, at in zip(masters or (), own) if t.numel() and t.data_ptr() != at]
    both = sorted([(*x, 1) for x in written] + [(*span(t), 0) for t in grads if t.numel()])
    end = [0, 0]                                                  # of the grads and of the written ones so far
    for a, b, writes in both:
        if a < end[1] or (writes and a < end[0]):
            raise ValueError("params, masters, moments and scales must share no memory with one another or with the grads")
        end[writes] = max(end[writes], b)


def adamw_step(params, grads, exp_avg, exp_avg_sq, step: torch.Tensor, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.01, masters=None, scales=None) -> None:
    """One AdamW step over all tensors of the lists, in place, in one launch (256 tensors each).

    params fp32 or bf16, grads fp32 or bf16; ``masters``: fp32 copies that the step is made on (the parameter is then the
    copy, rounded), or None.  exp_avg and exp_avg_sq: fp32 moments; or, with ``scales``, 8-bit ones: float8_e4m3fn tensors
    of m and of sqrt(v), in blocks of ADAMW_BLOCK elements with scales[i] (2, blocks) fp32 (value = e4m3 * scale), rounded to the
    nearest for betas up to 15/16 and 0.95, above by a chance that follows from the element's place and ``step`` (to the nearest
    they would stop moving).
    ``step``: int32 (1,) on the device, the number of this step, from 1 (read on the device: a captured step may be replayed;
    torch counts no writes of the replays, so nothing is kept from then on that was laid out from these params).
    hoa_adamw_step."""
    r = (_HOST or _host()).adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr, betas[0], betas[1], eps, weight_decay, masters, scales)
    if r is not None:
        _done("hoa_adamw_step", r)
        return
    n = len(params)
    lists = [("grads", grads), ("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)]
    lists += [(k, v) for k, v in (("masters", masters), ("scales", scales)) if v is not None]
    for name, v in lists:
        if len(v) != n:
            raise ValueError(f"{name} must have {n} tensors as params, got {len(v)}")
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0):
        raise ValueError("betas must lie in [0, 1) and eps be at least 0")
    if n == 0:
        return
    idx = _index(params[0])
    _ints(step, "step", (1,), idx)
    p_dt, g_dt = params[0].dtype, grads[0].dtype
    p_code, g_code = _dtype_code(p_dt), _dtype_code(g_dt)
    moment = torch.float32 if scales is None else torch.float8_e4m3fn
    # (one pass, the names only where something is wrong: a step of a few tensors takes as long as these checks)
    rows = zip(params, grads, exp_avg, exp_avg_sq)
    if not all(p.get_device() == g.get_device() == m.get_device() == v.get_device() == idx and p.dtype is p_dt and g.dtype is g_dt
               and m.dtype is moment and v.dtype is moment and p.shape == g.shape == m.shape == v.shape and p.is_contiguous()
               and g.is_contiguous() and m.is_contiguous() and v.is_contiguous() for p, g, m, v in rows):
        for i, p in enumerate(params):
            _like(p, f"params[{i}]", p.shape, p_dt, idx)
            _like(grads[i], f"grads[{i}]", p.shape, g_dt, idx)
            _like(exp_avg[i], f"exp_avg[{i}]", p.shape, moment, idx)
            _like(exp_avg_sq[i], f"exp_avg_sq[{i}]", p.shape, moment, idx)
    sizes = [p.numel() for p in params]
    if len({p.data_ptr() for p, k in zip(params, sizes) if k}) != sum(1 for k in sizes if k):
        raise ValueError("params must be different tensors: the step of one is not a place for another's")
    if masters is not None:
        for i, p in enumerate(params):
            _like(masters[i], f"masters[{i}]", p.shape, torch.float32, idx)
    if scales is not None:
        for i, n_i in enumerate(sizes):
            _like(scales[i], f"scales[{i}]", (2, -(-n_i // ADAMW_BLOCK)), torch.float32, idx)
    _apart(params, grads, exp_avg, exp_avg_sq, masters, scales)
    with _current(idx):
        if idx not in _DEVICES and not torch.cuda.is_current_stream_capturing():
            _device(idx)                       # (from now on the C++ side takes such calls)
        _lib.check("hoa_adamw_step", _fn("hoa_adamw_step")(
            _pointers(params), p_code, _pointers(masters) if masters is not None else None, _pointers(grads), g_code,
            _pointers(exp_avg), _pointers(exp_avg_sq), _pointers(scales) if scales is not None else None, 32 if scales is None else 8,
            _longs(*sizes), n, step.data_ptr(), lr, betas[0], betas[1], eps, weight_decay, torch._C._cuda_getCurrentRawStream(idx)))
        if torch.cuda.is_current_stream_capturing():
            for p in params:
                p.untyped_storage()._hoa_written_by_graphs = True
            _GRAPH_WRITES[0] += 1
    # written behind autograd's back: what was saved of them, or laid out from them, is out of date
    torch.autograd.graph.increment_version([t for t in (*params, *(masters or ())) if not t.is_inference()])
