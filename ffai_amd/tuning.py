"""Tuning a router and low-rank adapters beside frozen experts, and serving
many adapters at once, over PyTorch device buffers through the C ABI.

    counts and losses   b = balance_loss(router, logits, topk_idx, mask=mask)
    combine             dY, dw = unpermute_backward(d_out, Y, inv_perm, topk_weight)
    router              dl = router_backward(router, logits, topk_idx, d_weight=dw,
                                             counts=b.counts, balance_coef=.01, mask=mask)
    adapters            y = LoRAAdapters(a, b, scale).apply(x, adapter, y)
                        dx, da, db = adapters.backward(x, dy, adapter, dx=dx)

Gradients are plain results, not recorded by autograd. While autograd records,
balance_loss and apply refuse tensors that require a gradient, and every function
refuses to write into one: call them under torch.no_grad() or in a
torch.autograd.Function. A tensor of the caller's that a call writes counts as
changed in place, so that autograd notices where it had saved it.

Every function takes contiguous tensors of one device, checks them before any
launch, and runs on `stream` (default: that device's current stream), on which
its results and its workspace are allocated: a result used on another stream has
to be waited for there, and all calls can be captured into a graph. PyTorch only
provides memory and streams; every computation is a libmoehip.so kernel.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import Lora, check
from .layer import MoERouter, moe_dtype

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_MASK = (torch.bool, torch.uint8)
_I32, _F32 = (torch.int32,), (torch.float32,)

# The current device, and the handle of a device's current stream, without the
# objects of torch.cuda around them (0.1 us each instead of 0.3 and 1.8: a call's
# host work is as long as its kernels where there are few rows).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)


_grad_enabled = torch.is_grad_enabled
# (without the public call's look at its argument: 0.15 us)
_changed = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)


def _refuse_grad(name: str):
    raise ValueError(f"{name} requires a gradient, which this call does not record: call it under torch.no_grad() or in a "
                     "torch.autograd.Function")


def _check(name: str, t: Optional[torch.Tensor], shape, dtypes, index: int) -> Optional[int]:
    """The address of a tensor the kernels read or write through a raw pointer
    (None for None): of `shape`, one of `dtypes`, on GPU `index` (-1: on the
    host), contiguous."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.shape == shape and t.dtype in dtypes and t.get_device() == index and t.is_contiguous():
        return t.data_ptr()
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} dtype {t.dtype} is not {' or '.join(str(d) for d in dtypes)}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the others on {'cpu' if index < 0 else f'cuda:{index}'}")
    raise ValueError(f"{name} must be contiguous")


def _rows(name: str, t, dims: int) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dim() != dims:
        raise ValueError(f"{name} must be a tensor of {dims} dimensions")
    if t.dtype not in _FLOATS:
        raise ValueError(f"{name} dtype {t.dtype} is not a float32, float16 or bfloat16")
    if t.shape[0] <= 0:
        raise ValueError(f"{name} must have rows")
    return t


class _on:
    """The device and stream a call runs on where they are not the current ones."""
    __slots__ = ("_ctx",)

    def __init__(self, index: int, stream):
        self._ctx = torch.cuda.device(index) if stream is None else torch.cuda.stream(stream)
        self._ctx.__enter__()

    def leave(self):
        self._ctx.__exit__(None, None, None)


def _begin(index: int, stream):
    """(stream handle, context to leave afterwards or None) of a call on GPU
    `index`: `stream`, or the current stream of that GPU, which need not be the
    current one."""
    if index < 0:
        raise ValueError("tensors must be on a GPU")
    if stream is None:
        return _raw_stream(index), (None if index == _current_device() else _on(index, None))
    if stream.device.index != index:
        raise ValueError(f"stream is on {stream.device}, the tensors on cuda:{index}")
    return stream.cuda_stream, _on(index, stream)


class BalanceLoss(NamedTuple):
    """counts [E + 1] int32 (the last: counted rows), prob_sum [E] float32,
    losses [2] float32 (balance, z), as moe_balance_loss defines them."""
    counts: torch.Tensor
    prob_sum: torch.Tensor
    losses: torch.Tensor


def balance_loss(router: MoERouter, logits: torch.Tensor, topk_idx: torch.Tensor,
                 mask: Optional[torch.Tensor] = None, stream=None) -> BalanceLoss:
    """Per-expert counts, probability sums and the balance and z losses of
    logits [T, E] and their picks topk_idx [T, k] int32, over the rows where
    mask [T] (bool or uint8) is true."""
    T, E, k = _rows("logits", logits, 2).shape[0], router.nExperts, router.topK
    at, dev = logits.get_device(), logits.device
    lp = _check("logits", logits, (T, E), _FLOATS, at)
    ip = _check("topk_idx", topk_idx, (T, k), _I32, at)
    mp = _check("mask", mask, (T,), _MASK, at)
    if logits.requires_grad and _grad_enabled():
        _refuse_grad("logits")
    st, ctx = _begin(at, stream)
    try:
        lib = _lib.load()
        counts = torch.empty(E + 1, dtype=torch.int32, device=dev)
        prob_sum = torch.empty(E, dtype=torch.float32, device=dev)
        losses = torch.empty(2, dtype=torch.float32, device=dev)
        need = lib.moe_balance_loss_workspace_bytes(T, E)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        check(lib.moe_balance_loss(lp, moe_dtype(logits.dtype), T, E, k, router.gatingMode,
                                   router.logitScale, ip, mp, counts.data_ptr(), prob_sum.data_ptr(),
                                   losses.data_ptr(), None if ws is None else ws.data_ptr(), need, st))
    finally:
        if ctx is not None:
            ctx.leave()
    return BalanceLoss(counts, prob_sum, losses)


def router_backward(router: MoERouter, logits: torch.Tensor, topk_idx: torch.Tensor,
                    d_weight: Optional[torch.Tensor] = None,
                    counts: Optional[torch.Tensor] = None, balance_coef: float = 0.0,
                    z_coef: float = 0.0, mask: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Gradient of logits [T, E] for d_weight [T, k] float32, the gradient of
    the routing weights, and balance_coef * balance + z_coef * z, whose counts
    [E + 1] balance_loss returned (or their sum over a job's ranks)."""
    T, E, k = _rows("logits", logits, 2).shape[0], router.nExperts, router.topK
    at, dt = logits.get_device(), logits.dtype
    lp = _check("logits", logits, (T, E), _FLOATS, at)
    ip = _check("topk_idx", topk_idx, (T, k), _I32, at)
    dp = _check("d_weight", d_weight, (T, k), _F32, at)
    cp = _check("counts", counts, (E + 1,), _I32, at)
    mp = _check("mask", mask, (T,), _MASK, at)
    bp = _check("router.expertBias", router.expertBias, (E,), _F32, at)
    sp = _check("router.expertScale", router.expertScale, (E,), _F32, at)
    op = _check("out", out, (T, E), (dt,), at)
    if out is not None and out.requires_grad and _grad_enabled():
        _refuse_grad("out")
    st, ctx = _begin(at, stream)
    try:
        given = out is not None
        if not given:
            out = torch.empty_like(logits)
            op = out.data_ptr()
        check(_lib.load().moe_router_backward(
            lp, moe_dtype(dt), T, E, k, router.gatingMode, int(bool(router.normTopKProb)), bp,
            router.logitScale, router.routedScale, sp, ip, dp, cp, balance_coef, z_coef, mp, op, st))
        if given:
            _changed((out,))
    finally:
        if ctx is not None:
            ctx.leave()
    return out


def unpermute_backward(d_out: torch.Tensor, Y: torch.Tensor, inv_perm: torch.Tensor,
                       topk_weight: torch.Tensor, dY: Optional[torch.Tensor] = None, stream=None):
    """Gradient of the weighted combine of expert rows Y [T * k, hidden] for
    d_out [T, hidden]: (dY, d_weight [T, k] float32). inv_perm (T * k int32)
    comes from the dispatch plan, each position once; a position past T * k has a
    zero d_weight, and rows that no position names are not written (give dY to
    have them defined). dY may be Y itself."""
    T, H = _rows("d_out", d_out, 2).shape
    at, dts = d_out.get_device(), (d_out.dtype,)
    k = _rows("topk_weight", topk_weight, 2).shape[1]
    gp = _check("d_out", d_out, (T, H), _FLOATS, at)
    yp = _check("Y", Y, (T * k, H), dts, at)
    wp = _check("topk_weight", topk_weight, (T, k), _F32, at)
    flat = isinstance(inv_perm, torch.Tensor) and inv_perm.dim() == 1
    ip = _check("inv_perm", inv_perm, (T * k,) if flat else (T, k), _I32, at)
    op = _check("dY", dY, (T * k, H), dts, at)
    if dY is not None and dY.requires_grad and _grad_enabled():
        _refuse_grad("dY")
    st, ctx = _begin(at, stream)
    try:
        given = dY is not None
        if not given:
            dY = torch.empty_like(Y)
            op = dY.data_ptr()
        dw = torch.empty_like(topk_weight)
        check(_lib.load().moe_unpermute_backward(gp, yp, ip, wp, T, H, k, op, dw.data_ptr(),
                                                 moe_dtype(d_out.dtype), st))
        if given:
            _changed((dY,))
    finally:
        if ctx is not None:
            ctx.leave()
    return dY, dw


@dataclass(frozen=True, eq=False)
class LoRAAdapters:
    """A stack of low-rank adapters of one [N, K] projection: a [G, R, K],
    b [G, N, R], scale [G] float32 (None: 1). Ranks that differ are padded
    with zeros to a multiple of 8, at most 128. The tensors may be updated in
    place (a slot overwritten, an optimiser's step) and moved (their .data set);
    the latter, also where only shape, type or spacing change, is checked again by
    the next call."""
    a: torch.Tensor
    b: torch.Tensor
    scale: Optional[torch.Tensor] = None

    def __post_init__(self):
        G, R, K = _rows("a", self.a, 3).shape
        N = _rows("b", self.b, 3).shape[1]
        at = self.a.get_device()
        desc = Lora(_check("a", self.a, (G, R, K), _FLOATS, at),
                    _check("b", self.b, (G, N, R), (self.a.dtype,), at),
                    _check("scale", self.scale, (G,), _F32, at),
                    moe_dtype(self.a.dtype), R, N, K, G)
        check(_lib.load().moe_validate_lora(C.byref(desc)))
        # (workspaces grow with the rows: none for the most is none for all)
        object.__setattr__(self, "_no_workspace", _lib.load().moe_lora_workspace_bytes(C.byref(desc), 1 << 23) == 0)
        object.__setattr__(self, "_struct", desc)
        object.__setattr__(self, "_ref", C.byref(desc))
        object.__setattr__(self, "_dims", (N, K))
        a, b, s = self.a, self.b, self.scale
        object.__setattr__(self, "_as", (a.data_ptr(), b.data_ptr(), a.shape, b.shape, a.dtype, b.dtype))
        object.__setattr__(self, "_scale_as", None if s is None else (s.data_ptr(), s.shape, s.dtype))

    def _current(self) -> Lora:
        """The descriptor, of the memory the tensors have now."""
        a, b, s = self.a, self.b, self.scale
        if ((a.data_ptr(), b.data_ptr(), a.shape, b.shape, a.dtype, b.dtype) != self._as
                or not (a.is_contiguous() and b.is_contiguous())
                or (s is not None and ((s.data_ptr(), s.shape, s.dtype) != self._scale_as or not s.is_contiguous()))):
            self.__post_init__()
        return self._struct

    def apply(self, x: torch.Tensor, adapter: torch.Tensor, y: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """y + scale * b (a x) for x [T, K], row t with adapter[t] (int32; -1:
        none), sums in float32; in a 16-bit type the inner ones enter the second
        product as two parts, 16 (bfloat16) or 22 bits. y [T, N] is the shared projection's output (None: zeros); the
        result goes to out, by default to y itself."""
        self._current()
        a, b, s, (N, K) = self.a, self.b, self.scale, self._dims
        dts, at = (a.dtype,), a.get_device()
        T = _rows("x", x, 2).shape[0]
        xp = _check("x", x, (T, K), dts, at)
        ap = _check("adapter", adapter, (T,), _I32, at)
        yp = _check("y", y, (T, N), dts, at)
        op = _check("out", out, (T, N), dts, at)
        if _grad_enabled() and (x.requires_grad or a.requires_grad or b.requires_grad
                                or (y is not None and y.requires_grad) or (out is not None and out.requires_grad)
                                or (s is not None and s.requires_grad)):
            _refuse_grad(next(n for n, t in (("x", x), ("a", a), ("b", b), ("y", y), ("out", out), ("scale", s))
                              if t is not None and t.requires_grad))
        st, ctx = _begin(at, stream)
        try:
            lib = _lib.load()
            given = out is not None or y is not None
            if out is None:
                out = torch.empty(T, N, dtype=x.dtype, device=x.device) if y is None else y
                op = out.data_ptr()
            need = 0 if self._no_workspace else lib.moe_lora_workspace_bytes(self._ref, T)
            ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
            check(lib.moe_lora_apply(self._ref, xp, T, ap, yp, op, None if ws is None else ws.data_ptr(),
                                     need, st))
            if given:
                _changed((out,))
        finally:
            if ctx is not None:
                ctx.leave()
        return out

    def backward(self, x: torch.Tensor, dy: torch.Tensor, adapter: torch.Tensor,
                 dx: Optional[torch.Tensor] = None, dx_out: Optional[torch.Tensor] = None,
                 need_dx: bool = True, stream=None):
        """(dx, da, db) of apply for dy [T, N], the gradient of its result.
        dx [T, K] is the gradient from the shared projection that the adapters'
        is added to (None: zeros); the sum goes to dx_out, by default to dx
        itself. need_dx=False leaves it out (dx is then None)."""
        self._current()
        (N, K), dts, at = self._dims, (self.a.dtype,), self.a.get_device()
        T = _rows("x", x, 2).shape[0]
        xp = _check("x", x, (T, K), dts, at)
        yp = _check("dy", dy, (T, N), dts, at)
        ap = _check("adapter", adapter, (T,), _I32, at)
        dp = _check("dx", dx, (T, K), dts, at)
        op = _check("dx_out", dx_out, (T, K), dts, at)
        if not need_dx and (dx is not None or dx_out is not None):
            raise ValueError("dx or dx_out given with need_dx=False")
        into = dx if dx_out is None else dx_out
        if into is not None and into.requires_grad and _grad_enabled():
            _refuse_grad("dx" if dx_out is None else "dx_out")
        st, ctx = _begin(at, stream)
        try:
            lib = _lib.load()
            dx_out = into
            if need_dx and into is None:
                dx_out = torch.empty(T, K, dtype=x.dtype, device=x.device)
            if need_dx:
                op = dx_out.data_ptr()
            da, db = torch.empty_like(self.a), torch.empty_like(self.b)
            need = lib.moe_lora_backward_workspace_bytes(self._ref, T)
            ws = torch.empty(need, dtype=torch.uint8, device=x.device)
            check(lib.moe_lora_backward(self._ref, xp, yp, T, ap, dp, op, da.data_ptr(), db.data_ptr(),
                                        ws.data_ptr(), need, st))
            if into is not None:
                _changed((into,))
        finally:
            if ctx is not None:
                ctx.leave()
        return dx_out, da, db
