"""Tuning a router and low-rank adapters beside frozen experts, taking gradients
through those experts, and serving many adapters at once, over PyTorch device
buffers through the C ABI.

    counts and losses   b = balance_loss(router, logits, topk_idx, mask=mask)
    combine             dY, dw = unpermute_backward(d_out, Y, inv_perm, topk_weight)
    router              dl = router_backward(router, logits, topk_idx, d_weight=dw,
                                             counts=b.counts, balance_coef=.01, mask=mask)
    adapters            y = LoRAAdapters(a, b, scale).apply(x, adapter, y)
                        dx, da, db = adapters.backward(x, dy, adapter, dx=dx)
    experts             y, kept = FrozenExperts(gate, up, down).forward(x, topk_idx, topk_weight)
                        dx, dw = experts.backward(d_out, kept)
    and their parts     expert_matmul_backward, activation_save, activation_backward,
                        permute_backward; add_rmsnorm_backward before the layer

Gradients are plain results, not recorded by autograd. While autograd records,
balance_loss, apply, activation_save and the experts' forward refuse tensors that
require a gradient, and every function
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
from .layer import MoERouter, StackedExperts, moe_dtype

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


# ---------------------------------------- gradients through frozen experts --

def _stack(name: str, p: StackedExperts, at: int):
    """The descriptor of a quantised stack, its tensors checked."""
    if not isinstance(p, StackedExperts):
        raise ValueError(f"{name} must be StackedExperts")
    E, N, words = _dims(f"{name}.weight", p.weight, 3)
    groups = _dims(f"{name}.scales", p.scales, 3)[2]
    if words * 32 != groups * p.group_size * p.bits:
        raise ValueError(f"{name}: {words} words a row do not hold {groups} groups of {p.group_size} {p.bits}-bit codes")
    _check(f"{name}.weight", p.weight, (E, N, words), _WORDS, at)
    _check(f"{name}.scales", p.scales, (E, N, groups), _FLOATS, at)
    _check(f"{name}.biases", p.biases, (E, N, groups), (p.scales.dtype,), at)
    return C.byref(p.struct())


_WORDS = (torch.int32, torch.uint32)


def _dims(name: str, t, dims: int):
    if not isinstance(t, torch.Tensor) or t.dim() != dims:
        raise ValueError(f"{name} must be a tensor of {dims} dimensions")
    return t.shape


def expert_matmul_backward(proj: StackedExperts, dy: torch.Tensor, offsets: torch.Tensor,
                           perm: Optional[torch.Tensor] = None, top_k: int = 1,
                           proj2: Optional[StackedExperts] = None, dy2: Optional[torch.Tensor] = None,
                           dx: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                           stream=None) -> torch.Tensor:
    """dx [M, K]: the gradient of the sorted rows of a quantised stack's product
    for the gradient dy of its output, plus proj2's for dy2 (a gate and an up
    projection). offsets [E + 1] int32 are the plan's. Without perm dy is
    [M, N], a row per sorted position; with perm [M] it holds tokens, and
    position p takes row perm[p] // top_k. dx [M, K] is a gradient that this one
    is added to (None: zeros); the sum goes to out, by default to dx itself. Rows
    behind the last expert's are not written (give out to have them defined)."""
    at, dt = dy.get_device(), _rows("dy", dy, 2).dtype
    p, K = _stack("proj", proj, at), proj.k
    rows = dy.shape[0]
    if perm is None:
        M = rows
        pp = None
    else:
        M = _dims("perm", perm, 1)[0]
        pp = _check("perm", perm, (M,), _I32, at)
        if top_k <= 0 or M <= 0:
            raise ValueError("top_k must be positive and perm have entries")
        rows = -(-M // top_k)
    yp = _check("dy", dy, (rows, proj.n), _FLOATS, at)
    if (proj2 is None) != (dy2 is None):
        raise ValueError("proj2 and dy2 come together")
    p2 = None if proj2 is None else _stack("proj2", proj2, at)
    y2 = None if proj2 is None else _check("dy2", dy2, (rows, proj2.n), (dt,), at)
    op = _check("offsets", offsets, (proj.n_experts + 1,), _I32, at)
    ip = _check("dx", dx, (M, K), (dt,), at)
    into = dx if out is None else out
    xp = _check("out", into, (M, K), (dt,), at)
    if into is not None and into.requires_grad and _grad_enabled():
        _refuse_grad("dx" if out is None else "out")
    st, ctx = _begin(at, stream)
    try:
        given = into is not None
        if not given:
            into = torch.empty(M, K, dtype=dt, device=dy.device)
            xp = into.data_ptr()
        check(_lib.load().moe_expert_matmul_backward(p, yp, p2, y2, moe_dtype(dt), pp, top_k, M, op, ip, xp, st))
        if given:
            _changed((into,))
    finally:
        if ctx is not None:
            ctx.leave()
    return into


class Checkpoint8(NamedTuple):
    """Rows kept in 8 bits as moe_activation_save keeps them: codes [parts, M, n]
    int8 and the exponent bytes of their blocks of 32, scales [parts, M, n // 32]
    uint8; two parts (gate, up), or one (up) with squared ReLU."""
    codes: torch.Tensor
    scales: torch.Tensor

    def _checked(self, at: int):
        parts, M, n = _dims("codes", self.codes, 3)
        return (_check("codes", self.codes, (parts, M, n), (torch.int8,), at),
                _check("scales", self.scales, (parts, M, n // 32), (torch.uint8,), at))

    def restore(self, dtype: torch.dtype, stream=None) -> torch.Tensor:
        """The values kept, [parts, M, n] of dtype."""
        if dtype not in _FLOATS:
            raise ValueError(f"dtype {dtype} is not a float32, float16 or bfloat16")
        at = _dims("codes", self.codes, 3) and self.codes.get_device()
        cp, sp = self._checked(at)
        st, ctx = _begin(at, stream)
        try:
            out = torch.empty(self.codes.shape, dtype=dtype, device=self.codes.device)
            check(_lib.load().moe_checkpoint_restore(cp, sp, self.codes.numel(), out.data_ptr(), moe_dtype(dtype), st))
        finally:
            if ctx is not None:
                ctx.leave()
        return out


def _row_count(offsets: Optional[torch.Tensor], at: int) -> Optional[int]:
    """The address of a plan's number of rows, its last offset."""
    if offsets is None:
        return None
    n = _dims("offsets", offsets, 1)[0]
    if n < 2:
        raise ValueError("offsets must have a plan's entries")
    return _check("offsets", offsets, (n,), _I32, at) + 4 * (n - 1)


def activation_save(gate: Optional[torch.Tensor], up: torch.Tensor, activation: int = _lib.MOE_ACT_SWIGLU,
                    alpha: float = 1.702, limit: float = 7.0, offsets: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, stream=None):
    """(h, kept): the gated activation h [M, n] of gate and up [M, n] (gate None
    with squared ReLU), and both in 8 bits (Checkpoint8). offsets (a plan's, None:
    all rows): rows behind the plan's last are neither read nor written. h goes
    to out (None: a new tensor), which may be gate or up."""
    M, n = _rows("up", up, 2).shape
    at, dts = up.get_device(), (up.dtype,)
    gated = activation != _lib.MOE_ACT_RELU2
    if gated == (gate is None):
        raise ValueError("gate is None with squared ReLU, and with it alone")
    gp = _check("gate", gate, (M, n), dts, at)
    up_ = _check("up", up, (M, n), dts, at)
    op = _check("out", out, (M, n), dts, at)
    np_ = _row_count(offsets, at)
    if _grad_enabled():
        for name, t in (("gate", gate), ("up", up), ("out", out)):
            if t is not None and t.requires_grad:
                _refuse_grad(name)
    st, ctx = _begin(at, stream)
    try:
        given = out is not None
        if not given:
            out = torch.empty(M, n, dtype=up.dtype, device=up.device)
            op = out.data_ptr()
        codes = torch.empty(1 + gated, M, n, dtype=torch.int8, device=up.device)
        scales = torch.empty(1 + gated, M, n // 32, dtype=torch.uint8, device=up.device)
        check(_lib.load().moe_activation_save(gp, up_, M, n, moe_dtype(up.dtype), activation, alpha, limit, np_, op,
                                              codes.data_ptr(), scales.data_ptr(), st))
        if given:
            _changed((out,))
    finally:
        if ctx is not None:
            ctx.leave()
    return out, Checkpoint8(codes, scales)


class ActivationGradients(NamedTuple):
    """d_gate (None with squared ReLU) and d_up [M, n], d_weight of topk_weight's
    shape float32, h [M, n]; d_weight and h None where not asked for."""
    d_gate: Optional[torch.Tensor]
    d_up: torch.Tensor
    d_weight: Optional[torch.Tensor]
    h: Optional[torch.Tensor]


def activation_backward(kept: Checkpoint8, dh: torch.Tensor, activation: int = _lib.MOE_ACT_SWIGLU,
                        alpha: float = 1.702, limit: float = 7.0, topk_weight: Optional[torch.Tensor] = None,
                        perm: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                        want_h: bool = False, want_weight: bool = True, stream=None) -> ActivationGradients:
    """Gradients of activation_save at the values kept, for dh [M, n], the
    gradient of h before the routing weights. topk_weight (M float32, any shape)
    are those weights in token order and perm [M] int32 the plan's (None: in
    order; it names no pick twice, and an entry past M none); with them come their
    gradient too (unless want_weight is False) and h itself if want_h. offsets: as
    in activation_save. The weights of picks without a row get a zero gradient."""
    M, n = _rows("dh", dh, 2).shape
    at, dt = dh.get_device(), dh.dtype
    gated = activation != _lib.MOE_ACT_RELU2
    if not isinstance(kept, Checkpoint8):
        raise ValueError("kept must be a Checkpoint8")
    if _dims("codes", kept.codes, 3) != (1 + gated, M, n):
        raise ValueError(f"codes must be {[1 + gated, M, n]}, got {list(kept.codes.shape)}")
    cp, sp = kept._checked(at)
    hp = _check("dh", dh, (M, n), _FLOATS, at)
    if topk_weight is not None and (not isinstance(topk_weight, torch.Tensor) or topk_weight.numel() != M):
        raise ValueError(f"topk_weight must be a tensor of {M} weights")
    wp = None if topk_weight is None else _check("topk_weight", topk_weight, topk_weight.shape, _F32, at)
    pp = _check("perm", perm, (M,), _I32, at)
    np_ = _row_count(offsets, at)
    st, ctx = _begin(at, stream)
    try:
        d_gate = torch.empty_like(dh) if gated else None
        d_up = torch.empty_like(dh)
        dw = None
        if topk_weight is not None and want_weight:
            # (in order every pick has a row; a plan may leave one out)
            dw = torch.empty_like(topk_weight) if perm is None and offsets is None else torch.zeros_like(topk_weight)
        h = torch.empty_like(dh) if want_h else None
        check(_lib.load().moe_activation_backward(
            cp, sp, hp, M, n, moe_dtype(dt), activation, alpha, limit, wp, pp, np_,
            None if d_gate is None else d_gate.data_ptr(), d_up.data_ptr(), None if dw is None else dw.data_ptr(),
            None if h is None else h.data_ptr(), st))
    finally:
        if ctx is not None:
            ctx.leave()
    return ActivationGradients(d_gate, d_up, dw, h)


def permute_backward(dX: torch.Tensor, inv_perm: torch.Tensor, dx: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """dx [T, hidden]: the gradients dX [T * k, hidden] of rows sorted by expert
    added up per token, position inv_perm[t, s] for rank s (inv_perm [T, k]
    int32; a position past T * k adds nothing). dx is a gradient that they are
    added to (None: zeros); the sum goes to out, by default to dx itself."""
    T, k = _dims("inv_perm", inv_perm, 2)
    H = _rows("dX", dX, 2).shape[1]
    at, dts = dX.get_device(), (dX.dtype,)
    gp = _check("dX", dX, (T * k, H), _FLOATS, at)
    ip = _check("inv_perm", inv_perm, (T, k), _I32, at)
    xp = _check("dx", dx, (T, H), dts, at)
    into = dx if out is None else out
    op = _check("out", into, (T, H), dts, at)
    if into is not None and into.requires_grad and _grad_enabled():
        _refuse_grad("dx" if out is None else "out")
    st, ctx = _begin(at, stream)
    try:
        given = into is not None
        if not given:
            into = torch.empty(T, H, dtype=dX.dtype, device=dX.device)
            op = into.data_ptr()
        check(_lib.load().moe_permute_backward(gp, ip, T, H, k, xp, op, moe_dtype(dX.dtype), st))
        if given:
            _changed((into,))
    finally:
        if ctx is not None:
            ctx.leave()
    return into


def add_rmsnorm_backward(residual: torch.Tensor, weight: torch.Tensor, d_normed: torch.Tensor, eps: float,
                         d_residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                         stream=None):
    """(d_in [T, hidden], d_weight [hidden] float32) of the residual add and RMS
    norm that moe_add_rmsnorm runs, at its sum residual [T, hidden]: d_in is the
    gradient of both rows added, for the normed rows' gradient d_normed and the
    sum's own d_residual (None: zeros). out (None: a new tensor) may be either."""
    T, H = _rows("residual", residual, 2).shape
    at, dts = residual.get_device(), (residual.dtype,)
    rp = _check("residual", residual, (T, H), _FLOATS, at)
    wp = _check("weight", weight, (H,), dts, at)
    np_ = _check("d_normed", d_normed, (T, H), dts, at)
    dp = _check("d_residual", d_residual, (T, H), dts, at)
    op = _check("out", out, (T, H), dts, at)
    if out is not None and out.requires_grad and _grad_enabled():
        _refuse_grad("out")
    st, ctx = _begin(at, stream)
    try:
        lib = _lib.load()
        given = out is not None
        if not given:
            out = torch.empty_like(residual)
            op = out.data_ptr()
        dw = torch.empty(H, dtype=torch.float32, device=residual.device)
        need = lib.moe_add_rmsnorm_backward_workspace_bytes(T, H)
        ws = torch.empty(need, dtype=torch.uint8, device=residual.device) if need else None
        check(lib.moe_add_rmsnorm_backward(rp, wp, np_, dp, eps, T, H, moe_dtype(residual.dtype), op, dw.data_ptr(),
                                           None if ws is None else ws.data_ptr(), need, st))
        if given:
            _changed((out,))
    finally:
        if ctx is not None:
            ctx.leave()
    return out, dw


class KeptExperts(NamedTuple):
    """What FrozenExperts.forward keeps for its backward: the plan, the routing
    weights (the tensor itself, not to change before), the activation's inputs in
    8 bits, and the experts' rows where the
    down projection has an output bias (its part of a routing weight's gradient
    is not in the activation)."""
    perm: torch.Tensor
    inv_perm: torch.Tensor
    offsets: torch.Tensor
    topk_weight: torch.Tensor
    kept: Checkpoint8
    Y: Optional[torch.Tensor]


@dataclass(frozen=True, eq=False)
class FrozenExperts:
    """The routed experts of a layer, quantised and frozen, with a gradient for
    what lies below them and for the routing weights: gate (None with squared
    ReLU), up [E, I, hidden] and down [E, hidden, I] as MoELayer takes them."""
    gate: Optional[StackedExperts]
    up: StackedExperts
    down: StackedExperts
    activation: int = _lib.MOE_ACT_SWIGLU
    alpha: float = 1.702
    limit: float = 7.0

    def __post_init__(self):
        E, I, H = self.up.n_experts, self.up.n, self.up.k
        if (self.gate is None) != (self.activation == _lib.MOE_ACT_RELU2):
            raise ValueError("gate is None with squared ReLU, and with it alone")
        if (self.down.n_experts, self.down.n, self.down.k) != (E, H, I):
            raise ValueError(f"down must be [{E}, {H}, {I}], got [{self.down.n_experts}, {self.down.n}, {self.down.k}]")
        if self.gate is not None and (self.gate.n_experts, self.gate.n, self.gate.k) != (E, I, H):
            raise ValueError("gate must have up's shape")

    def _product(self, lib, name, p, a, perm, k, M, offsets, st):
        at = a.get_device()
        desc = _stack(name, p, at)
        if p.out_bias is not None:
            _check(f"{name}.out_bias", p.out_bias, (p.n_experts, p.n), (a.dtype,), at)
        out = torch.empty(M, p.n, dtype=a.dtype, device=a.device)
        need = lib.moe_expert_matmul_workspace_bytes(desc, moe_dtype(a.dtype), M)
        ws = torch.empty(need, dtype=torch.uint8, device=a.device)
        check(lib.moe_expert_matmul(desc, a.data_ptr(), moe_dtype(a.dtype), None if perm is None else perm.data_ptr(),
                                    k, M, offsets.data_ptr(), out.data_ptr(), ws.data_ptr(), need, st))
        return out

    def forward(self, x: torch.Tensor, topk_idx: torch.Tensor, topk_weight: torch.Tensor, stream=None):
        """(y, kept) for x [T, hidden], its picks topk_idx [T, k] int32 (-1: none)
        and their weights [T, k] float32: y[t] = sum of weight * expert(x[t])."""
        T, k = _dims("topk_idx", topk_idx, 2)
        E, H = self.up.n_experts, self.up.k
        at, dev = x.get_device(), x.device
        _check("x", _rows("x", x, 2), (T, H), _FLOATS, at)
        _check("topk_idx", topk_idx, (T, k), _I32, at)
        _check("topk_weight", topk_weight, (T, k), _F32, at)
        if _grad_enabled():
            for name, t in (("x", x), ("topk_weight", topk_weight)):
                if t.requires_grad:
                    _refuse_grad(name)
        st, ctx = _begin(at, stream)
        try:
            lib, M = _lib.load(), T * k
            counts, offsets = (torch.empty(E + i, dtype=torch.int32, device=dev) for i in (0, 1))
            # a pick of no expert has no position, and leaves one at the end unwritten
            perm = torch.zeros(M, dtype=torch.int32, device=dev)
            inv = torch.full((T, k), -1, dtype=torch.int32, device=dev)
            need = lib.moe_dispatch_workspace_bytes(T, k, E)
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            check(lib.moe_dispatch_plan(topk_idx.data_ptr(), T, k, E, counts.data_ptr(), offsets.data_ptr(),
                                        perm.data_ptr(), inv.data_ptr(), ws.data_ptr(), need, st))
            u = self._product(lib, "up", self.up, x, perm, k, M, offsets, st)
            g = None if self.gate is None else self._product(lib, "gate", self.gate, x, perm, k, M, offsets, st)
            h, kept = activation_save(g, u, self.activation, self.alpha, self.limit, offsets=offsets, out=u)
            Y = self._product(lib, "down", self.down, h, None, 1, M, offsets, st)
            y = torch.empty_like(x)
            check(lib.moe_unpermute(Y.data_ptr(), inv.data_ptr(), topk_weight.data_ptr(), T, H, k, y.data_ptr(),
                                    moe_dtype(x.dtype), st))
        finally:
            if ctx is not None:
                ctx.leave()
        return y, KeptExperts(perm, inv, offsets, topk_weight, kept, None if self.down.out_bias is None else Y)

    def backward(self, d_out: torch.Tensor, kept: KeptExperts, dx: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, stream=None):
        """(dx [T, hidden], d_weight [T, k] float32) of forward for d_out
        [T, hidden]. dx is a gradient that x's is added to (None: zeros), from the
        router or a shared expert; the sum goes to out, by default to dx itself.
        Gate and up of two formats (bits, group size, scales' type) take a launch
        each, and the sorted rows' gradient is rounded to their type between the two."""
        T, k = kept.inv_perm.shape
        H, at = self.up.k, d_out.get_device()
        gp = _check("d_out", _rows("d_out", d_out, 2), (T, H), _FLOATS if kept.Y is None else (kept.Y.dtype,), at)
        st, ctx = _begin(at, stream)
        try:
            dh = expert_matmul_backward(self.down, d_out, kept.offsets, perm=kept.perm, top_k=k)
            d = activation_backward(kept.kept, dh, self.activation, self.alpha, self.limit, kept.topk_weight,
                                    kept.perm, kept.offsets, want_weight=kept.Y is None)
            dw = d.d_weight
            if kept.Y is not None:
                dw = torch.empty_like(kept.topk_weight)
                check(_lib.load().moe_unpermute_backward(gp, kept.Y.data_ptr(), kept.inv_perm.data_ptr(),
                                                         kept.topk_weight.data_ptr(), T, H, k, None, dw.data_ptr(),
                                                         moe_dtype(d_out.dtype), st))
            if self.gate is None:
                dX = expert_matmul_backward(self.up, d.d_up, kept.offsets)
            elif (self.gate.bits, self.gate.group_size, self.gate.scales.dtype) == (
                    self.up.bits, self.up.group_size, self.up.scales.dtype):
                dX = expert_matmul_backward(self.gate, d.d_gate, kept.offsets, proj2=self.up, dy2=d.d_up)
            else:  # projections of two formats: one after the other
                dX = expert_matmul_backward(self.gate, d.d_gate, kept.offsets)
                dX = expert_matmul_backward(self.up, d.d_up, kept.offsets, dx=dX)
            return permute_backward(dX, kept.inv_perm, dx=dx, out=out), dw
        finally:
            if ctx is not None:
                ctx.leave()
