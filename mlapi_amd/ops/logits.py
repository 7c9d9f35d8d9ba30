"""Row operators over class logits: a teacher's top logits, distillation from them, sampling.

Each takes logits ``Z`` [B, K] (f32, bf16 or f16; B rows of one sample's K class scores, 1 <= K <= 2^20) as
:func:`mlapi_amd.ops.linear.gemm_logits` or any other model gives them, with contiguous columns and any row
stride, and launches on the current stream of Z's device. They allocate their results and workspace from
torch's allocator and do not synchronise, so they can be captured into a HIP graph. GPU tensors only;
plain oracles are in :mod:`mlapi_amd.ops.reference`. Gradients are results like any other: nothing here is recorded by
autograd (``Z.backward(dZ)`` hands them on to the model that gave Z).

The order of a row's classes is everywhere: larger logit first, then lower class. A class whose logit is
-inf is masked; so is NaN in :func:`top_logits` and :func:`sample_logits`, while in the distillation loss a
NaN or +inf makes its row NaN.

    values, idx = top_logits(teacher_Z, 16)                               # the teacher's list
    loss, dZ = distill_loss_grad(student_Z, idx, values, temperature=2.0)  # the student's step
    label, prob = sample_logits(student_Z, u, temperature=0.8, top_p=0.95)  # its answer, u in [0, 1)
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from mlapi_amd._native import C

_DT = {torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}
MAX_CLASSES, MAX_TOP = 1 << 20, 1024  # the launchers' LOGIT_MAX_CLASSES, LOGIT_MAX_TOP

# The current stream of a device as a number: 0.06 us where a torch.cuda.Stream takes 1.8, of the 7 us that a
# call on a small batch spends on the host.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


class _On:
    """Launch on a tensor's device, whichever is current: ``with _On(Z) as stream``."""

    __slots__ = ("index", "before")

    def __init__(self, t: torch.Tensor):
        self.index = t.device.index

    def __enter__(self) -> int:
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc) -> None:
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _logits(name: str, Z: torch.Tensor) -> Tuple[int, int, int]:
    """(B, K, row stride) of a logit matrix that the kernels can read."""
    if not isinstance(Z, torch.Tensor) or not Z.is_cuda:
        raise ValueError(f"{name}: inputs must be GPU tensors (no CPU fallback)")
    if Z.dtype not in _DT:
        raise TypeError(f"{name}: logits must be f32, bf16 or f16 (got {Z.dtype})")
    if Z.dim() != 2 or Z.shape[1] < 1:
        raise ValueError(f"{name}: logits must be [B, K] with K >= 1")
    B, K = Z.shape
    if K > MAX_CLASSES:
        raise ValueError(f"{name}: at most {MAX_CLASSES} classes (got {K})")
    if K > 1 and Z.stride(1) != 1:
        raise ValueError(f"{name}: the classes of a row must be contiguous")
    ld = Z.stride(0) if B > 1 else K
    if ld < K:
        raise ValueError(f"{name}: rows overlap (row stride {ld} below K = {K})")
    return B, K, ld


def _vector(name: str, what: str, v: torch.Tensor, Z: torch.Tensor, dtype: torch.dtype) -> int:
    if not isinstance(v, torch.Tensor) or v.device != Z.device:
        raise ValueError(f"{name}: {what} must be a tensor on {Z.device}")
    if v.dtype != dtype:
        raise TypeError(f"{name}: {what} must be {dtype} (got {v.dtype})")
    if v.shape != (Z.shape[0],) or not v.is_contiguous():
        raise ValueError(f"{name}: {what} must be a contiguous [B] tensor")
    return v.data_ptr()


def _span(t: torch.Tensor) -> Tuple[int, int]:
    n = 1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride())) if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _apart(name: str, outs, ins) -> None:
    """Results given by the caller must not lie on inputs (which other rows' blocks may still read)."""
    ins = [_span(v) for v in ins if isinstance(v, torch.Tensor)]
    outs = [_span(v) for v in outs]
    for i, (a, b) in enumerate(outs):
        if any(a < q and p < b for p, q in ins + outs[:i]):
            raise ValueError(f"{name}: out overlaps an input or another result")


def _workspace(nbytes: int, device) -> Tuple[Optional[torch.Tensor], int]:
    """(the tensor that keeps it alive, its address)"""
    if nbytes == 0:
        return None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr()


# -------------------------------------------------------------------------------------------- top
def top_logits(Z: torch.Tensor, k: int, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The k first classes of every row (1 <= k <= 1024): (values [B, k] in Z's type, idx int32 [B, k]),
    in order. Past a row's last unmasked class (and past K) value is -inf and idx -1. ``out=(values, idx)``
    writes into preallocated contiguous tensors."""
    B, K, ld = _logits("top_logits", Z)
    k = int(k)
    if not 1 <= k <= MAX_TOP:
        raise ValueError(f"top_logits: k must be in [1, {MAX_TOP}] (got {k})")
    if out is None:
        values = torch.empty((B, k), dtype=Z.dtype, device=Z.device)
        idx = torch.empty((B, k), dtype=torch.int32, device=Z.device)
    else:
        values, idx = out
        for t, dt in ((values, Z.dtype), (idx, torch.int32)):
            if t.dtype != dt or t.shape != (B, k) or not t.is_contiguous() or t.device != Z.device:
                raise ValueError("top_logits: out must be contiguous (Z's type [B, k], int32 [B, k]) on Z's device")
        _apart("top_logits", out, (Z,))
    dt = _DT[Z.dtype]
    c = C()
    with _On(Z) as stream:
        n = c.top_logits_workspace(dt, B, K, k)
        ws, at = _workspace(n, Z.device)
        c.top_logits(dt, Z.data_ptr(), ld, B, K, k, values.data_ptr(), idx.data_ptr(), at, n, stream)
    return values, idx


# ------------------------------------------------------------------------------------ distillation
def _distill(name: str, Z, idx, t, temperature, alpha, y, *, g=None, stats_in=None, loss=False, stats=False, pred=None,
             dz=None, out=None):
    """One call: (loss, statistics) where asked for; the gradient goes to ``out``, or with ``dz`` to a new tensor."""
    B, K, ld = _logits(name, Z)
    dev = Z.device
    for what, v in (("idx", idx), ("t", t)):
        if not isinstance(v, torch.Tensor) or v.device != dev:
            raise ValueError(f"{name}: {what} must be a tensor on {dev}")
        if v.dim() != 2 or v.shape[0] != B or v.shape[1] < 1 or (v.shape[1] > 1 and v.stride(1) != 1):
            raise ValueError(f"{name}: {what} must be [B, k], k >= 1, with contiguous rows")
    if idx.dtype != torch.int32 or t.dtype not in _DT:
        raise TypeError(f"{name}: idx must be int32 and t f32, bf16 or f16")
    k = idx.shape[1]
    if t.shape[1] != k or k > MAX_TOP:
        raise ValueError(f"{name}: idx and t must both be [B, k], k <= {MAX_TOP}")
    temperature, alpha = float(temperature), float(alpha)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"{name}: temperature must be in [1e-6, 1e6] (got {temperature})")
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"{name}: alpha must be in [0, 1] (got {alpha})")
    if alpha != 1.0 and y is None:
        raise ValueError(f"{name}: alpha below 1 mixes in hard labels and needs y")
    yp = 0 if y is None else _vector(name, "y", y, Z, torch.int32)
    gp = 0 if g is None else _vector(name, "g", g, Z, torch.float32)
    pp = 0
    if pred is not None:
        pp = _vector(name, "pred", pred, Z, torch.int32)
        _apart(name, (pred,), (Z, idx, t, y, g))
    dt = ddt = _DT[Z.dtype]
    ldd = dp = 0
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.device != dev or out.shape != Z.shape or out.dtype not in (
                Z.dtype, *((torch.bfloat16,) if Z.dtype == torch.float32 else ())):
            raise ValueError(f"{name}: out must be [B, K] on Z's device in Z's type (or bf16 for f32 logits)")
        ldd = out.stride(0) if B > 1 else K
        if (K > 1 and out.stride(1) != 1) or ldd < K:
            raise ValueError(f"{name}: out must have contiguous, separate rows")
        ddt, dp = _DT[out.dtype], out.data_ptr()
        same = dp == Z.data_ptr() and ld == ldd and Z.dtype == out.dtype
        _apart(name, (out,), (None if same else Z, idx, t, y, g, stats_in, pred))
    elif dz:
        out = torch.empty((B, K), dtype=Z.dtype, device=dev)
        ldd, dp = K, out.data_ptr()
    loss = torch.empty(B, dtype=torch.float32, device=dev) if loss else None
    stats = torch.empty((B, 4), dtype=torch.float32, device=dev) if stats else None
    c = C()
    with _On(Z) as stream:
        n = c.distill_workspace(dt, B, K, temperature, stats_in is not None)
        ws, at = _workspace(n, dev)
        c.distill(dt, _DT[t.dtype], ddt, Z.data_ptr(), ld, B, K, idx.data_ptr(), idx.stride(0) if B > 1 else k,
                  t.data_ptr(), t.stride(0) if B > 1 else k, k, temperature, alpha, yp, gp,
                  0 if stats_in is None else stats_in.data_ptr(), 0 if loss is None else loss.data_ptr(),
                  0 if stats is None else stats.data_ptr(), pp, dp, ldd, at, n, stream)
    return loss, stats, out


def distill_loss(Z: torch.Tensor, idx: torch.Tensor, t: torch.Tensor, *, temperature: float = 1.0, alpha: float = 1.0,
                 y: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Every row's distillation loss, and the row statistics :func:`distill_grad` takes (opaque, 16 bytes a row).

    The teacher's list is ``idx`` int32 [B, k] (classes) and ``t`` [B, k] (logits, f32, bf16 or f16), k <= 1024, as
    :func:`top_logits` writes it; an entry with a negative class or a logit of -inf is absent, a class may be
    listed twice. With q = softmax(t / T) over the row's entries and p = softmax(Z / T) over all K classes

        loss = alpha T^2 sum_j q_j (ln q_j - ln p[idx_j])  -  (1 - alpha) ln softmax(Z)[y]        (f32 [B])

    T in [1e-6, 1e6]; above 16, where T^2 would count what 32-bit sums are off, a row whose list holds nearly all of p is
    evaluated in 64 bits.
    A row without entries has no first part, a row with y < 0 no second, a row whose logits are all -inf
    neither. A listed class that the student masks makes the loss +inf. A class >= K in idx or y makes its
    row's loss and gradient NaN."""
    loss, stats, _ = _distill("distill_loss", Z, idx, t, temperature, alpha, y, loss=True, stats=True)
    return loss, stats


def distill_grad(Z: torch.Tensor, idx: torch.Tensor, t: torch.Tensor, stats: torch.Tensor, *,
                 g: Optional[torch.Tensor] = None, temperature: float = 1.0, alpha: float = 1.0,
                 y: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """d(sum_r g_r loss_r)/dZ, [B, K] in Z's type, from the statistics :func:`distill_loss` gave for the same
    arguments. ``g`` f32 [B] weights the rows (None: 1). ``out``: where to write it - any row stride, bf16 for f32
    logits, or Z itself. The teacher's logits get no gradient."""
    if not isinstance(Z, torch.Tensor) or not isinstance(stats, torch.Tensor) or stats.device != Z.device or \
            stats.dtype != torch.float32 or stats.shape != (Z.shape[0], 4) or not stats.is_contiguous():
        raise ValueError("distill_grad: stats must be the [B, 4] statistics of distill_loss")
    return _distill("distill_grad", Z, idx, t, temperature, alpha, y, g=g, stats_in=stats, dz=True, out=out)[2]


def distill_loss_grad(Z: torch.Tensor, idx: torch.Tensor, t: torch.Tensor, *, g: Optional[torch.Tensor] = None,
                      temperature: float = 1.0, alpha: float = 1.0, y: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None, pred: Optional[torch.Tensor] = None
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`distill_loss` and :func:`distill_grad` in one pass over the logits: (loss f32 [B], dZ). ``g`` weights the
    gradient alone. ``pred`` int32 [B], if given, receives every row's first maximum."""
    loss, _, dz = _distill("distill_loss_grad", Z, idx, t, temperature, alpha, y, g=g, loss=True, pred=pred, dz=True,
                           out=out)
    return loss, dz


# ---------------------------------------------------------------------------------------- sampling
Setting = Union[float, int, torch.Tensor]


def _setting(name: str, v: Setting, Z: torch.Tensor, dtype: torch.dtype, number, most: float):
    """(address of a per-row setting or 0, the number for all rows)"""
    if isinstance(v, torch.Tensor):
        return _vector("sample_logits", name, v, Z, dtype), 0
    n = number(v)
    if not 0 <= n <= most:
        raise ValueError(f"sample_logits: {name} must be in [0, {most}] (got {v})")
    return 0, n


def sample_logits(Z: torch.Tensor, u: torch.Tensor, *, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One class drawn from every row with the given random numbers ``u`` f32 [B]: (idx int32 [B], prob f32 [B]).

    With w = exp((Z - max) / temperature) the filters keep, one after another: the ``top_k`` first classes of the
    order (<= 0: all); of those, the classes whose preceding mass in the order is below ``top_p`` times their
    mass, the first always (>= 1: all); of those, the ones with w >= ``min_p`` (<= 0: all; the maximum has w = 1).
    The draw is the first class, counting up, whose cumulative kept mass exceeds u times the kept mass; ``prob`` is
    its share of that mass. u is taken into [0, 1), a NaN as 0. A temperature of 0 takes the first maximum; one of
    infinity or NaN, in a tensor, counts as the largest finite number.
    A row whose classes are all masked gives (-1, 0).

    Each setting is one number for all rows, or a [B] tensor (f32; top_k int32) with one for each. Numbers are
    rounded to 32 bits; masses are summed exactly (fixed point, 2^-42 of the largest weight), so the same inputs
    always draw the same class."""
    B, K, ld = _logits("sample_logits", Z)
    up = _vector("sample_logits", "u", u, Z, torch.float32)
    Tp, T = _setting("temperature", temperature, Z, torch.float32, float, torch.finfo(torch.float32).max)
    kp, k = _setting("top_k", top_k, Z, torch.int32, int, float("inf"))
    pp, p = _setting("top_p", top_p, Z, torch.float32, float, 1.0)
    mp, least = _setting("min_p", min_p, Z, torch.float32, float, 1.0)
    k = min(k, K)
    if out is None:
        idx = torch.empty(B, dtype=torch.int32, device=Z.device)
        prob = torch.empty(B, dtype=torch.float32, device=Z.device)
    else:
        idx, prob = out
        _vector("sample_logits", "out idx", idx, Z, torch.int32)
        _vector("sample_logits", "out prob", prob, Z, torch.float32)
        _apart("sample_logits", out, (Z, u, temperature, top_k, top_p, min_p))
    dt = _DT[Z.dtype]
    c = C()
    with _On(Z) as stream:
        n = c.sample_workspace(dt, B, K, kp != 0, k)
        ws, at = _workspace(n, Z.device)
        c.sample_logits(dt, Z.data_ptr(), ld, B, K, up, Tp, T, kp, k, pp, p, mp, least, idx.data_ptr(),
                        prob.data_ptr(), at, n, stream)
    return idx, prob
