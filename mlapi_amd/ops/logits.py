"""Row operators over class logits: a teacher's top logits, distillation from them, sampling.

Each takes logits ``Z`` [B, K] (f32, bf16 or f16; B rows of one sample's K class scores, 1 <= K <= 2^20) as
:func:`mlapi_amd.ops.linear.gemm_logits` or any other model gives them, with contiguous columns and any row
stride, and launches on the current stream of Z's device. They allocate their results and workspace from
torch's allocator and do not synchronise, so they can be captured into a HIP graph. GPU tensors only;
plain oracles are in :mod:`mlapi_amd.ops.reference`.

The order of a row's classes is everywhere: larger logit first, then lower class. A class whose logit is
-inf is masked; so is NaN in :func:`top_logits` and :func:`sample_logits`, while in the distillation loss a
NaN makes its row NaN.

    values, idx = top_logits(teacher_Z, 16)                               # the teacher's list
    loss, dZ = distill_loss_grad(student_Z, idx, values, temperature=2.0)  # the student's step
    label, prob = sample_logits(student_Z, u, temperature=0.8, top_p=0.95)  # its answer, u in [0, 1)
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from mlapi_amd._native import C

_DT = {torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _logits(name: str, Z: torch.Tensor) -> Tuple[int, int, int]:
    """(B, K, row stride) of a logit matrix that the kernels can read."""
    if not isinstance(Z, torch.Tensor) or not Z.is_cuda:
        raise ValueError(f"{name}: inputs must be GPU tensors (no CPU fallback)")
    if Z.dtype not in _DT:
        raise TypeError(f"{name}: logits must be f32, bf16 or f16 (got {Z.dtype})")
    if Z.dim() != 2 or Z.shape[1] < 1:
        raise ValueError(f"{name}: logits must be [B, K] with K >= 1")
    B, K = Z.shape
    if K > C().LOGIT_MAX_CLASSES:
        raise ValueError(f"{name}: at most {C().LOGIT_MAX_CLASSES} classes (got {K})")
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


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


# -------------------------------------------------------------------------------------------- top
def top_logits(Z: torch.Tensor, k: int, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The k first classes of every row (1 <= k <= 1024): (values [B, k] in Z's type, idx int32 [B, k]),
    in order. Past a row's last unmasked class (and past K) value is -inf and idx -1. ``out=(values, idx)``
    writes into preallocated contiguous tensors."""
    B, K, ld = _logits("top_logits", Z)
    k = int(k)
    if not 1 <= k <= C().LOGIT_MAX_TOP:
        raise ValueError(f"top_logits: k must be in [1, {C().LOGIT_MAX_TOP}] (got {k})")
    if out is None:
        out = (torch.empty(B, k, dtype=Z.dtype, device=Z.device), torch.empty(B, k, dtype=torch.int32, device=Z.device))
    values, idx = out
    for t, dt in ((values, Z.dtype), (idx, torch.int32)):
        if t.dtype != dt or t.shape != (B, k) or not t.is_contiguous() or t.device != Z.device:
            raise ValueError("top_logits: out must be contiguous (Z's type [B, k], int32 [B, k]) on Z's device")
    dt = _DT[Z.dtype]
    with torch.cuda.device(Z.device):
        ws = _workspace(C().top_logits_workspace(dt, B, K, k), Z.device)
        C().top_logits(dt, Z.data_ptr(), ld, B, K, k, values.data_ptr(), idx.data_ptr(), ws.data_ptr(), ws.numel(),
                       _stream(Z.device))
    return values, idx


# ------------------------------------------------------------------------------------ distillation
def _distill(name: str, Z, idx, t, temperature, alpha, y, *, g=None, stats_in=None, loss=None, stats_out=None,
             pred=None, dz=None) -> None:
    B, K, ld = _logits(name, Z)
    for what, v in (("idx", idx), ("t", t)):
        if not isinstance(v, torch.Tensor) or v.device != Z.device:
            raise ValueError(f"{name}: {what} must be a tensor on {Z.device}")
        if v.dim() != 2 or v.shape[0] != B or v.shape[1] < 1 or (v.shape[1] > 1 and v.stride(1) != 1):
            raise ValueError(f"{name}: {what} must be [B, k], k >= 1, with contiguous rows")
    if idx.dtype != torch.int32 or t.dtype not in _DT:
        raise TypeError(f"{name}: idx must be int32 and t f32, bf16 or f16")
    k = idx.shape[1]
    if t.shape[1] != k or k > C().LOGIT_MAX_TOP:
        raise ValueError(f"{name}: idx and t must both be [B, k], k <= {C().LOGIT_MAX_TOP}")
    temperature, alpha = float(temperature), float(alpha)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"{name}: temperature must be in [1e-6, 1e6] (got {temperature})")
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"{name}: alpha must be in [0, 1] (got {alpha})")
    if alpha != 1.0 and y is None:
        raise ValueError(f"{name}: alpha below 1 mixes in hard labels and needs y")
    yp = 0 if y is None else _vector(name, "y", y, Z, torch.int32)
    gp = 0 if g is None else _vector(name, "g", g, Z, torch.float32)
    ldd, ddt = 0, _DT[Z.dtype]
    if dz is not None:
        if not isinstance(dz, torch.Tensor) or dz.device != Z.device or dz.shape != Z.shape or dz.dtype not in (
                Z.dtype, *((torch.bfloat16,) if Z.dtype == torch.float32 else ())):
            raise ValueError(f"{name}: out must be [B, K] on Z's device in Z's type (or bf16 for f32 logits)")
        ldd = dz.stride(0) if B > 1 else K
        if (K > 1 and dz.stride(1) != 1) or ldd < K:
            raise ValueError(f"{name}: out must have contiguous, separate rows")
        ddt = _DT[dz.dtype]
        (a, b), (c, d) = _span(Z), _span(dz)
        if a < d and c < b and not (a == c and ld == ldd and Z.dtype == dz.dtype):
            raise ValueError(f"{name}: out overlaps the logits without being the logits")
    ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    dt = _DT[Z.dtype]
    with torch.cuda.device(Z.device):
        ws = _workspace(0 if stats_in is not None else C().distill_workspace(dt, B, K), Z.device)
        C().distill(dt, _DT[t.dtype], ddt, Z.data_ptr(), ld, B, K, idx.data_ptr(), idx.stride(0) if B > 1 else k,
                    t.data_ptr(), t.stride(0) if B > 1 else k, k, temperature, alpha, yp, gp, ptr(stats_in), ptr(loss),
                    ptr(stats_out), ptr(pred), ptr(dz), ldd, ws.data_ptr(), ws.numel(), _stream(Z.device))


def distill_loss(Z: torch.Tensor, idx: torch.Tensor, t: torch.Tensor, *, temperature: float = 1.0, alpha: float = 1.0,
                 y: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Every row's distillation loss, and the row statistics :func:`distill_grad` takes (opaque, 16 bytes a row).

    The teacher's list is ``idx`` int32 [B, k] (classes) and ``t`` [B, k] (logits, f32, bf16 or f16), k <= 1024, as
    :func:`top_logits` writes it; an entry with a negative class or a logit of -inf is absent, a class may be
    listed twice. With q = softmax(t / T) over the row's entries and p = softmax(Z / T) over all K classes

        loss = alpha T^2 sum_j q_j (ln q_j - ln p[idx_j])  -  (1 - alpha) ln softmax(Z)[y]        (f32 [B])

    A row without entries has no first part, a row with y < 0 no second, a row whose logits are all -inf
    neither. A listed class that the student masks makes the loss +inf. A class >= K in idx or y makes its
    row's loss and gradient NaN."""
    B = _logits("distill_loss", Z)[0]
    loss = torch.empty(B, dtype=torch.float32, device=Z.device)
    stats = torch.empty(B, 4, dtype=torch.float32, device=Z.device)
    _distill("distill_loss", Z, idx, t, temperature, alpha, y, loss=loss, stats_out=stats)
    return loss, stats


def distill_grad(Z: torch.Tensor, idx: torch.Tensor, t: torch.Tensor, stats: torch.Tensor, *,
                 g: Optional[torch.Tensor] = None, temperature: float = 1.0, alpha: float = 1.0,
                 y: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """d(sum_r g_r loss_r)/dZ, [B, K] in Z's type, from the statistics :func:`distill_loss` gave for the same
    arguments. ``g`` f32 [B] weights the rows (None: 1). ``out``: where to write it - any row stride, bf16 for f32
    logits, or Z itself. The teacher's logits get no gradient."""
    B = _logits("distill_grad", Z)[0]
    if not isinstance(stats, torch.Tensor) or stats.device != Z.device or stats.dtype != torch.float32 or \
            stats.shape != (B, 4) or not stats.is_contiguous():
        raise ValueError("distill_grad: stats must be the [B, 4] statistics of distill_loss")
    dz = torch.empty(Z.shape, dtype=Z.dtype, device=Z.device) if out is None else out
    _distill("distill_grad", Z, idx, t, temperature, alpha, y, g=g, stats_in=stats, dz=dz)
    return dz


def distill_loss_grad(Z: torch.Tensor, idx: torch.Tensor, t: torch.Tensor, *, g: Optional[torch.Tensor] = None,
                      temperature: float = 1.0, alpha: float = 1.0, y: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None, pred: Optional[torch.Tensor] = None
                      ) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`distill_loss` and :func:`distill_grad` in one pass over the logits: (loss f32 [B], dZ). ``g`` weights the
    gradient alone. ``pred`` int32 [B], if given, receives every row's first maximum."""
    B = _logits("distill_loss_grad", Z)[0]
    loss = torch.empty(B, dtype=torch.float32, device=Z.device)
    dz = torch.empty(Z.shape, dtype=Z.dtype, device=Z.device) if out is None else out
    if pred is not None:
        _vector("distill_loss_grad", "pred", pred, Z, torch.int32)
    _distill("distill_loss_grad", Z, idx, t, temperature, alpha, y, g=g, loss=loss, pred=pred, dz=dz)
    return loss, dz


# ---------------------------------------------------------------------------------------- sampling
Setting = Union[float, int, torch.Tensor]


def sample_logits(Z: torch.Tensor, u: torch.Tensor, *, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One class drawn from every row with the given random numbers ``u`` f32 [B]: (idx int32 [B], prob f32 [B]).

    With w = exp((Z - max) / temperature) the filters keep, one after another: the ``top_k`` first classes of the
    order (<= 0: all); of those, the classes whose preceding mass in the order is below ``top_p`` times their
    mass, the first always (>= 1: all); of those, the ones with w >= ``min_p`` (<= 0: all; the maximum has w = 1).
    The draw is the first class, counting up, whose cumulative kept mass exceeds u times the kept mass; ``prob`` is
    its share of that mass. u is taken into [0, 1), a NaN as 0. A temperature of 0 takes the first maximum.
    A row whose classes are all masked gives (-1, 0).

    Each setting is one number for all rows, or a [B] tensor (f32; top_k int32) with one for each. Numbers are
    rounded to 32 bits; masses are summed exactly (fixed point, 2^-42 of the largest weight), so the same inputs
    always draw the same class."""
    B, K, ld = _logits("sample_logits", Z)
    up = _vector("sample_logits", "u", u, Z, torch.float32)
    ptrs, nums = {}, {}
    for name, v, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if isinstance(v, torch.Tensor):
            ptrs[name], nums[name] = _vector("sample_logits", name, v, Z, dtype), 0
        else:
            ptrs[name], nums[name] = 0, int(v) if name == "top_k" else float(v)
    if not nums["temperature"] >= 0.0:
        raise ValueError(f"sample_logits: temperature must be >= 0 (got {temperature})")
    if nums["top_k"] < 0:
        raise ValueError(f"sample_logits: top_k must be >= 0 (got {top_k})")
    if not 0.0 <= nums["top_p"] <= 1.0 or not 0.0 <= nums["min_p"] <= 1.0:
        raise ValueError(f"sample_logits: top_p and min_p must be in [0, 1] (got {top_p}, {min_p})")
    nums["top_k"] = min(nums["top_k"], K)
    if out is None:
        out = (torch.empty(B, dtype=torch.int32, device=Z.device), torch.empty(B, dtype=torch.float32, device=Z.device))
    idx, prob = out
    _vector("sample_logits", "out idx", idx, Z, torch.int32)
    _vector("sample_logits", "out prob", prob, Z, torch.float32)
    dt = _DT[Z.dtype]
    with torch.cuda.device(Z.device):
        ws = _workspace(C().sample_workspace(dt, B, K, ptrs["top_k"] != 0, nums["top_k"]), Z.device)
        C().sample_logits(dt, Z.data_ptr(), ld, B, K, up, ptrs["temperature"], nums["temperature"], ptrs["top_k"],
                          nums["top_k"], ptrs["top_p"], nums["top_p"], ptrs["min_p"], nums["min_p"], idx.data_ptr(),
                          prob.data_ptr(), ws.data_ptr(), ws.numel(), _stream(Z.device))
    return idx, prob
