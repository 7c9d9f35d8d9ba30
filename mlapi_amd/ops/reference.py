"""Plain-PyTorch fp32/fp64 reference implementations of every HIP kernel (test oracles)."""
from __future__ import annotations

import torch

from mlapi_amd.models.linear import Kind


def predict_ref(X: torch.Tensor, W: torch.Tensor, b: torch.Tensor, kind: int, dtype=torch.float64):
    X, W, b = X.to(dtype), W.to(dtype), b.to(dtype)
    z = X @ W.T + b
    if kind in (Kind.BINARY, Kind.BINARY_SOFTMAX):
        z = z[:, 0]
        a = z.abs() * (2.0 if kind == Kind.BINARY_SOFTMAX else 1.0)
        return (z > 0).to(torch.int32), torch.sigmoid(a)
    idx = torch.argmax(z, dim=1).to(torch.int32)  # first max (torch.argmax is first-occurrence)
    if kind == Kind.MULTINOMIAL:
        return idx, torch.softmax(z, dim=1).max(dim=1).values
    s = torch.sigmoid(z)
    return idx, (s / s.sum(dim=1, keepdim=True)).max(dim=1).values


def logits_ref(X, W, b, dtype=torch.float32):
    return X.to(dtype) @ W.to(dtype).T + b.to(dtype)


def train_binary_ref(X, y, w, b):
    X = X.to(torch.float64)
    z = X @ w.to(torch.float64) + b.to(torch.float64)
    y = y.to(torch.float64)
    g = torch.sigmoid(z) - y
    loss = (torch.clamp(z, min=0) - z * y + torch.log1p(torch.exp(-z.abs()))).sum()
    correct = ((z > 0) == (y > 0.5)).sum()
    return torch.cat([X.T @ g, g.sum().reshape(1), loss.reshape(1), correct.to(torch.float64).reshape(1)])


def train_small_ref(X, y, W, b, kind: int):
    X, W, b = X.to(torch.float64), W.to(torch.float64), b.to(torch.float64)
    y = y.long()
    z = X @ W.T + b
    K = W.shape[0]
    if kind in (Kind.BINARY, Kind.BINARY_SOFTMAX):
        sc = 2.0 if kind == Kind.BINARY_SOFTMAX else 1.0
        zz = sc * z[:, 0]
        yy = y.to(torch.float64)
        g = (sc * (torch.sigmoid(zz) - yy))[:, None]
        loss = (torch.clamp(zz, min=0) - zz * yy + torch.log1p(torch.exp(-zz.abs()))).sum()
        correct = ((z[:, 0] > 0) == (y == 1)).sum()
    elif kind == Kind.MULTINOMIAL:
        p = torch.softmax(z, dim=1)
        Y = torch.nn.functional.one_hot(y, K).to(torch.float64)
        g = p - Y
        loss = (torch.logsumexp(z, dim=1) - z.gather(1, y[:, None])[:, 0]).sum()
        correct = (torch.argmax(z, dim=1) == y).sum()
    else:
        Y = torch.nn.functional.one_hot(y, K).to(torch.float64)
        g = torch.sigmoid(z) - Y
        loss = (torch.clamp(z, min=0) - z * Y + torch.log1p(torch.exp(-z.abs()))).sum()
        correct = (torch.argmax(z, dim=1) == y).sum()
    return torch.cat([(g.T @ X).reshape(-1), g.sum(0), loss.reshape(1), correct.to(torch.float64).reshape(1)])


def softmax_train_ref(X_aug, y, W_aug, kind: int, dtype=torch.float32):
    """Oracle of ops.linear.softmax_train_grad: (G [B, K], dW_aug [K, F_aug], loss_sum, n_correct).

    Also the CPU path of the multiclass SGD trainer (dtype float32)."""
    X, W = X_aug.to(dtype), W_aug.to(dtype)
    y = y.long()
    z = X @ W.T
    K = W.shape[0]
    Y = torch.nn.functional.one_hot(y, K).to(dtype)
    if kind == Kind.MULTINOMIAL:
        G = torch.softmax(z, dim=1) - Y
        loss = (torch.logsumexp(z, dim=1) - z.gather(1, y[:, None])[:, 0]).sum()
    else:
        G = torch.sigmoid(z) - Y
        loss = (torch.clamp(z, min=0) - z * Y + torch.log1p(torch.exp(-z.abs()))).sum()
    correct = (torch.argmax(z, dim=1) == y).sum().to(dtype)
    return G, G.T @ X, loss, correct


# --------------------------------------------------------------- row operators over class logits
def _class_order(Z):
    """Classes of every row in order (larger logit first, then lower class; NaN counts as -inf), float64 logits."""
    z = Z.to(torch.float64)
    z = torch.where(z.isnan(), torch.full_like(z, -float("inf")), z)
    return z, torch.sort(z, dim=1, descending=True, stable=True).indices


def top_logits_ref(Z, k: int):
    """Oracle of ops.logits.top_logits (any device)."""
    z, order = _class_order(Z)
    B, K = z.shape
    n = min(k, K)
    idx = torch.full((B, k), -1, dtype=torch.int32, device=Z.device)
    val = torch.full((B, k), -float("inf"), dtype=Z.dtype, device=Z.device)
    top = order[:, :n]
    live = z.gather(1, top) > -float("inf")
    idx[:, :n] = torch.where(live, top, -1).to(torch.int32)
    val[:, :n] = torch.where(live, Z.gather(1, top), torch.full_like(val[:, :n], -float("inf")))
    return val, idx


def distill_ref(Z, idx, t, *, temperature: float = 1.0, alpha: float = 1.0, y=None, g=None, dtype=torch.float64):
    """Oracle of ops.logits.distill_*: (loss [B], dZ [B, K]); also the CPU path of the trainer's distillation."""
    if alpha != 1.0 and y is None:
        raise ValueError("distill_ref: alpha below 1 mixes in hard labels and needs y")
    z, T = Z.to(dtype), float(temperature)
    B, K = z.shape
    inf = float("inf")
    idx, tt = idx.long(), t.to(dtype)
    bad = (idx >= K).any(1)
    there = (idx >= 0) & (idx < K) & (tt != -inf)
    some = ~(z == -inf).all(1, keepdim=True)
    x = torch.where(there, tt / T, torch.full_like(tt, -inf))
    mx = x.amax(1, keepdim=True)
    e = torch.where(there, torch.exp(x - torch.where(mx == -inf, torch.zeros_like(mx), mx)), torch.zeros_like(x))
    s = e.sum(1, keepdim=True)
    q = torch.where(some & (s != 0), e / s, torch.zeros_like(e))
    target = torch.zeros_like(z).scatter_add_(1, idx.clamp(0, K - 1), torch.where(there, q, torch.zeros_like(q)))

    def part(scale, target):
        w = torch.where(some, z / scale, torch.zeros_like(z))
        lp = torch.log_softmax(w, 1)
        cross = -torch.where(target != 0, target * lp, torch.zeros_like(lp)).sum(1)
        grad = torch.exp(lp) * target.sum(1, keepdim=True) - target
        return cross, torch.where(some, grad, torch.zeros_like(grad))

    cross, grad = part(T, target)
    ent = torch.where(q != 0, q * torch.log(torch.where(q != 0, q, torch.ones_like(q))), torch.zeros_like(q)).sum(1)
    masked = there & (z.gather(1, idx.clamp(0, K - 1)) == -inf) & some  # also where q underflows
    cross = cross.masked_fill(masked.any(1), inf)
    if alpha == 0.0:
        cross = ent = torch.zeros_like(cross)
    loss, dz = alpha * T * T * (cross + ent), alpha * T * grad
    if y is not None and alpha != 1.0:
        y = y.long()
        bad |= y >= K
        hot = torch.zeros_like(z)
        hot.scatter_(1, y.clamp(0, K - 1)[:, None], ((y >= 0) & some[:, 0]).to(dtype)[:, None])
        cross, grad = part(1.0, hot)
        loss, dz = loss + (1 - alpha) * cross, dz + (1 - alpha) * grad
    nan = float("nan")
    loss, dz = loss.masked_fill(bad, nan), dz.masked_fill(bad[:, None], nan)
    return loss, dz if g is None else dz * g.to(dtype)[:, None]


def sample_ref(Z, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Oracle of ops.logits.sample_logits in float64 (any device): (idx int32 [B], prob f64 [B])."""
    B, K = Z.shape
    z, order = _class_order(Z)
    col = lambda v: (v.float() if isinstance(v, torch.Tensor) else  # noqa: E731
                     torch.full((B,), float(v), dtype=torch.float32, device=Z.device)).double()[:, None]
    T, k, p, least = col(temperature), col(top_k), col(top_p), col(min_p).clamp(max=1.0)
    most = torch.finfo(torch.float32).max
    T = T.nan_to_num(most).clamp(max=most)
    m = z.amax(1, keepdim=True)
    live = z > -float("inf")
    x = torch.where(z == m, torch.zeros_like(z), (z - m) / T)
    w = torch.where(live, torch.exp(x), torch.zeros_like(z)).nan_to_num(0.0).gather(1, order)
    rank = torch.arange(K, device=Z.device)[None]
    w = torch.where(((rank < k) | (k <= 0)) & ((rank == 0) | (T > 0)), w, torch.zeros_like(w))
    mass = w.cumsum(1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    keep = (before < p * mass[:, -1:]) | (rank == 0) | ~(p < 1)
    keep &= (w >= least) | ~(least > 0)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    mass = w.cumsum(1)
    uu = u.float().nan_to_num(0.0).clamp(0.0, 1.0 - 2.0 ** -24).double()[:, None]
    idx = (mass <= uu * mass[:, -1:]).sum(1).clamp(max=K - 1)
    prob = w.gather(1, idx[:, None])[:, 0] / mass[:, -1].clamp(min=1e-300)
    none = mass[:, -1] == 0
    return torch.where(none, -1, idx).to(torch.int32), torch.where(none, torch.zeros_like(prob), prob)


def softmax_distill_ref(X_aug, W_aug, idx, t, *, temperature=1.0, alpha=1.0, y=None, dtype=torch.float32):
    """Oracle of ops.linear.softmax_distill_grad: (G [B, K], dW_aug [K, F_aug], loss_sum, n_correct). Also the CPU path of
    the trainer's distillation (dtype float32)."""
    X = X_aug.to(dtype)
    z = X @ W_aug.to(dtype).T
    loss, G = distill_ref(z, idx, t, temperature=temperature, alpha=alpha, y=y, dtype=dtype)
    correct = 0.0 if y is None else (torch.argmax(z, dim=1) == y.long()).sum().to(dtype)
    return G, G.T @ X, loss.sum(), correct
