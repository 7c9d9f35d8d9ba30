"""Rows of class logits at which the row operators could go wrong, and bounds on their rounding."""
import torch

INF = float("inf")
LOWEST = {torch.float32: torch.finfo(torch.float32).min, torch.bfloat16: torch.finfo(torch.bfloat16).min,
          torch.float16: torch.finfo(torch.float16).min}


def rows(B, K, dtype, seed, kind="bell", pad=0, device="cpu"):
    """[B, K] logits. bell: normal with one raised class; ties: a few distinct values; masked: half of them -inf, row
    0 wholly, row 1 but for one class; lowest: masked with the type's lowest value; odd: NaN, both infinities
    and both zeros among them; flat: all equal; steep: spread over the exponent range of the type."""
    g = torch.Generator().manual_seed(seed)
    Z = torch.randn(B, K, generator=g) * 2
    Z[torch.arange(B), torch.randint(0, K, (B,), generator=g)] += 8 * torch.rand(B, generator=g)
    if kind == "ties":
        Z = torch.round(Z)
    elif kind in ("masked", "lowest"):
        hide = torch.rand(B, K, generator=g) < 0.5
        hide[0] = True
        if B > 1:
            hide[1] = True
            hide[1, K // 2] = False
        Z[hide] = -INF if kind == "masked" else LOWEST[dtype]
    elif kind == "odd":
        r = torch.rand(B, K, generator=g)
        Z[r < 0.05] = float("nan")
        Z[(r > 0.1) & (r < 0.2)] = -0.0
        Z[(r > 0.2) & (r < 0.3)] = 0.0
        Z[(r > 0.3) & (r < 0.4)] = -INF
        if B > 2:
            Z[2, K // 3] = INF
            Z[2, K - 1] = INF
        Z[0] = float("nan")
    elif kind == "flat":
        Z = torch.full((B, K), 1.25)
    elif kind == "steep":
        Z = torch.sign(Z) * torch.exp2(torch.rand(B, K, generator=g) * 28 - 13)
    store = torch.full((B, K + pad), 7.0, dtype=dtype)
    store[:, :K] = Z.to(dtype)
    return store.to(device)[:, :K]


def teacher(Z, k, seed, dtype=None, device="cpu"):
    """A teacher's list for Z: the top of a noisy copy; row 0 short, row 1 empty, row 2 with classes twice."""
    g = torch.Generator().manual_seed(seed)
    B, K = Z.shape
    z = Z.detach().float().cpu().nan_to_num(0.0, posinf=4.0)
    n = min(k, K)
    t, i = torch.topk(z + 0.5 * torch.randn(B, K, generator=g), n, dim=1)
    idx = torch.full((B, k), -1, dtype=torch.int32)
    val = torch.full((B, k), -INF)
    idx[:, :n] = torch.where(t == -INF, -1, i).to(torch.int32)
    val[:, :n] = t.clamp(min=-60.0).masked_fill(t == -INF, -INF)
    if k > 1:
        idx[0, k // 2:] = -1
    if B > 1:
        val[1] = -INF
    if B > 2 and k > 2:
        idx[2, 1], idx[2, 2] = idx[2, 0], idx[2, 0]
        val[2, 1:3] = val[2, :1] - 0.5
    return idx.to(device), val.to(dtype or Z.dtype).to(device)


def distill_bounds(Z, idx, t, loss, dz, *, temperature, alpha, y=None, g=None, adds=512):
    """Elementwise bounds on an f32 evaluation, its gradient rounded once to Z's type, around the f64 results.

    An exponential of x = (z - m) / T takes x rounded three times (difference, scale, product with log2 e) and
    one more rounding: relative error (3 |x| + 2) 2^-24. A sum of n positive terms, cut over threads that add at
    most ``adds`` terms each and joined by trees of at most 16 levels, adds (adds + 16) 2^-24. Terms with x < -20
    are below 2^-28 of the sum, so |x| counts up to 20 in a sum, and in full in a term of its own."""
    u = 2.0 ** -24
    z, T = Z.double(), temperature
    B, K = z.shape
    m = z.masked_fill(z == INF, 0).amax(1, keepdim=True).clamp(min=-1e300)
    x = ((m - z) / T).nan_to_num(0.0, posinf=0.0)
    x1 = x * T
    sums = (3 * 20 + 2 + adds + 16) * u
    there = (idx >= 0) & (idx < K) & (t > -INF)
    tt = t.double().masked_fill(~there, -INF)
    mt = tt.amax(1, keepdim=True).clamp(min=-1e300)
    xt = ((mt - tt) / T).nan_to_num(0.0, posinf=0.0)
    w = torch.exp((tt - mt) / T)
    q = torch.where(there, w / w.sum(1, keepdim=True).clamp(min=1e-300), torch.zeros_like(w))
    live = torch.isfinite(z).any(1, keepdim=True)
    p = torch.softmax(torch.where(live, z / T, torch.zeros_like(z)), 1) * live
    p1 = torch.softmax(torch.where(live, z, torch.zeros_like(z)), 1) * live
    q_err = q * ((3 * xt + 3) * u + sums)  # numerator, sum, division
    dense = torch.zeros_like(z).scatter_add_(1, idx.long().clamp(0, K - 1), q)
    dense_err = torch.zeros_like(z).scatter_add_(1, idx.long().clamp(0, K - 1), q_err + 2 * q * u)
    d_at = x.gather(1, idx.long().clamp(0, K - 1))
    ln_q = torch.where(q > 0, -torch.log(q.clamp(min=1e-300)), torch.zeros_like(q))
    # every term q (ln q - (z - m) / T + ln s): its parts rounded, and their own errors
    part = q * ((ln_q + d_at + 14) * 6 * u + 2 * sums) + q_err * (ln_q + d_at + 14)
    tol_loss = alpha * T * T * part.sum(1)
    tol_dz = alpha * T * (p * ((3 * x + 8) * u + sums) + dense_err + (p + dense) * 4 * u)
    if y is not None and alpha != 1.0:
        on = (y >= 0)[:, None]
        at = y.long().clamp(0, K - 1)[:, None]
        tol_loss = tol_loss + (1 - alpha) * (((x1.gather(1, at) + 14) * 4 * u + sums) * on)[:, 0]
        hot = torch.zeros_like(z).scatter_(1, at, on.double())
        tol_dz = tol_dz + (1 - alpha) * on * (p1 * ((3 * x1 + 8) * u + sums) + (p1 + hot) * 4 * u)
    if g is not None:
        tol_dz = tol_dz * g.double().abs()[:, None]
    fi = torch.finfo(Z.dtype)
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[Z.dtype]
    tol_dz = tol_dz + half * dz.abs().nan_to_num(0.0, posinf=0.0) + fi.tiny * (half if Z.dtype == torch.float16 else 2)
    return tol_loss + 2 * u * loss.abs().nan_to_num(0.0, posinf=0.0) + 1e-37, tol_dz
