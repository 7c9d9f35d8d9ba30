"""Row operators over class logits (top_logits, distill_*, sample_logits) against plain 64-bit forms."""
import math
import random

import pytest
import torch

from logits_cases import INF, LOWEST, distill_bounds, rows, teacher
from mlapi_amd.ops import logits as ops
from mlapi_amd.ops import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (3, 2), (5, 63), (4, 64), (7, 257), (9, 1000), (2, 1025), (3, 2051), (2, 8192), (3, 8200), (2, 33333),
          (1, 131075)]
KINDS = ["bell", "ties", "masked", "lowest", "odd", "flat", "steep"]


def same(a, b):
    """Bit equality of values, NaN and signed zeros included."""
    a, b = a.detach().cpu(), b.detach().cpu()
    v = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return a.shape == b.shape and torch.equal(a.view(v), b.view(v))


# -------------------------------------------------------------------------------------------- top
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K", SHAPES)
@pytest.mark.parametrize("k", [1, 8, 65, 300])
def test_top_logits(dtype, B, K, k):
    for n, kind in enumerate(KINDS):
        Z = rows(B, K, dtype, 10 * n + k, kind, pad=(0, 3)[n % 2], device=DEV)
        val, idx = ops.top_logits(Z, k)
        rv, ri = ref.top_logits_ref(Z, k)
        assert torch.equal(idx, ri), kind
        assert same(val, rv), kind


@pytest.mark.parametrize("k", [1000, 1024])
def test_top_logits_longest_lists(k):
    for kind in ("bell", "flat", "masked"):
        for K in (999, 1024, 5000, 40000):
            Z = rows(3, K, torch.float32, 5, kind, device=DEV)
            val, idx = ops.top_logits(Z, k)
            rv, ri = ref.top_logits_ref(Z, k)
            assert torch.equal(idx, ri) and same(val, rv), (kind, K)


@pytest.mark.parametrize("B", [33, 400, 2000])
def test_top_logits_many_rows(B):
    Z = rows(B, 1003, torch.bfloat16, 8, "bell", device=DEV)
    val, idx = ops.top_logits(Z, 16)
    rv, ri = ref.top_logits_ref(Z, 16)
    assert torch.equal(idx, ri) and same(val, rv)


# ------------------------------------------------------------------------------------ distillation
def check_distill(Z, idx, t, temperature, alpha, y=None, g=None):
    kw = dict(temperature=temperature, alpha=alpha, y=y)
    rl, rd = ref.distill_ref(Z, idx, t, g=g, **kw)
    tl, td = distill_bounds(Z.cpu(), idx.cpu(), t.cpu(), rl.cpu(), rd.cpu(), temperature=temperature, alpha=alpha,
                            y=None if y is None else y.cpu(), g=None if g is None else g.cpu())
    loss, dz = ops.distill_loss_grad(Z, idx, t, g=g, **kw)
    loss2, stats = ops.distill_loss(Z, idx, t, **kw)
    dz2 = ops.distill_grad(Z, idx, t, stats, g=g, **kw)
    for l, d in ((loss, dz), (loss2, dz2)):
        l, d, el, ed = l.double().cpu(), d.double().cpu(), rl.cpu(), rd.cpu()
        assert torch.equal(l.isnan(), el.isnan()) and torch.equal(d.isnan(), ed.isnan())
        ok = el.isnan() | (l == el) | ((l - el).abs() <= tl)
        assert ok.all(), (l[~ok][:4], el[~ok][:4], tl[~ok][:4])
        ok = ed.isnan() | (d == ed) | ((d - ed).abs() <= td)
        assert ok.all(), (d[~ok][:4], ed[~ok][:4], td[~ok][:4], ok.logical_not().nonzero()[:4])
    return loss, dz


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K", SHAPES)
@pytest.mark.parametrize("k,temperature,alpha", [(1, 1.0, 1.0), (8, 2.0, 1.0), (33, 0.7, 0.4), (65, 3.0, 0.0), (12, 1.0, 0.5)])
def test_distill(dtype, B, K, k, temperature, alpha):
    for n, kind in enumerate(["bell", "ties", "masked", "lowest", "flat"]):
        Z = rows(B, K, dtype, 3 * n + k, kind, pad=(0, 5)[n % 2], device=DEV)
        idx, t = teacher(Z, k, n, dtype=TYPES[(n + k) % 3], device=DEV)
        y = g = None
        if alpha != 1.0:
            gen = torch.Generator().manual_seed(n)
            y = torch.randint(-1, K, (B,), generator=gen).to(torch.int32).to(DEV)
            g = (torch.rand(B, generator=gen) * 2 - 1).to(DEV)
        check_distill(Z, idx, t, temperature, alpha, y, g)


@pytest.mark.parametrize("temperature", [0.01, 0.7, 1.0, 1.4, 2.0])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [9, 3000, 70001])
def test_distill_lists_with_logits_of_the_types_lowest(K, dtype, temperature):
    """A teacher that masks with its type's lowest logit lists such classes wherever fewer than k are left."""
    k = min(K, 40)
    Zt = torch.full((5, K), LOWEST[dtype])
    Zt[1:, ::max(2, K // 7)] = rows(4, len(range(0, K, max(2, K // 7))), torch.float32, 3)
    Zt = Zt.to(dtype).to(DEV)
    t, idx = ops.top_logits(Zt, k)
    assert (t.double().min(1).values == LOWEST[dtype]).all()
    y = torch.tensor([0, 3, -1, K - 1, 2], dtype=torch.int32, device=DEV)
    g = torch.full((5,), -0.5, device=DEV)
    Z = rows(5, K, dtype, 4, "bell", device=DEV)
    loss, dz = check_distill(Z, idx, t, temperature, 1.0)
    assert loss.isfinite().all() and dz.isfinite().all()
    check_distill(Z, idx, t, temperature, 0.3, y, g)
    # a student that masks so too: its loss may be past the largest f32, whose place +inf takes
    Z = rows(5, K, dtype, 4, "lowest", device=DEV)
    kw = dict(temperature=temperature, alpha=0.3, y=y)
    rl, rd = (v.cpu() for v in ref.distill_ref(Z, idx, t, g=g, **kw))
    tl, td = distill_bounds(Z.cpu(), idx.cpu(), t.cpu(), rl, rd, temperature=temperature, alpha=0.3, y=y.cpu(), g=g.cpu())
    loss, dz = (v.double().cpu() for v in ops.distill_loss_grad(Z, idx, t, g=g, **kw))
    past = rl + tl > torch.finfo(torch.float32).max
    assert ((loss - rl).abs() <= tl)[~past].all() and ((loss == INF) | (loss >= rl - tl))[past].all(), (loss, rl, tl)
    assert ((dz - rd).abs() <= td).all()


@pytest.mark.parametrize("B,K", [(5, 1000), (3, 2048), (6, 1100), (2, 9000), (2, 150001)])
def test_distill_longest_lists(B, K):
    for k in (1000, 1024):
        Z = rows(B, K, torch.float32, k, "bell", device=DEV)
        idx, t = teacher(Z, k, 3, device=DEV)
        y = torch.arange(B, dtype=torch.int32, device=DEV)
        check_distill(Z, idx, t, 1.5, 0.6, y)


@pytest.mark.parametrize("dtype,B,K", [(torch.float32, 33, 33001), (torch.float32, 40, 65536), (torch.float32, 35, 32769)] +
                         [(t, B, K) for t in TYPES[1:] for B, K in ((33, 65537), (40, 131072), (34, 131071))])
def test_distill_longest_rows_in_registers(dtype, B, K):
    """1024 threads of 16 vectors each: more than 32 rows of 8193 to 16384 vectors."""
    k = 12
    Z = rows(B, K, dtype, 9, "bell", pad=3, device=DEV)
    idx, t = teacher(Z, k, 3, device=DEV)
    idx[4, 0], idx[5, 1] = K - 1, 0
    g = torch.linspace(-1, 1, B).to(DEV)
    y = torch.randint(-1, K, (B,), generator=torch.Generator().manual_seed(K)).to(torch.int32).to(DEV)
    y[4], y[6] = K - 1, idx[6, 2]
    for kw in (dict(temperature=2.0, alpha=1.0), dict(temperature=1.0, alpha=0.5, y=y, g=g),
               dict(temperature=0.7, alpha=0.4, y=y, g=g)):
        loss, dz = check_distill(Z, idx, t, **kw)
        pred = torch.empty(B, dtype=torch.int32, device=DEV)
        own = Z.clone()  # the row stride of the clone: K
        l2, d2 = ops.distill_loss_grad(own, idx, t, out=own, pred=pred, **kw)
        assert d2.data_ptr() == own.data_ptr() and same(l2, loss) and same(d2, dz)
        assert torch.equal(pred.long(), Z.float().argmax(1))
        if dtype == torch.float32:
            _, d3 = ops.distill_loss_grad(Z, idx, t, out=torch.empty(B, K, dtype=torch.bfloat16, device=DEV), **kw)
            assert same(d3, dz.to(torch.bfloat16))


def test_distill_one_list_for_all_rows():
    """idx and t may be expanded: a row stride of 0."""
    Z = rows(9, 700, torch.bfloat16, 2, "bell", device=DEV)
    idx, t = teacher(Z[3:4], 6, 3, device=DEV)
    loss, dz = ops.distill_loss_grad(Z, idx.expand(9, -1), t.expand(9, -1), temperature=2.0)
    l2, d2 = ops.distill_loss_grad(Z, idx.repeat(9, 1), t.repeat(9, 1), temperature=2.0)
    assert same(loss, l2) and same(dz, d2)


def hot_bounds(Z, idx, t, loss, dz, *, temperature, alpha, y=None, g=None):
    """Bounds at temperatures above 16. Rows whose list holds all but 1/64 of p (and 2^-16, what f32 may see amiss): sums, listed
    classes and the loss are 64-bit: both sides' exponentials (2
    steps of 2^-52) and sums over at most 64 terms a thread, a wave's and a block's, count T^2 in the loss; the loss is rounded
    to f32 once. A class that is not listed: an f32 exponential, its argument rounded three times, two factors. The
    gradient is rounded to its type through f32. Other rows are evaluated in f32, a thread adding K / 64 terms at most."""
    T, z, u, w = temperature, Z.double(), 2.0 ** -24, 2.0 ** -52
    K = z.shape[1]
    x = (z.masked_fill(z == INF, 0).amax(1, keepdim=True).clamp(min=-1e300) - z).nan_to_num(0.0, posinf=0.0)
    live = (z > -INF).any(1, keepdim=True)
    p, p1 = (torch.softmax(torch.where(live, z / s, torch.zeros_like(z)), 1) * live for s in (T, 1.0))
    far = x.amax(1) / T  # the logarithms are at most this and ln K
    tol_loss = 2 * u * loss.abs() + alpha * T * T * (100 * w + (math.log(K) + far) * 8 * w)
    listed = torch.zeros(z.shape, dtype=torch.bool).scatter_(1, idx.long().clamp(0, K - 1), (idx >= 0) & (t > -INF))
    tol_dz = alpha * T * (p + 1) * 100 * w + alpha * T * p * (3 * x / T + 8) * u * ~listed
    if y is not None and alpha != 1.0:
        tol_dz = tol_dz + (1 - alpha) * p1 * (3 * x + 8) * u
    if g is not None:
        tol_dz = tol_dz * g.double().abs()[:, None]
    half = {torch.float32: u, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[Z.dtype]
    tiny = torch.finfo(Z.dtype).tiny * (half if Z.dtype == torch.float16 else 2)
    tol_dz = tol_dz + (half + u) * dz.abs() + tiny
    on = torch.where((idx >= 0) & (t > -INF), p.gather(1, idx.long().clamp(0, K - 1)), torch.zeros(())).sum(1)
    near = on > 63 / 64 + 2.0 ** -16 if alpha else torch.zeros(len(z), dtype=torch.bool)
    tl, td = distill_bounds(Z, idx, t, loss, dz, temperature=T, alpha=alpha, y=y, g=g, adds=min(512, 16 + K // 64))
    return torch.where(near, tol_loss, torch.maximum(tl, tol_loss)), torch.where(near[:, None], tol_dz, torch.maximum(td, tol_dz))


@pytest.mark.parametrize("temperature", [16.0, 16.5, 100.0, 1e4, 1e6])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,k", [(3, 2, 2), (5, 64, 64), (4, 1000, 1000), (6, 1024, 40), (3, 3000, 900), (2, 20000, 700),
                                   (2, 140001, 900)])
def test_distill_at_high_temperatures(B, K, k, dtype, temperature):
    """Lists of every class that the student does not mask (and, k = 40, of some): p nears q, the loss does not vanish."""
    hidden = torch.ones(K, dtype=torch.bool)
    hidden[torch.randperm(K, generator=torch.Generator().manual_seed(1))[:max(k, 64)]] = False
    Z = rows(B, K, torch.float32, 5)
    t = Z + 0.7 * torch.randn(B, K, generator=torch.Generator().manual_seed(2))
    Z = Z.masked_fill(hidden, -INF).to(dtype).to(DEV)
    t, idx = ops.top_logits(t.masked_fill(hidden, -INF).to(dtype).to(DEV), k)
    if k > 2:
        idx[0, 1], t[0, 2] = idx[0, 0], -INF  # a class twice, an entry absent
    for alpha in (1.0, 0.4):
        y = g = None
        if alpha != 1.0:
            y = idx[:, min(k - 1, 7)].clone()
            y[0] = -1
            g = torch.linspace(-1, 2, B).to(DEV)
        kw = dict(temperature=temperature, alpha=alpha, y=y)
        rl, rd = ref.distill_ref(Z, idx, t, g=g, **kw)
        cpu = lambda v: None if v is None else v.cpu()  # noqa: E731
        how = dict(temperature=temperature, alpha=alpha, y=cpu(y), g=cpu(g))
        bounds = hot_bounds if temperature > 16 else distill_bounds
        tl, td = bounds(Z.cpu(), idx.cpu(), t.cpu(), rl.cpu(), rd.cpu(), **how)
        if temperature == 1e4 and k == K and alpha == 1.0:
            assert (tl <= 1e-4 * rl.cpu().abs() + 1e-5)[1:].all()  # the bound itself is far below the loss
        loss, dz = ops.distill_loss_grad(Z, idx, t, g=g, **kw)
        l2, stats = ops.distill_loss(Z, idx, t, **kw)
        d2 = ops.distill_grad(Z, idx, t, stats, g=g, **kw)
        own = Z.clone()
        l3, d3 = ops.distill_loss_grad(own, idx, t, g=g, out=own, **kw)
        assert temperature <= 16 or same(loss, l2) and same(loss, l3) and same(dz, d3)
        assert temperature <= 16 or K > 65536 or same(dz, d2)  # rows in parts: a merge's order shows in the last bit
        l, d, rl, rd = loss.double().cpu(), dz.double().cpu(), rl.cpu(), rd.cpu()
        ok = (l - rl).abs() <= tl
        assert ok.all(), (l[~ok], rl[~ok], tl[~ok])
        if temperature > 16:  # in f32 a loss of T^2 / 64 at least, a sum off by 64 + 16 roundings at most: 2^-11 of it
            assert ((l - rl).abs() <= 2.0 ** -11 * rl + tl.clamp(max=1e-2)).all()
        ok = (d - rd).abs() <= td
        assert ok.all(), (d[~ok][:4], rd[~ok][:4], td[~ok][:4], ok.logical_not().nonzero()[:4])


@pytest.mark.parametrize("K", [300, 5000, 40000, 150001])
def test_distill_at_high_temperatures_next_to_rows_that_take_32_bits(K):
    """Near rows and others in one batch, into bf16 and in place, with padded rows: each as it is alone."""
    B, k, T = 40, 200, 40.0
    Z = rows(B, K, torch.float32, 5, pad=3)
    t = Z + 0.7 * torch.randn(B, K, generator=torch.Generator().manual_seed(2))
    hidden = torch.ones(K, dtype=torch.bool)
    hidden[torch.randperm(K, generator=torch.Generator().manual_seed(1))[:k]] = False
    for v in (Z, t):
        v[::2] = v[::2].masked_fill(hidden, -INF)
    store = torch.empty(B, K + 3, device=DEV)
    Z, t = store[:, :K].copy_(Z.to(DEV)), t.to(DEV)
    t, idx = ops.top_logits(t, k)
    y = idx[:, 3].clone()
    g = torch.linspace(-1, 2, B).to(DEV)
    kw = dict(temperature=T, alpha=0.7)
    rl, rd = (v.cpu() for v in ref.distill_ref(Z, idx, t, y=y, g=g, **kw))
    tl, td = hot_bounds(Z.cpu(), idx.cpu(), t.cpu(), rl, rd, y=y.cpu(), g=g.cpu(), **kw)
    assert (tl[::2] < 1e-4).all()
    pred = torch.empty(B, dtype=torch.int32, device=DEV)
    loss, dz = ops.distill_loss_grad(Z, idx, t, y=y, g=g, pred=pred, **kw)
    assert ((loss.double().cpu() - rl).abs() <= tl).all() and ((dz.double().cpu() - rd).abs() <= td).all()
    assert torch.equal(pred.long(), Z.argmax(1))
    _, half = ops.distill_loss_grad(Z, idx, t, y=y, g=g, out=torch.empty(B, K, dtype=torch.bfloat16, device=DEV), **kw)
    assert same(half, dz.to(torch.bfloat16))
    for part in (slice(0, None, 2), slice(1, None, 2)):
        l2, d2 = ops.distill_loss_grad(Z[part], idx[part], t[part], y=y[part].contiguous(), g=g[part].contiguous(), **kw)
        if K <= 32768:  # longer rows are cut into as many parts as the batch has room for
            assert same(l2, loss[part].contiguous()) and same(d2, dz[part].contiguous())
    own, pad = ops.distill_loss_grad(Z, idx, t, y=y, g=g, out=Z, **kw), store[:, K:].clone()
    assert same(own[0], loss) and same(own[1].contiguous(), dz) and same(store[:, K:].contiguous(), pad)
    l2, stats = ops.distill_loss(Z, idx, t, y=y, **kw)  # now of the gradient's rows: only that it runs
    assert l2.isfinite().all()


@pytest.mark.parametrize("B,K", [(3, 40), (3, 3000), (2, 150001)])
def test_distill_at_high_temperatures_captured(B, K):
    Z = rows(B, K, torch.float32, 5, device=DEV)
    t, idx = ops.top_logits(Z + 0.5, min(K, 60))
    call = lambda: ops.distill_loss_grad(Z, idx, t, temperature=30.0)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, dz = call()
    for r in range(4):
        Z.copy_(rows(B, K, torch.float32, 10 + r, device=DEV))
        t.copy_(ops.top_logits(Z + 0.1 * r, t.shape[1], out=(torch.empty_like(t), idx))[0])
        loss.fill_(-3), dz.fill_(-3)
        graph.replay()
        l2, d2 = call()
        torch.cuda.synchronize()
        assert same(loss, l2) and same(dz, d2)


def test_distill_at_high_temperatures_of_rows_without_a_class_or_out_of_range():
    for K in (40, 5000, 40000):
        Z = rows(8, K, torch.float32, 1, device=DEV)
        idx, t = teacher(Z, 8, 1, device=DEV)
        y = torch.zeros(8, dtype=torch.int32, device=DEV)
        Z[0], Z[2, 5], Z[3, 7] = -INF, float("nan"), INF
        idx[4, 2], y[5] = K, K + 9
        t[6, 1] = float("nan")
        Z[7, idx[7, 0].long()] = -INF
        pred = torch.empty(8, dtype=torch.int32, device=DEV)
        loss, dz = ops.distill_loss_grad(Z, idx, t, temperature=50.0, alpha=0.5, y=y, pred=pred)
        assert loss[0] == 0 and (dz[0] == 0).all() and loss[2:7].isnan().all() and dz[2:7].isnan().all()
        assert loss[1].isfinite() and dz[1].isfinite().all() and loss[7] == INF and dz[7].isfinite().all()
        assert pred[1] == Z[1].argmax() and pred[3] == 7 and pred[0] == 0


def test_distill_nan_inf_and_classes_out_of_range():
    for K in (100, 3000, 70000):
        Z = rows(8, K, torch.float32, 1, "bell", device=DEV)
        idx, t = teacher(Z, 8, 1, device=DEV)
        y = torch.zeros(8, dtype=torch.int32, device=DEV)
        Z[3, 5], Z[4, 7] = float("nan"), INF
        idx[5, 2], y[6] = K, K + 9
        t[7, 1] = float("nan")
        loss, dz = ops.distill_loss_grad(Z, idx, t, temperature=2.0, alpha=0.5, y=y)
        assert loss[3:].isnan().all() and dz[3:].isnan().all()
        assert loss[:3].isfinite().all() and dz[:3].isfinite().all()
        loss, stats = ops.distill_loss(Z, idx, t, temperature=2.0, alpha=0.5, y=y)
        dz = ops.distill_grad(Z, idx, t, stats, temperature=2.0, alpha=0.5, y=y)
        assert loss[3:].isnan().all() and dz[3:].isnan().all() and dz[:3].isfinite().all()


@pytest.mark.parametrize("K", [500, 5000, 50000])
def test_distill_gradient_sums_to_zero_and_matches_differences(K):
    """Both softmaxes sum to one, so a row's gradient sums to zero; and a step along a random direction
    changes the 64-bit loss by the gradient's product with it."""
    B, k, T, alpha = 4, 12, 1.7, 0.6
    Z = rows(B, K, torch.float32, 2, "bell", device=DEV)
    idx, t = teacher(Z, k, 2, device=DEV)
    y = torch.randint(0, K, (B,), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(DEV)
    kw = dict(temperature=T, alpha=alpha, y=y)
    _, dz = ops.distill_loss_grad(Z, idx, t, **kw)
    # every element is off by at most (adds + 100) 2^-24 of its two parts, whose sums over a row are 2 (a T + 1 - a)
    assert (dz.double().sum(1).abs() <= 2 * (alpha * T + 1 - alpha) * 700 * 2.0 ** -24).all()
    D = torch.randn(B, K, generator=torch.Generator().manual_seed(3), dtype=torch.float64).to(DEV)
    h = 1e-4
    up, dn = (ref.distill_ref(Z.double() + s * h * D, idx, t, **kw)[0] for s in (1, -1))
    slope, want = (dz.double() * D).sum(1), (up - dn) / (2 * h)
    # third differences: h^2 / 6 times a third derivative below 8 max|D|^3 / T; rounding of dz as above
    tol = h * h * 8 * D.abs().amax() ** 3 + 700 * 2.0 ** -24 * 2 * T * D.abs().amax()
    assert ((slope - want).abs() <= tol).all()


@pytest.mark.parametrize("K", [1000, 9000, 150001])
def test_distill_in_place_and_bf16_out(K):
    Z = rows(5, K, torch.float32, 4, "bell", pad=7, device=DEV)
    idx, t = teacher(Z, 20, 4, device=DEV)
    y = torch.arange(5, dtype=torch.int32, device=DEV)
    kw = dict(temperature=2.0, alpha=0.5, y=y)
    loss, dz = ops.distill_loss_grad(Z, idx, t, **kw)
    wide = torch.full((5, K + 24), 3.0, dtype=torch.bfloat16, device=DEV)
    l2, d2 = ops.distill_loss_grad(Z, idx, t, out=wide[:, :K], **kw)
    assert same(d2, dz.to(torch.bfloat16)) and same(l2, loss)
    assert (wide[:, K:] == 3.0).all()
    store = torch.empty(5, K + 7, device=DEV).copy_(torch.nn.functional.pad(Z, (0, 7), value=5.0))
    own = store[:, :K]
    l3, d3 = ops.distill_loss_grad(own, idx, t, out=own, **kw)
    assert d3.data_ptr() == own.data_ptr() and same(d3.contiguous(), dz) and same(l3, loss)
    assert (store[:, K:] == 5.0).all()


@pytest.mark.parametrize("K", [40, 3000, 40000])
def test_distill_pred_is_the_first_maximum(K):
    for kind in ("bell", "ties", "flat"):
        Z = rows(6, K, torch.bfloat16, 6, kind, device=DEV)
        idx, t = teacher(Z, 4, 6, device=DEV)
        pred = torch.full((6,), -7, dtype=torch.int32, device=DEV)
        ops.distill_loss_grad(Z, idx, t, pred=pred)
        assert torch.equal(pred.long(), Z.float().argmax(1)), kind


# ---------------------------------------------------------------------------------------- sampling
def check_sample(Z, u, **kw):
    idx, prob = ops.sample_logits(Z, u, **kw)
    ri, rp = ref.sample_ref(Z, u, **kw)
    assert torch.equal(idx, ri), (idx[idx != ri][:4], ri[idx != ri][:4], kw)
    # one rounding of the quotient to f32; the masses' own steps are 2^-42 of the largest weight
    assert ((prob.double() - rp).abs() <= rp * (2.0 ** -24 + 2.0 ** -40) + Z.shape[1] * 2.0 ** -42).all()
    return idx, prob


FILTERS = [dict(), dict(temperature=0.3), dict(top_k=1), dict(top_k=50), dict(top_k=400, temperature=1.4),
           dict(top_p=0.9), dict(top_p=0.05), dict(min_p=0.1), dict(min_p=1.0), dict(top_p=0.0),
           dict(top_k=2000, top_p=0.8, min_p=0.02, temperature=0.8), dict(top_k=7, top_p=0.99), dict(temperature=0.0),
           dict(temperature=1e30), dict(temperature=1e-30)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K", SHAPES)
@pytest.mark.parametrize("kind", KINDS)
def test_sample(dtype, B, K, kind):
    Z = rows(B, K, dtype, 11, kind, pad=3, device=DEV)
    for n, f in enumerate(FILTERS):
        u = torch.rand(B, generator=torch.Generator().manual_seed(n)).to(DEV)
        check_sample(Z, u, **f)


def test_sample_settings_per_row():
    B, K = 60, 1000
    Z = rows(B, K, torch.float32, 12, "bell", device=DEV)
    g = torch.Generator().manual_seed(9)
    r = torch.arange(B)
    kw = dict(temperature=torch.where(r % 5 == 0, 0.0, 0.3 + torch.rand(B, generator=g)),
              top_k=torch.where(r % 3 == 0, -1, r * 25).to(torch.int32),
              top_p=torch.where(r % 4 == 0, 1.5, torch.rand(B, generator=g)),
              min_p=torch.where(r % 7 == 0, -1.0, 0.1 * torch.rand(B, generator=g)))
    check_sample(Z, torch.rand(B, generator=g).to(DEV), **{n: v.to(DEV) for n, v in kw.items()})


@pytest.mark.parametrize("K", [50, 1900, 7000, 40000])
def test_sample_infinite_temperatures_keep_masked_classes_out(K):
    Z = rows(8, K, torch.float32, 12, "masked", device=DEV)
    inf = torch.full((8,), INF, device=DEV)
    inf[5] = float("nan")
    u = torch.rand(8, generator=torch.Generator().manual_seed(1)).to(DEV)
    for f in (dict(), dict(top_p=0.5), dict(top_k=20), dict(top_k=300, min_p=0.5)):
        idx, _ = check_sample(Z, u, temperature=inf, **f)
        assert idx[0] == -1 and (Z[torch.arange(1, 8), idx[1:].long()] > -INF).all()


@pytest.mark.parametrize("K", [1500, 20000])
def test_sample_list_lengths_of_all_kinds_in_one_batch(K):
    B = 40
    Z = rows(B, K, torch.bfloat16, 13, "bell", device=DEV)
    k = torch.tensor([0, 1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1023, K - 1, K, K + 5, -3] * 3)[:B].to(torch.int32)
    u = torch.rand(B, generator=torch.Generator().manual_seed(2)).to(DEV)
    check_sample(Z, u, top_k=k.to(DEV))
    check_sample(Z, u, top_k=k.to(DEV), top_p=0.7, temperature=1.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [1900, 7001, 40000])
def test_sample_border_among_weights_of_nothing(dtype, K):
    """The last class kept has next to no weight, and thousands behind it have none at all."""
    u = torch.tensor([0.0, 0.3, 0.7, 0.999, 1.0], device=DEV)
    for kind in ("bell", "steep", "lowest", "odd", "ties"):
        Z = rows(5, K, dtype, 14, kind, pad=1, device=DEV)
        for f in (dict(), dict(top_k=900), dict(top_k=K - 1), dict(min_p=1e-3), dict(top_k=900, min_p=1e-12)):
            for T in (0.02, 1.0, 1e4):
                check_sample(Z, u, top_p=1 - 2.0 ** -24, temperature=T, **f)


@pytest.mark.parametrize("K,large,ones,k,p", [
    (4096, 50, 1930, 2552, 0.945574164390564), (4096, 3, 1529, 3604, 0.8711135387420654),
    (4096, 0, 1417, 2745, 0.9906483888626099), (8192, 0, 3005, 6398, 0.9207276105880737),
    (4096, 0, 754, 3752, 0.956817090511322), (4096, 3, 1805, 2558, 0.9588007926940918)])
def test_sample_borders_among_zeros_above_a_border_among_ties(K, large, ones, k, p):
    """top-k ends among equal logits below zero and the nucleus among more zeros than its list holds, so that its
    border is searched from one that lies between two logits: zeros of either sign are kept by their class alone."""
    z = torch.zeros(K)
    z[:large], z[K - ones:] = 2.0, -1.0
    z[large:K - ones:2] = -0.0
    z = z[torch.tensor(random.Random(K + large + ones).sample(range(K), K))]
    u = torch.tensor([0.0, 0.2, 0.4, 0.6, 0.8, 0.999, 1.0], device=DEV)
    for dtype in TYPES:
        Z = z.to(dtype).to(DEV).expand(7, K).contiguous()
        check_sample(Z, u, top_k=k, top_p=p)
        check_sample(Z, u, top_k=torch.full((7,), k, dtype=torch.int32, device=DEV), top_p=p, min_p=0.3)


def test_sample_random_numbers_at_their_ends():
    """Four equal classes: u splits [0, 1) exactly in quarters; 1 and above, NaN and negative are taken in."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, float("nan"), 0.25 - 2.0 ** -26], device=DEV)
    Z = torch.full((10, 9), -INF, device=DEV)
    Z[:, [1, 3, 4, 8]] = 2.0
    idx, prob = ops.sample_logits(Z, u)
    assert idx.tolist() == [1, 3, 4, 8, 8, 8, 8, 1, 1, 1]
    assert (prob == 0.25).all()


def test_sample_frequencies_follow_the_probabilities():
    """n draws of one row with u at the n midpoints: every class comes n p times, to within its two ends."""
    n, K = 4096, 50
    z = rows(1, K, torch.float32, 3, "bell", device=DEV)
    idx, _ = ops.sample_logits(z.expand(n, K).contiguous(), (torch.arange(n, device=DEV) + 0.5) / n)
    got = torch.bincount(idx.long(), minlength=K).double()
    assert ((got - n * torch.softmax(z[0].double(), 0)).abs() <= 1.0 + 1e-6 * n).all()


# ------------------------------------------------------------------- together, captured, elsewhere
def step(Zt, Zs, y, u):
    val, idx = ops.top_logits(Zt, 16)
    loss, dz = ops.distill_loss_grad(Zs, idx, val, temperature=2.0, alpha=0.5, y=y)
    label, prob = ops.sample_logits(Zs, u, temperature=0.7, top_k=20, top_p=0.9)
    return val, idx, loss, dz, label, prob


@pytest.mark.parametrize("B,K", [(4, 1000), (200, 1000), (3, 50000), (40, 9000)])
def test_captured_run_matches_eager_on_every_replay(B, K):
    Zt, Zs = (rows(B, K, torch.float32, s, "bell", device=DEV) for s in (1, 2))
    y = torch.zeros(B, dtype=torch.int32, device=DEV)
    u = torch.rand(B, generator=torch.Generator().manual_seed(0)).to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(Zt, Zs, y, u)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(Zt, Zs, y, u)
    for r in range(4):
        Zt.copy_(rows(B, K, torch.float32, 10 + r, "bell", device=DEV))
        Zs.copy_(rows(B, K, torch.float32, 20 + r, "bell", device=DEV))
        for t in got:
            t.fill_(-3)
        torch.cuda.synchronize()
        graph.replay()
        want = step(Zt, Zs, y, u)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert same(a, b)


def test_runs_on_a_side_stream_and_two_at_once():
    a, b = (rows(64, 20000, torch.float32, s, "bell", device=DEV) for s in (1, 2))
    y = torch.zeros(64, dtype=torch.int32, device=DEV)
    u = torch.rand(64, generator=torch.Generator().manual_seed(0)).to(DEV)
    want = [step(a, b, y, u), step(b, a, y, u)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        g1 = step(a, b, y, u)
    with torch.cuda.stream(s2):
        g2 = step(b, a, y, u)
    torch.cuda.synchronize()
    for got, w in zip((g1, g2), want):
        for x, v in zip(got, w):
            assert same(x, v)


def test_same_inputs_give_the_same_bits():
    Z = rows(64, 30000, torch.bfloat16, 5, "ties", device=DEV)
    y = torch.zeros(64, dtype=torch.int32, device=DEV)
    u = torch.rand(64, generator=torch.Generator().manual_seed(0)).to(DEV)
    first = step(Z, Z, y, u)
    for _ in range(3):
        for a, b in zip(first, step(Z, Z, y, u)):
            assert same(a, b)


def test_offsets_past_32_bits():
    """A row beyond 2^31 elements of its buffer: a strided view reads and writes there."""
    ld = 1 << 30
    store = torch.empty(3 * ld, dtype=torch.bfloat16, device=DEV)
    Z = store.as_strided((3, 1000), (ld, 1))
    src = rows(3, 1000, torch.bfloat16, 7, "bell", device=DEV)
    Z.copy_(src)
    val, idx = ops.top_logits(Z, 8)
    rv, ri = ref.top_logits_ref(src, 8)
    assert torch.equal(idx, ri) and same(val, rv)
    u = torch.full((3,), 0.4, device=DEV)
    assert torch.equal(ops.sample_logits(Z, u)[0], ref.sample_ref(src, u)[0])
    loss, dz = ops.distill_loss_grad(src, idx, val)
    l2, d2 = ops.distill_loss_grad(Z, idx, val, out=Z)
    assert same(l2, loss) and same(d2.contiguous(), dz)


def test_empty_batches():
    Z = torch.empty(0, 50, device=DEV)
    val, idx = ops.top_logits(Z, 4)
    assert val.shape == (0, 4) and idx.shape == (0, 4)
    loss, dz = ops.distill_loss_grad(Z, idx, val)
    assert loss.shape == (0,) and dz.shape == (0, 50)
    assert ops.sample_logits(Z, torch.empty(0, device=DEV))[0].shape == (0,)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [40000, 200000])
def test_empty_batches_of_long_rows(dtype, K):
    Z = torch.empty(0, K, dtype=dtype, device=DEV)
    val, idx = ops.top_logits(Z, 4)
    loss, stats = ops.distill_loss(Z, idx, val)
    dz = ops.distill_grad(Z, idx, val, stats)
    l2, d2 = ops.distill_loss_grad(Z, idx, val, temperature=2.0)
    assert loss.shape == l2.shape == (0,) and dz.shape == d2.shape == (0, K)
    assert ops.sample_logits(Z, torch.empty(0, device=DEV), top_k=5)[0].shape == (0,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_most_classes(dtype):
    K = 1 << 20
    Z = rows(2, K, dtype, 3, "bell", device=DEV)
    for k in (5, 200, 1000):
        val, idx = ops.top_logits(Z, k)
        rv, ri = ref.top_logits_ref(Z, k)
        assert torch.equal(idx, ri) and same(val, rv)
    for n, f in enumerate((dict(), dict(top_p=0.9), dict(top_k=40), dict(top_k=700, min_p=0.01), dict(temperature=2.0))):
        check_sample(Z, torch.rand(2, generator=torch.Generator().manual_seed(n)).to(DEV), **f)
    idx, t = teacher(Z, 100, 3, device=DEV)
    check_distill(Z, idx, t, 2.0, 0.5, torch.tensor([K - 1, 0], dtype=torch.int32, device=DEV))


def test_many_short_rows():
    B = 70001
    Z = rows(B, 3, torch.float16, 4, "ties", device=DEV)
    val, idx = ops.top_logits(Z, 2)
    rv, ri = ref.top_logits_ref(Z, 2)
    assert torch.equal(idx, ri) and same(val, rv)
    u = torch.rand(B, generator=torch.Generator().manual_seed(1)).to(DEV)
    for f in (dict(), dict(top_p=0.6), dict(top_k=2)):
        check_sample(Z, u, **f)
    loss, dz = ops.distill_loss_grad(Z, idx, val, temperature=1.5)
    rl, rd = ref.distill_ref(Z, idx, val, temperature=1.5)
    # three terms of at most 8 each and their exponentials: 200 roundings of 2^-24; f16 gradients below 1.5 once more
    assert ((loss.double() - rl).abs() <= 200 * 2.0 ** -24 * 8).all()
    assert ((dz.double() - rd).abs() <= rd.abs() * 2.0 ** -11 + 200 * 2.0 ** -24 * 8 + 2.0 ** -25).all()


def test_more_rows_than_a_launch_holds_threads_for():
    """A wave to a row: 2^26 rows are 2^32 threads. The same 4099 rows again and again give the same again and again."""
    n, times, K = 4099, 16373, 2
    base = rows(n, K, torch.float16, 4, "bell", device=DEV)
    Z = base.repeat(times, 1)
    assert Z.shape[0] > 1 << 26
    again = lambda v, one: same(v[:n], one) and torch.equal(v.view(times, *one.shape), one.expand(times, *one.shape))  # noqa: E731
    val, idx = ops.top_logits(base, 2)
    V, I = ops.top_logits(Z, 2)
    assert again(V, val) and again(I, idx)
    for T in (1.5, 20.0):
        loss, dz = ops.distill_loss_grad(base, idx, val, temperature=T)
        L, D = ops.distill_loss_grad(Z, I, V, temperature=T)
        assert again(L, loss) and again(D, dz)
        L, stats = ops.distill_loss(Z, I, V, temperature=T)
        assert again(L, loss) and again(ops.distill_grad(Z, I, V, stats, temperature=T), dz)
    del V, I, L, D, stats
    u = torch.rand(n, generator=torch.Generator().manual_seed(1)).to(DEV)
    k = torch.randint(0, 3, (n,), generator=torch.Generator().manual_seed(2)).to(torch.int32).to(DEV)
    for f, F in ((dict(), dict()), (dict(top_k=k, top_p=0.6, temperature=1 + u, min_p=u),
                                    dict(top_k=k.repeat(times), top_p=0.6, temperature=(1 + u).repeat(times), min_p=u.repeat(times)))):
        idx, prob = ops.sample_logits(base, u, **f)
        I, P = ops.sample_logits(Z, u.repeat(times), **F)
        assert again(I, idx) and again(P, prob)


def test_more_long_rows_than_a_grid_dimension():
    """Rows that are cut into parts, past 65535 of them (17 GB, written in place)."""
    B, K = 65539, 131077
    src = rows(3, K, torch.bfloat16, 5, "bell", device=DEV)
    idx, t = teacher(src, 8, 5, device=DEV)
    loss, dz = ops.distill_loss_grad(src, idx, t, temperature=2.0)
    Z = torch.zeros(B, K, dtype=torch.bfloat16, device=DEV)
    Z[-3:] = src
    idx, t = (torch.cat([v[:1].expand(B - 3, -1), v]) for v in (idx, t))
    l2, d2 = ops.distill_loss_grad(Z, idx, t, temperature=2.0, out=Z)
    assert (d2[:5].float().sum(1).abs() <= 2.0 ** -7 * 4).all()  # p - q, each entry rounded to bf16: half steps of 2 T
    # the batch is cut into other parts than three rows are: the sums' trees differ
    assert ((l2[-3:] - loss).abs() <= 1000 * 2.0 ** -24 * (loss.abs() + 8)).all()
    d = (d2[-3:].double() - dz.double()).abs()
    assert (d <= dz.double().abs() * 2.0 ** -7 + 1e-6).all()
