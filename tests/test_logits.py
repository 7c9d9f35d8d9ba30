"""Oracles of the row operators over class logits, and the calls the operators refuse (no GPU needed)."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from logits_cases import INF, rows, teacher
from mlapi_amd.ops import logits as ops
from mlapi_amd.ops import reference as ref


def test_top_oracle_orders_ties_by_class():
    Z = torch.tensor([[1.0, 3.0, 3.0, -INF, 0.0], [-INF] * 5, [float("nan"), -0.0, 0.0, -INF, -1.0]])
    val, idx = ref.top_logits_ref(Z, 4)
    assert idx.tolist() == [[1, 2, 0, 4], [-1] * 4, [1, 2, 4, -1]]
    assert val[0].tolist() == [3.0, 3.0, 1.0, 0.0] and (val[1] == -INF).all()


@pytest.mark.parametrize("alpha", [1.0, 0.3, 0.0])
def test_distill_oracle_matches_autograd(alpha):
    torch.manual_seed(0)
    B, K, k, T = 6, 40, 7, 1.8
    Z = torch.randn(B, K, dtype=torch.float64, requires_grad=True)
    idx, t = teacher(Z, k, 1, dtype=torch.float64)
    y = torch.tensor([3, -1, 0, 39, 5, 5], dtype=torch.int32)
    g = torch.rand(B, dtype=torch.float64)
    loss, dz = ref.distill_ref(Z.detach(), idx, t, temperature=T, alpha=alpha, y=y, g=g)
    total = 0.0
    for r in range(B):
        on = (idx[r] >= 0) & (t[r] > -INF)
        part = Z.sum() * 0
        if on.any():
            q = torch.softmax(t[r][on] / T, 0)
            part = part + alpha * T * T * (q * (q.log() - torch.log_softmax(Z[r] / T, 0)[idx[r][on].long()])).sum()
        if y[r] >= 0:
            part = part - (1 - alpha) * torch.log_softmax(Z[r], 0)[y[r]]
        assert abs(part.item() - loss[r].item()) <= 1e-12
        total = total + g[r] * part
    total.backward()
    assert (Z.grad - dz).abs().max() <= 1e-12


def test_distill_oracle_empty_rows():
    Z = torch.zeros(3, 4)
    Z[1] = -INF
    idx = torch.tensor([[-1, -1], [0, 1], [2, 4]], dtype=torch.int32)
    loss, dz = ref.distill_ref(Z, idx, torch.zeros(3, 2), y=torch.tensor([-1, 0, 0]), alpha=0.5)
    assert loss[:2].tolist() == [0.0, 0.0] and (dz[:2] == 0).all() and loss[2].isnan() and dz[2].isnan().all()


def sample_plainly(z, u, T, k, p, least):
    """The definition, class by class, in Python floats."""
    order = sorted((i for i in range(len(z)) if z[i] > -np.inf), key=lambda i: (-z[i], i))
    if not order:
        return -1, 0.0
    if T == 0:
        return order[0], 1.0
    w = {i: np.exp((z[i] - z[order[0]]) / T) for i in order}
    kept = order[:k] if k > 0 else order
    if p < 1:
        mass, run, nucleus = sum(w[i] for i in kept), 0.0, []
        for n, i in enumerate(kept):
            if n == 0 or run < p * mass:
                nucleus.append(i)
            run += w[i]
        kept = nucleus
    kept = sorted(i for i in kept if w[i] >= least)
    total, run = sum(w[i] for i in kept), 0.0
    for i in kept:
        run += w[i]
        if run > u * total:
            return i, w[i] / total
    return kept[-1], w[kept[-1]] / total


def test_sample_oracle_follows_the_definition():
    rng = np.random.default_rng(0)
    for n in range(200):
        K = int(rng.integers(1, 30))
        z = np.round(rng.standard_normal(K) * 2, int(rng.integers(0, 3))).astype(np.float32)
        if n % 5 == 0:
            z[rng.random(K) < 0.6] = -np.inf
        u = np.float32(rng.random())
        T, k = np.float32(rng.choice([0.0, 0.5, 1.3])), int(rng.choice([0, 1, 3, 40]))
        p, least = np.float32(rng.choice([1.0, 0.6, 0.1])), np.float32(rng.choice([0.0, 0.2]))
        i, q = ref.sample_ref(torch.tensor(z)[None], torch.tensor([u]), temperature=float(T), top_k=k, top_p=float(p),
                              min_p=float(least))
        wi, wq = sample_plainly([float(v) for v in z], float(u), float(T), k, float(p), float(least))
        assert i.item() == wi and abs(q.item() - wq) <= 1e-12, n


def test_rows_cover_what_they_name():
    assert rows(3, 50, torch.float32, 0, "odd").isnan().any() and (rows(3, 50, torch.float16, 0, "masked")[0] == -INF).all()


@pytest.mark.skipif(not (Path("/opt/rocm/bin/hipcc").exists() or shutil.which("hipcc")), reason="needs hipcc")
def test_a_border_between_places_keeps_whole_logits(tmp_path):
    """csrc/tests/order_host.cpp: a filter's border may have a key that no logit has, the one below the zeros' among them."""
    from mlapi_amd import _build

    exe = tmp_path / "order_host"
    src = _build.CSRC / "tests" / "order_host.cpp"
    r = subprocess.run([_build.hipcc(), "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", f"-I{_build.CSRC}", str(src),
                        "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_cpu_tensors_are_refused(native):
    Z = torch.zeros(2, 5)
    with pytest.raises(ValueError, match="GPU"):
        ops.top_logits(Z, 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.sample_logits(Z, torch.zeros(2))
    with pytest.raises(ValueError, match="GPU"):
        ops.distill_loss(Z, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1))


def test_native_calls_refuse_before_any_launch(native):
    """The launchers check sizes on the host: no GPU is touched."""
    with pytest.raises(ValueError, match="1 <= k <= 1024"):
        native.top_logits(1, 0, 10, 4, 10, 1025, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="2\\^20"):
        native.top_logits(1, 0, 1 << 21, 4, 1 << 21, 8, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="row stride"):
        native.top_logits(1, 0, 9, 4, 10, 8, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="f32, bf16 or f16"):
        native.top_logits(0, 0, 10, 4, 10, 8, 0, 0, 0, 0)

    def distill(**kw):
        a = dict(dt=1, t_dt=1, out_dt=1, Z=0, ldz=100, B=4, K=100, idx=0, ldi=8, t=0, ldt=8, k=8, temperature=1.0,
                 alpha=1.0, y=0, g=0, stats_in=0, loss=0, stats_out=0, pred=0, dz=0, ldd=100, ws=0, ws_bytes=1 << 30)
        a.update(kw)
        native.distill(**a)

    for kw, what in ((dict(k=0), "entries"), (dict(K=0), "classes"), (dict(temperature=0.0), "temperature"),
                     (dict(temperature=float("nan")), "temperature"), (dict(alpha=1.5), "alpha"),
                     (dict(alpha=0.5), "labels"), (dict(ldz=99), "stride"), (dict(dz=16, ldd=99), "stride"),
                     (dict(K=200000, ldz=200000, ws_bytes=0), "workspace"), (dict(out_dt=3), "gradient in their type")):
        with pytest.raises(ValueError, match=what):
            distill(**kw)
    with pytest.raises(ValueError, match="2\\^20"):
        native.sample_logits(1, 0, 10, 4, 0, 0, 0, 1.0, 0, 0, 0, 1.0, 0, 0.0, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="stride"):
        native.sample_logits(1, 0, 9, 4, 10, 0, 0, 1.0, 0, 0, 0, 1.0, 0, 0.0, 0, 0, 0, 0)


@pytest.mark.parametrize("K", [1, 50, 40000, 200000, 1 << 20])
def test_no_rows_need_no_workspace(native, K):
    for dt in (1, 2, 3):
        for B in (0, -1):
            assert native.distill_workspace(dt, B, K) == 0
            assert native.top_logits_workspace(dt, B, K, 8) == 0
            assert native.sample_workspace(dt, B, K, False, 8) == 0
    assert native.softmax_distill_workspace(0, K, 128) == 0
    native.distill(dt=1, t_dt=1, out_dt=1, Z=0, ldz=K, B=0, K=K, idx=0, ldi=8, t=0, ldt=8, k=8, temperature=1.0, alpha=1.0,
                   y=0, g=0, stats_in=0, loss=0, stats_out=0, pred=0, dz=0, ldd=K, ws=0, ws_bytes=0)


@pytest.mark.gpu
def test_wrapper_refusals():
    d = "cuda:0"
    Z, u = torch.zeros(3, 20, device=d), torch.zeros(3, device=d)
    idx, t = torch.zeros(3, 4, dtype=torch.int32, device=d), torch.zeros(3, 4, device=d)
    for bad, err in ((Z.double(), TypeError), (Z.long(), TypeError), (Z[0], ValueError), (Z.t(), ValueError),
                     (Z[:, ::2], ValueError), (Z[:1].expand(3, 20), ValueError), (Z[:, :0], ValueError)):
        for call in (lambda z: ops.top_logits(z, 2), lambda z: ops.sample_logits(z, u),
                     lambda z: ops.distill_loss(z, idx, t)):
            with pytest.raises(err):
                call(bad)
    for k in (0, -1, 1025):
        with pytest.raises(ValueError):
            ops.top_logits(Z, k)
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=1.1), dict(top_p=-0.1),
               dict(min_p=2.0), dict(top_p=u[:2]), dict(min_p=u.cpu()), dict(temperature=torch.zeros(6, device=d)[::2])):
        with pytest.raises(ValueError):
            ops.sample_logits(Z, u, **kw)
    with pytest.raises(TypeError):
        ops.sample_logits(Z, u, top_k=u)
    with pytest.raises(TypeError):
        ops.sample_logits(Z, u.double())
    for kw in (dict(temperature=0.0), dict(alpha=-0.1), dict(alpha=0.5), dict(y=idx[:, 0]), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            ops.distill_loss(Z, idx, t, **kw)
    with pytest.raises(ValueError):
        ops.distill_loss(Z, idx, t[:, :3])
    with pytest.raises(TypeError):
        ops.distill_loss(Z, idx.long(), t)
    _, stats = ops.distill_loss(Z, idx, t)
    with pytest.raises(ValueError):
        ops.distill_grad(Z, idx, t, stats[:2])
    big = torch.zeros(100, device=d)
    with pytest.raises(ValueError, match="overlap"):
        ops.distill_grad(big[:60].view(3, 20), idx, t, stats, out=big[4:64].view(3, 20))
    with pytest.raises(ValueError):
        ops.distill_grad(Z, idx, t, stats, out=torch.zeros(3, 20, dtype=torch.float16, device=d))
    with pytest.raises(ValueError, match="overlaps"):
        ops.sample_logits(Z, u, out=(torch.zeros(3, dtype=torch.int32, device=d), u))
    k = torch.ones(3, dtype=torch.int32, device=d)
    with pytest.raises(ValueError, match="overlaps"):
        ops.sample_logits(Z, u, top_k=k, out=(k, torch.zeros(3, device=d)))
    with pytest.raises(ValueError, match="overlaps"):
        ops.top_logits(Z, 2, out=(Z.view(-1)[:6].view(3, 2), torch.zeros(3, 2, dtype=torch.int32, device=d)))
    with pytest.raises(ValueError, match="overlaps"):
        ops.distill_loss_grad(Z, idx, t, y=k, pred=k)
    with pytest.raises(ValueError):
        ops.sample_logits(Z, u, temperature=float("inf"))
    with pytest.raises(ValueError):
        ops.top_logits(Z, 2, out=(torch.zeros(3, 2, device=d), torch.zeros(3, 2, device=d)))
