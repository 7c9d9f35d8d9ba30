"""The row operators over class logits: their measured cases, inputs and plain forms.

A row holds one sample's class logits (a classifier's scores, a language model's vocabulary). Three operators
read such rows, and a run of them trains and uses a student: ``top_logits`` writes down a teacher's k largest
logits, ``distill_*`` gives the student's loss and gradient against them, ``sample_logits`` draws the answer.
``run`` computes the plain form with elementary torch operations, or, where ``own`` is true, calls
:mod:`mlapi_amd.ops.logits`.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------ cases
def listed():
    """1000 classes are this repository's multiclass workload (serving batches of 64, training batches of
    65536 rows); 40 its middle one; the long rows are vocabularies, at round and at odd sizes."""
    return [
        # a served batch's eight best classes: latency
        dict(name="top served batch", op="top", rows=64, classes=1000, k=8, dtype="f32", pad=0, masked=0.0),
        # a teacher labels a training batch
        dict(name="top training batch", op="top", rows=65536, classes=1000, k=16, dtype="f32", pad=0, masked=0.0),
        # a language model's teacher labels the positions of a few sequences
        dict(name="top vocabulary", op="top", rows=1023, classes=131072, k=64, dtype="bf16", pad=0, masked=0.0),
        # a small student's step: latency
        dict(name="distill small step", op="distill", rows=512, classes=40, k=5, dtype="f32", pad=0, masked=0.0,
             temperature=2.0, alpha=1.0, form="both"),
        # the training batch, soft and hard targets mixed
        dict(name="distill training batch", op="distill", rows=65536, classes=1000, k=16, dtype="f32", pad=0,
             masked=0.0, temperature=2.0, alpha=0.5, form="both"),
        # forward, then backward with the weights of the positions, as a model's own backward pass calls them
        dict(name="distill vocabulary", op="distill", rows=2048, classes=65536, k=64, dtype="bf16", pad=0, masked=0.0,
             temperature=1.0, alpha=1.0, form="apart"),
        # few long rows: the row is the only axis left to share
        dict(name="distill few long rows", op="distill", rows=7, classes=200001, k=33, dtype="f32", pad=0, masked=0.0,
             temperature=1.5, alpha=1.0, form="both"),
        # odd rows inside a padded buffer, some classes masked
        dict(name="distill ragged", op="distill", rows=1501, classes=32003, k=100, dtype="f16", pad=5, masked=0.1,
             temperature=3.0, alpha=0.7, form="both"),
        # one sequence's next token
        dict(name="sample one", op="sample", rows=1, classes=131072, dtype="f32", pad=0, masked=0.0, filters="fixed",
             temperature=0.8, top_k=50, top_p=0.95, min_p=0.0),
        # a decoding batch, nucleus only
        dict(name="sample nucleus", op="sample", rows=256, classes=65537, dtype="bf16", pad=0, masked=0.0,
             filters="fixed", temperature=1.0, top_k=0, top_p=0.9, min_p=0.0),
        # answers drawn for a whole training batch
        dict(name="sample training batch", op="sample", rows=65536, classes=1000, dtype="f32", pad=0, masked=0.0,
             filters="fixed", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0),
        # a served batch whose requests each bring their own settings
        dict(name="sample served batch", op="sample", rows=64, classes=1000, dtype="f32", pad=0, masked=0.2,
             filters="rows", temperature=0.0, top_k=0, top_p=0.0, min_p=0.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Any operator on 1 to 65536 rows of 2 to 262144 classes, at most 2^26 logits in all."""
    classes = _log_uniform(rng, 2, 262144)
    rows = _log_uniform(rng, 1, max(1, min(65536, (1 << 26) // classes)))
    case = dict(op=rng.choice(["top", "distill", "distill", "sample", "sample"]), rows=rows, classes=classes,
                dtype=rng.choice(["f32", "bf16", "f16"]), pad=rng.choice([0, 0, 1, 8, 13]),
                masked=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if case["op"] != "sample":
        case["k"] = min(_log_uniform(rng, 1, 256), classes)
    if case["op"] == "distill":
        case.update(temperature=round(rng.uniform(0.5, 4.0), 2), alpha=rng.choice([1.0, round(rng.uniform(0.1, 0.9), 2)]),
                    form=rng.choice(["both", "apart"]))
    if case["op"] == "sample":
        case.update(filters=rng.choice(["fixed", "rows"]), temperature=round(rng.uniform(0.3, 1.5), 2),
                    top_k=rng.choice([0, min(_log_uniform(rng, 1, 1024), classes)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.5, 0.99), 2)]),
                    min_p=rng.choice([0.0, round(rng.uniform(0.01, 0.2), 2)]))
    return case


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    """Logits as a classifier gives them: a bell of scores with one class of every row raised by 0 to 12, so
    some rows are nearly flat and some nearly certain. The teacher's list is the top of a noisy copy; some
    rows' lists are short (classes of -1), a few are empty, and where classes are masked (-inf) a few rows
    are masked throughout."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, K, dt = case["rows"], case["classes"], _TYPES[case["dtype"]]
    rand = lambda *shape: torch.rand(*shape, generator=g, device="cuda")  # noqa: E731
    Z32 = torch.randn(B, K, generator=g, device="cuda").mul_(2.0)
    best = torch.randint(0, K, (B, 1), generator=g, device="cuda")
    Z32.scatter_add_(1, best, rand(B, 1) * 12)
    row = torch.arange(B, device="cuda")
    if case["masked"]:
        hidden = rand(K) < case["masked"]
        hidden[0] = False
        Z32.masked_fill_(hidden, -math.inf)
        Z32[row % 97 == 96] = -math.inf
    store = torch.empty(B, K + case["pad"], dtype=dt, device="cuda")
    Z = store[:, :K]
    Z.copy_(Z32)
    s = dict(case=case, Z=Z)
    if case["op"] == "distill":
        k = case["k"]
        t, idx = torch.topk(Z32.add_(torch.randn(B, K, generator=g, device="cuda"), alpha=0.7), k, dim=1)
        full = torch.where(row % 64 == 5, 0, torch.where(row % 16 == 3, (k + 1) // 2, k))[:, None]
        gone = (torch.arange(k, device="cuda") >= full) | (t == -math.inf)
        s["idx"] = torch.where(gone, -1, idx).to(torch.int32)
        s["t"] = torch.where(gone, -math.inf, t).to(dt)
        s["y"] = None
        if case["alpha"] != 1.0:
            y = torch.where(rand(B, 1) < 0.8, best, torch.randint(0, K, (B, 1), generator=g, device="cuda"))
            if case["masked"]:
                y = torch.where(hidden[y], 0, y)
            s["y"] = torch.where(row % 32 == 7, -1, y[:, 0]).to(torch.int32)
        s["g"] = rand(B) / B if case["form"] == "apart" else None
    if case["op"] == "sample":
        s["u"] = rand(B)
        s["set"] = {n: case[n] for n in ("temperature", "top_k", "top_p", "min_p")}
        if case["filters"] == "rows":
            k = torch.exp(rand(B) * math.log(min(K, 1024))).to(torch.int32)
            s["set"] = dict(temperature=torch.where(row % 16 == 1, 0.0, 0.4 + rand(B)),
                            top_k=torch.where(rand(B) < 0.3, 0, k).to(torch.int32),
                            top_p=torch.where(rand(B) < 0.3, 1.0, 0.6 + 0.4 * rand(B)),
                            min_p=torch.where(rand(B) < 0.5, 0.0, 0.1 * rand(B)))
    return s


# ------------------------------------------------------------------------------------ plain forms
def _order_keys(Z):
    """int64 keys that order the classes of a row: larger logit first, then lower class; masked ones last."""
    x = Z.float() + 0.0
    x = torch.where(x.isnan(), -math.inf, x)
    bits = x.view(torch.int32).long()
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    return (bits << 32) - torch.arange(Z.shape[1], device=Z.device)


def _plain_top(s):
    Z, k = s["Z"], s["case"]["k"]
    idx = torch.topk(_order_keys(Z), k, dim=1).indices
    v = Z.gather(1, idx)
    gone = v == -math.inf
    return v, torch.where(gone, -1, idx).to(torch.int32)


def _log_softmax_parts(x):
    """x minus its row maximum, and the logarithm of the sum of its exponentials (rows without any: 0)."""
    m = x.amax(1, keepdim=True)
    d = x - torch.where(m == -math.inf, 0.0, m)
    total = torch.exp(d).sum(1, keepdim=True)
    return d, torch.where(total > 0, total, 1.0).log()


def _plain_distill(s):
    c, Z, idx = s["case"], s["Z"].float(), s["idx"].long()
    T, alpha = c["temperature"], c["alpha"]
    some = (Z > -math.inf).any(1, keepdim=True)
    there = (idx >= 0) & (s["t"] > -math.inf) & some
    at = idx.clamp(min=0)
    d, ln = _log_softmax_parts(torch.where(there, s["t"].float() / T, -math.inf))
    q = torch.exp(d - ln) * there
    D, LN = _log_softmax_parts(Z / T)
    off = torch.where(there, d - ln - (D.gather(1, at) - LN), 0.0)
    loss = alpha * T * T * (q * off).sum(1)
    dz = torch.exp(D - LN) * q.sum(1, keepdim=True)
    dz.scatter_add_(1, at, -q)
    dz *= alpha * T
    if s["y"] is not None:
        y = s["y"].long()[:, None]
        hard = (y >= 0) & some
        at = y.clamp(min=0)
        D, LN = _log_softmax_parts(Z)
        loss += (1 - alpha) * torch.where(hard, LN - D.gather(1, at), 0.0)[:, 0]
        h = torch.exp(D - LN)
        h.scatter_add_(1, at, torch.full_like(LN, -1.0))
        dz += (1 - alpha) * torch.where(hard, h, 0.0)
    if s["g"] is not None:
        dz *= s["g"][:, None]
    return loss, dz.to(s["Z"].dtype)


def _column(v, like):
    """A setting as a [rows, 1] column in 64 bits, through the 32 that the operator takes."""
    v = v.float() if isinstance(v, torch.Tensor) else torch.full((like.shape[0],), float(v), device=like.device)
    return v.double()[:, None]


def _plain_sample(s):
    """In 64 bits: a draw next to a border between two classes must fall on the same side."""
    Z, K = s["Z"], s["Z"].shape[1]
    T, k, p, least = (_column(s["set"][n], Z) for n in ("temperature", "top_k", "top_p", "min_p"))
    order = torch.sort(_order_keys(Z), dim=1, descending=True).indices
    z = Z.double().gather(1, order)
    top = z[:, :1]
    w = torch.where(z == top, 1.0, torch.exp((z - top) / T)) * (z > -math.inf)
    rank = torch.arange(K, device=Z.device)
    w *= (rank < k) | (k <= 0)
    w *= (rank < 1) | (T > 0)
    mass = w.cumsum(1)
    before = torch.cat([torch.zeros_like(top), mass[:, :-1]], 1)
    w *= (before < p * mass[:, -1:]) | (rank < 1) | (p >= 1)
    w *= w >= least
    w = torch.zeros_like(w).scatter_(1, order, w)
    mass = w.cumsum(1)
    total = mass[:, -1:]
    idx = (mass <= s["u"].double()[:, None] * total).sum(1).clamp(max=K - 1)
    prob = w.gather(1, idx[:, None]) / total
    none = total[:, 0] == 0
    return torch.where(none, -1, idx).to(torch.int32), torch.where(none, 0.0, prob[:, 0]).float()


def run(s):
    c = s["case"]
    if not own:
        return {"top": _plain_top, "distill": _plain_distill, "sample": _plain_sample}[c["op"]](s)
    from mlapi_amd.ops import logits as ops

    if c["op"] == "top":
        return ops.top_logits(s["Z"], c["k"])
    if c["op"] == "sample":
        return ops.sample_logits(s["Z"], s["u"], **s["set"])
    how = dict(temperature=c["temperature"], alpha=c["alpha"], y=s["y"])
    if c["form"] == "both":
        return ops.distill_loss_grad(s["Z"], s["idx"], s["t"], **how)
    loss, stats = ops.distill_loss(s["Z"], s["idx"], s["t"], **how)
    return loss, ops.distill_grad(s["Z"], s["idx"], s["t"], stats, g=s["g"], **how)


# ------------------------------------------------------------------------------------------- work
def work(case):
    """Logits read once (twice where backward is a call of its own), lists and results once. Operations per
    logit: a comparison for the top, maximum / difference / scale / exponential / sum for a softmax, two more
    for its gradient."""
    B, K, e = case["rows"], case["classes"], _BYTES[case["dtype"]]
    n = B * K
    if case["op"] == "top":
        return {"bytes": n * e + B * case["k"] * (e + 4), "flops": n}
    if case["op"] == "sample":
        return {"bytes": n * e + B * (4 + 8 + (16 if case["filters"] == "rows" else 0)), "flops": 6 * n}
    softs = 2 if case["alpha"] != 1.0 else 1
    reads = 2 if case["form"] == "apart" else 1
    lists = B * (case["k"] * (e + 4) * reads + 4 + 4 * (softs - 1) * reads + 4 * (reads - 1))
    return {"bytes": n * e * (reads + 1) + lists, "flops": 7 * n * softs}


# ------------------------------------------------------------------------------------------ exact
def _exact_top(s):
    Z, k = s["Z"].double(), s["case"]["k"]
    v, i = torch.sort(torch.where(Z.isnan(), -math.inf, Z), dim=1, descending=True, stable=True)
    v, i = v[:, :k].contiguous(), i[:, :k]
    return v, torch.where(v == -math.inf, -1, i).to(torch.int32)


def _exact_distill(s):
    """Dense target distributions: loss = sum q ln(q / p), gradient = p - q, all over K classes."""
    c, Z = s["case"], s["Z"].double()
    T, alpha, (B, K) = c["temperature"], c["alpha"], Z.shape
    live = torch.isfinite(Z).any(1)
    w = torch.exp(s["t"].double() / T - (s["t"].double() / T).amax(1, keepdim=True).clamp(min=-1e300))
    w = torch.where((s["idx"] >= 0) & live[:, None], w, 0.0)
    Q = torch.zeros(B, K, dtype=torch.float64, device=Z.device)
    r, j = (s["idx"] >= 0).nonzero(as_tuple=True)
    total = w.sum(1, keepdim=True)
    w = torch.where(total > 0, w / total, 0.0)
    Q.index_put_((r, s["idx"][r, j].long()), w[r, j], accumulate=True)
    ent = torch.where(w > 0, w * w.clamp(min=1e-300).log(), 0.0).sum(1)

    def part(x, target):
        x = torch.where(live[:, None], x, 0.0)
        lse = torch.logsumexp(x, 1, keepdim=True)
        lp = x - lse
        cross = -torch.where(target > 0, target * lp, 0.0).sum(1)
        return cross, torch.exp(lp) * target.sum(1, keepdim=True) - target

    cross, dz = part(Z / T, Q)
    loss, dz = alpha * T * T * (cross + ent), alpha * T * dz
    if s["y"] is not None:
        Y = torch.zeros_like(Q)
        r = ((s["y"] >= 0) & live).nonzero()[:, 0]
        Y[r, s["y"][r].long()] = 1.0
        cross, h = part(Z, Y)
        loss, dz = loss + (1 - alpha) * cross, dz + (1 - alpha) * h
    return loss, dz if s["g"] is None else dz * s["g"].double()[:, None]


def _exact_sample_rows(Z, u, T, k, p, least):
    B, K = Z.shape
    Z = torch.where(Z.isnan(), -math.inf, Z)
    m = Z.amax(1, keepdim=True)
    live = m > -math.inf
    x = torch.where(Z == m, 0.0, (Z - torch.where(live, m, 0.0)) / T.clamp(min=1e-300))
    e = torch.where(live & (Z > -math.inf), torch.exp(x), 0.0)
    v, perm = torch.sort(Z, dim=1, descending=True, stable=True)
    place = torch.empty_like(perm).scatter_(1, perm, torch.arange(K, device=Z.device).expand(B, K).contiguous())
    keep = place < torch.where(k > 0, k, K).long()
    keep &= (place == 0) | (T > 0)
    run = torch.where(keep, e, 0.0).gather(1, perm).cumsum(1)
    lead = torch.nn.functional.pad(run, (1, 0))[:, :-1].gather(1, place)
    keep &= (place == 0) | (p >= 1) | (lead < p * run[:, -1:])
    keep &= e >= least
    e = torch.where(keep, e, 0.0)
    total = e.sum(1)
    c = e.cumsum(1)
    idx = torch.searchsorted(c, (u[:, None] * c[:, -1:]).contiguous(), right=True)[:, 0].clamp(max=K - 1)
    prob = e.gather(1, idx[:, None])[:, 0] / torch.where(total > 0, total, 1.0)
    return torch.where(total > 0, idx, -1).to(torch.int32), torch.where(total > 0, prob, 0.0)


def _exact_sample(s):
    Z = s["Z"]
    B, step = Z.shape[0], max(1, (1 << 25) // Z.shape[1])
    cols = [_column(s["set"][n], Z) for n in ("temperature", "top_k", "top_p", "min_p")]
    parts = [_exact_sample_rows(Z[a:a + step].double(), s["u"][a:a + step].double(), *(v[a:a + step] for v in cols))
             for a in range(0, B, step)]
    return torch.cat([x[0] for x in parts]), torch.cat([x[1] for x in parts])


def exact(case, seed):
    s = prepare(case, seed)
    return {"top": _exact_top, "distill": _exact_distill, "sample": _exact_sample}[case["op"]](s)
