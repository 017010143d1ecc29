"""Operators for learned buckets, as cases that can be prepared, run and compared: layer norm, routing with a balance loss,
Newton-Schulz orthogonalisation and the Muon step.

  norm    layer norm of rows of features, forward (y, mean, 1 / deviation) or backward (dx, dweight, dbias)
  route   top-k choice of a bucket (expert) per row with gates, counts, balance and z loss, forward or backward
  orth    Newton-Schulz orthogonalisation of a batch of matrices
  muon    momentum, orthogonalisation and weight update of a batch of matrices

With `own` false, `run` computes them by elementary torch operations in 32 bits, rounded once at the end; with `own` true by the
library.  `exact` computes them in 64 bits.  A case is a dict of plain values; `listed()` holds the ones that are always measured,
`draw(rng)` gives more of the same ranges.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
NORM_EPS, ORTH_EPS = 1e-5, 1e-7
LR, BETA, DECAY, CLIP = 0.02, 0.95, 0.01, 127.0 / 64.0  # the clip is the trainer's for hidden weights


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # a validation batch's feature rows in front of a gate: the smallest call, where launches count
        dict(kind="norm", back=False, dtype="f32", rows=256, n=256, strided=False, name="norm_fwd_256x256"),
        # feature rows of a full batch of the widest net
        dict(kind="norm", back=False, dtype="f32", rows=65536, n=1536, strided=False, name="norm_fwd_65536x1536"),
        # a ragged batch in the 16-bit mode, one perspective's columns of a wider buffer
        dict(kind="norm", back=False, dtype="f16", rows=10000, n=1000, strided=True, name="norm_fwd_10000x1000_f16"),
        # the backward pass of a full batch of the widest net
        dict(kind="norm", back=True, dtype="f32", rows=65536, n=1536, strided=False, name="norm_bwd_65536x1536"),
        # ... of the mid-size net's batch in the 16-bit mode
        dict(kind="norm", back=True, dtype="f16", rows=16384, n=768, strided=False, name="norm_bwd_16384x768_f16"),
        # one bucket of nine for every position of a full batch, as the trainer takes it
        dict(kind="route", back=False, dtype="f32", rows=65536, experts=9, k=1, renormalise=False, padding=0.0, forbidden=0.0, name="route_fwd_65536x9"),
        # a wide mixture in 16 bits with padding rows and experts that some rows may not choose
        dict(kind="route", back=False, dtype="bf16", rows=40000, experts=256, k=8, renormalise=True, padding=0.1, forbidden=0.05, name="route_fwd_40000x256_k8"),
        # the gate's gradient for two of nine buckets, a large ragged batch
        dict(kind="route", back=True, dtype="f32", rows=50001, experts=9, k=2, renormalise=True, padding=0.05, forbidden=0.0, name="route_bwd_50001x9"),
        # the first hidden layer of the LayerStack net: nine buckets' small matrices, a latency chain
        dict(kind="orth", dtype="f32", batch=9, rows=16, cols=1536, name="orth_9x16x1536"),
        # a batch of half-precision gradients of ordinary hidden matrices, odd sizes
        dict(kind="orth", dtype="bf16", batch=4, rows=1000, cols=777, name="orth_4x1000x777_bf16"),
        # the Simple net's first hidden layer, stored inputs first
        dict(kind="muon", dtype="f32", batch=1, rows=1024, cols=32, nesterov=True, name="muon_1024x32"),
        # a large hidden matrix in fp32
        dict(kind="muon", dtype="f32", batch=1, rows=4096, cols=4096, nesterov=True, name="muon_4096x4096"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "route", "orth", "muon"])
    dtype = rng.choice(["f32", "f32", "f16", "bf16"])
    if kind == "norm":
        n = _log(rng, 8, 6144)
        rows = _log(rng, 1, min(65536, 65536 * 1536 // n))
        return dict(kind=kind, back=rng.random() < 0.5, dtype=dtype, rows=rows, n=n, strided=rng.random() < 0.3)
    if kind == "route":
        experts = _log(rng, 2, 512)
        return dict(kind=kind, back=rng.random() < 0.5, dtype=dtype, rows=_log(rng, 1, min(262144, (1 << 24) // experts)), experts=experts,
                    k=rng.randint(1, min(8, experts)), renormalise=rng.random() < 0.5, padding=rng.choice([0.0, 0.1, 0.5]),
                    forbidden=rng.choice([0.0, 0.0, 0.1]))
    batch, rows, cols = _log(rng, 1, 16), _log(rng, 1, 4096), _log(rng, 1, 4096)
    while batch * rows * cols > 4096 * 4096:
        batch = max(1, batch // 2)
    case = dict(kind=kind, dtype=dtype, batch=batch, rows=rows, cols=cols)
    return dict(case, nesterov=rng.random() < 0.5) if kind == "muon" else case


# ---- inputs ------------------------------------------------------------------------------------------------------
def _gradients(case, g):
    """Matrices as gradients are: a few strong directions over a floor of noise, scales that differ from matrix to matrix."""
    b, r, c = case["batch"], case["rows"], case["cols"]
    rank = min(r, c, 24)
    decay = 0.8 ** torch.arange(rank, device="cuda")
    left, right = (torch.randn(b, d, rank, generator=g, device="cuda") for d in (r, c))
    x = (left * decay) @ right.transpose(1, 2) + torch.randn(b, r, c, generator=g, device="cuda")
    return (x * 1e-3 * torch.rand(b, 1, 1, generator=g, device="cuda").add_(0.5)).to(TYPES[case["dtype"]])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kind = case["kind"]
    s = dict(case=case)
    if kind == "norm":
        rows, n, t = case["rows"], case["n"], TYPES[case["dtype"]]
        # clipped activations with an offset and a scale of their own in every row; strided: the first columns of a wider buffer
        x = (rand(rows, 2 * n if case["strided"] else n) * torch.rand(rows, 1, generator=g, device="cuda").add_(0.2) + 0.5).clamp_(-1, 2).to(t)
        s["x"] = x[:, :n]
        s["weight"], s["bias"] = 1 + 0.1 * rand(n), 0.1 * rand(n)
        if case["back"]:
            s["dy"] = (rand(rows, n) * 1e-2).to(t)
            s["mean"], s["rstd"] = _norm_statistics(s["x"])
    elif kind == "route":
        rows, e, t = case["rows"], case["experts"], TYPES[case["dtype"]]
        x = rand(rows, e) + 0.5 * rand(e)
        if case["forbidden"]:
            x = x.masked_fill(torch.rand(rows, e, generator=g, device="cuda") < case["forbidden"], -math.inf)
        s["logits"] = x.to(t)
        s["mask"] = torch.rand(rows, generator=g, device="cuda") >= case["padding"] if case["padding"] else None
        if case["back"]:
            s["forward"] = _plain_route(s["logits"], case["k"], case["renormalise"], s["mask"])
            s["dgate"] = 1e-2 * rand(rows, case["k"])
            s["dlosses"] = torch.tensor([1e-2, 1e-3], device="cuda")
    else:
        s["grad"] = _gradients(case, g)
        if kind == "muon":
            s["weight"] = 0.02 * rand(case["batch"], case["rows"], case["cols"])
            s["momentum"] = 5 * _gradients(dict(case, dtype="f32"), g)
            s["weight_out"], s["momentum_out"] = torch.empty_like(s["weight"]), torch.empty_like(s["momentum"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _norm_statistics(x):
    x = x.float()
    mean = x.mean(1)
    return mean, 1 / ((x - mean[:, None]).square().mean(1) + NORM_EPS).sqrt()


def _plain_norm(s):
    x = s["x"].float()
    if not s["case"]["back"]:
        mean, rstd = _norm_statistics(x)
        y = (x - mean[:, None]) * rstd[:, None] * s["weight"] + s["bias"]
        return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xh = (x - s["mean"][:, None]) * rstd
    t = dy * s["weight"]
    dx = rstd * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum(0), "dbias": dy.sum(0)}


def _softmax_rows(logits, mask):
    """Probabilities and log-sum-exp, zero in rows that are masked or have no expert to choose, and which rows are not."""
    x = logits.float()
    best = x.amax(1, keepdim=True)
    live = best > -math.inf
    if mask is not None:
        live = live & mask[:, None]
    best = torch.where(live, best, 0)
    e = torch.where(live, (x - best).exp(), 0)
    total = torch.where(live, e.sum(1, keepdim=True), 1)
    return e / total, torch.where(live, best + total.log(), 0), live


def _plain_route(logits, k, renormalise, mask):
    experts = logits.shape[1]
    p, lse, live = _softmax_rows(logits, mask)
    chosen, order = logits.float().sort(dim=1, descending=True, stable=True)
    chosen, order = chosen[:, :k], order[:, :k]
    ok = live & (chosen > -math.inf)
    if renormalise:
        e = torch.where(ok, (chosen - chosen[:, :1]).exp(), 0)
        gate = torch.where(ok, e / e.sum(1, keepdim=True), 0)
    else:
        gate = torch.where(ok, p.gather(1, order), 0)
    counts = torch.zeros(experts + 1, dtype=torch.int32, device=logits.device)
    counts.index_add_(0, torch.where(ok, order, experts).flatten(), torch.ones_like(order, dtype=torch.int32).flatten())
    counts = counts[:experts]
    rows = live.sum().to(torch.int32)
    n = rows.clamp(min=1).float()
    prob_mean = p.sum(0) / n
    losses = torch.stack([experts / (n * k) * (counts.float() * prob_mean).sum(), lse.square().sum() / n])
    return {"index": torch.where(ok, order, -1).to(torch.int32), "gate": gate, "counts": counts, "rows": rows.reshape(1),
            "prob_mean": prob_mean, "losses": losses}


def _plain_route_backward(s):
    case, f, dgate = s["case"], s["forward"], s["dgate"]
    p, lse, live = _softmax_rows(s["logits"], s["mask"])
    n = f["rows"].clamp(min=1).float()
    h = s["dlosses"][0] * p.shape[1] / (n * case["k"]) / n * f["counts"].float()
    d = p * (h - (p * h).sum(1, keepdim=True) + s["dlosses"][1] * 2 * lse / n)
    ok = f["index"] >= 0
    total = (f["gate"] * dgate).sum(1, keepdim=True)
    part = torch.where(ok, f["gate"] * (dgate - total if case["renormalise"] else dgate), 0)
    if not case["renormalise"]:
        d = d - p * total
    d = d.scatter_add(1, f["index"].clamp(min=0).long(), part)
    return torch.where(live, d, 0).to(s["logits"].dtype)


def _plain_orthogonalise(u):
    x = u.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + ORTH_EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        g = x @ x.transpose(1, 2)
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.transpose(1, 2) if tall else x


def _scale(case):
    return math.sqrt(max(1.0, case["rows"] / case["cols"]))


def _plain_muon(s):
    case = s["case"]
    grad = s["grad"].float()
    m = BETA * s["momentum"] + grad
    o = _plain_orthogonalise(grad + BETA * m if case["nesterov"] else m)
    w = (s["weight"] * (1 - LR * DECAY) - LR * _scale(case) * o).clamp(-CLIP, CLIP)
    return {"weight": w, "momentum": m}


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "norm":
            return _plain_norm(s)
        if kind == "route":
            return {"dlogits": _plain_route_backward(s)} if case["back"] else _plain_route(s["logits"], case["k"], case["renormalise"], s["mask"])
        return _plain_muon(s) if kind == "muon" else {"out": _plain_orthogonalise(s["grad"]).to(s["grad"].dtype)}
    from tatara_b200 import ops
    if kind == "norm":
        if case["back"]:
            dx, dweight, dbias = ops.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
            return {"dx": dx, "dweight": dweight, "dbias": dbias}
        y, mean, rstd = ops.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=NORM_EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    if kind == "route":
        if case["back"]:
            f = s["forward"]
            return {"dlogits": ops.route_backward(s["logits"], ops.Routing(f["index"], f["gate"], f["counts"], f["rows"], f["prob_mean"], f["losses"]),
                                                  s["dgate"], s["dlosses"], renormalise=case["renormalise"], mask=s["mask"])}
        return ops.route_forward(s["logits"], case["k"], renormalise=case["renormalise"], mask=s["mask"])._asdict()
    if kind == "orth":
        return {"out": ops.orthogonalise(s["grad"], steps=STEPS, coefficients=COEFFICIENTS, eps=ORTH_EPS)}
    w, m = ops.muon_step(s["weight"], s["momentum"], s["grad"], lr=LR, beta=BETA, nesterov=case["nesterov"], weight_decay=DECAY,
                         scale=_scale(case), clip=CLIP, steps=STEPS, coefficients=COEFFICIENTS, eps=ORTH_EPS,
                         weight_out=s["weight_out"], momentum_out=s["momentum_out"])
    return {"weight": w, "momentum": m}


# ---- in 64 bits --------------------------------------------------------------------------------------------------
def _exact_orthogonalise(u):
    """Newton-Schulz as a polynomial of the Gram matrix, applied once to the normalised matrix."""
    wide = u if u.shape[-2] <= u.shape[-1] else u.mT
    wide = wide / (torch.linalg.vector_norm(wide, dim=(-2, -1), keepdim=True) + ORTH_EPS)
    gram = torch.bmm(wide, wide.mT)
    eye = torch.eye(gram.shape[-1], dtype=torch.float64, device=u.device)
    poly = eye.expand_as(gram)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        q = a * eye + torch.bmm(gram, b * eye + c * gram)
        poly, gram = torch.bmm(q, poly), torch.bmm(torch.bmm(q, gram), q)
    out = torch.bmm(poly, wide)
    return out if u.shape[-2] <= u.shape[-1] else out.mT


def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in prepare(case, seed).items() if not k.endswith("_out")}
    if case["kind"] == "norm":
        x, n = s["x"], case["n"]
        if not case["back"]:
            var, mean = torch.var_mean(x, 1, correction=0)
            r = (var + NORM_EPS).rsqrt()
            return {"y": torch.addcmul(s["bias"], torch.einsum("ij,i,j->ij", x - mean[:, None], r, torch.ones_like(s["weight"])), s["weight"]), "mean": mean, "rstd": r}
        xh = torch.einsum("ij,i->ij", x - s["mean"][:, None], s["rstd"])
        t = torch.einsum("ij,j->ij", s["dy"], s["weight"])
        along = torch.einsum("ij,ij->i", t, xh) / n
        dx = torch.einsum("ij,i->ij", t - t.sum(1, keepdim=True) / n - torch.einsum("i,ij->ij", along, xh), s["rstd"])
        return {"dx": dx, "dweight": torch.einsum("ij,ij->j", s["dy"], xh), "dbias": s["dy"].sum(0)}
    if case["kind"] == "route":
        x, k, experts = s["logits"], case["k"], case["experts"]
        live = torch.isfinite(x).any(1)
        if s["mask"] is not None:
            live &= s["mask"]
        n = max(1, int(live.sum()))
        p, lse = torch.zeros_like(x), torch.zeros(len(x), dtype=torch.float64, device=x.device)
        p[live], lse[live] = torch.softmax(x[live], 1), torch.logsumexp(x[live], 1)
        if not case["back"]:
            index = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
            ok = live[:, None] & torch.isfinite(x.gather(1, index))
            gate = p.gather(1, index) * ok
            if case["renormalise"]:
                gate = gate / gate.sum(1, keepdim=True).clamp(min=1e-300)
            counts = torch.bincount(index[ok], minlength=experts).double()
            mean = p.sum(0) / n
            return {"index": None, "gate": gate, "counts": None, "rows": None, "prob_mean": mean,
                    "losses": torch.stack([experts * torch.dot(counts / (n * k), mean), torch.dot(lse, lse) / n])}
        # the derivative along every softmax, from what the forward pass chose
        index, chosen = s["forward"]["index"].long(), s["forward"]["index"] >= 0
        dp = torch.zeros_like(x) + s["dlosses"][0] * experts * s["forward"]["counts"] / (n * k) / n
        extra = torch.zeros_like(x)
        if case["renormalise"]:
            g = torch.softmax(torch.where(chosen, x.gather(1, index.clamp(min=0)), -1e300), 1) * chosen
            extra.scatter_add_(1, index.clamp(min=0), g * (s["dgate"] - (g * s["dgate"]).sum(1, keepdim=True)) * chosen)
        else:
            dp = dp.scatter_add(1, index.clamp(min=0), s["dgate"] * chosen)
        d = p * (dp - torch.einsum("ij,ij->i", p, dp)[:, None]) + extra + (2 * s["dlosses"][1] / n) * lse[:, None] * p
        return {"dlogits": d * live[:, None]}
    if case["kind"] == "orth":
        return {"out": _exact_orthogonalise(s["grad"])}
    m = torch.add(s["grad"], s["momentum"], alpha=BETA)
    o = _exact_orthogonalise(torch.add(s["grad"], m, alpha=BETA) if case["nesterov"] else m)
    return {"weight": torch.clamp(torch.add(s["weight"] * (1 - LR * DECAY), o, alpha=-LR * _scale(case)), -CLIP, CLIP), "momentum": m}


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    size = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        # forward: x in, y out, mean and rstd out; backward: x, dy, mean, rstd in, dx out; weight and bias, or weight and both gradients
        return {"bytes": (3 if case["back"] else 2) * rows * n * size + 8 * rows + (12 if case["back"] else 8) * n,
                "flops": (14 if case["back"] else 8) * rows * n}
    if case["kind"] == "route":
        rows, e, k = case["rows"], case["experts"], case["k"]
        mask = rows if case["padding"] else 0
        if case["back"]:  # logits, index, gate, dgate in, dlogits out
            return {"bytes": 2 * rows * e * size + 12 * rows * k + mask, "flops": 12 * rows * e}
        return {"bytes": rows * e * size + 8 * rows * k + mask + 8 * e, "flops": (8 + k) * rows * e}
    b, n, m = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # a step: the Gram matrix and its square are symmetric, so half of each is computed, and the product with the matrix
    flops = b * STEPS * (n * n * m + n ** 3 + 2 * n * n * m)
    bytes_ = b * n * m * (2 * size if case["kind"] == "orth" else size + 16)
    return {"bytes": bytes_, "flops": flops}
