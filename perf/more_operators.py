"""Operators around a router and its experts, as cases that can be prepared, run and compared: root-mean-square norm with the residual's
addition and an 8-bit output, rows sorted by expert and back, embedding rows and their gradient by sorted tokens.

  rms     root-mean-square norm of x, or of the sum of x and a residual: forward (y, the sum, 1 / rms), forward with an output of 8 bits and
          scales, or backward (dx, dweight)
  order   a router's choices sorted by expert: where every choice goes, which choice every place holds, where every expert begins
  send    rows to the places of their experts
  join    rows back from their places, summed by their gates (or plainly, which is the gradient of `send`); backward: the places' rows and the gates
  look    rows of a table by token, scaled
  learn   the gradient of a table from the rows of its tokens

With `own` false, `run` computes them by elementary torch operations in 32 bits, rounded once at the end; with `own` true by the
library.  `exact` computes them in 64 bits.  A case is a dict of plain values; `listed()` holds the ones that are always measured,
`draw(rng)` gives more of the same ranges.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
RMS_EPS = 1e-6
E4M3_MOST, LEAST_SCALE = 448.0, 2.0 ** -126
FEATURES = 73305  # rows of the halfka-hm-merged feature table


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of positions that are evaluated as they come: the smallest call, where launches count
        dict(kind="rms", back=False, dtype="bf16", rows=16, n=1536, residual=True, group=None, strided=False, name="rms_16x1536_bf16"),
        # feature rows of a full batch of the widest net on their residual stream
        dict(kind="rms", back=False, dtype="bf16", rows=65536, n=1536, residual=True, group=None, strided=False, name="rms_65536x1536_bf16"),
        # a ragged batch for an 8-bit product: columns of a wider buffer, scales of 128 columns with a short last one
        dict(kind="rms", back=False, dtype="f16", rows=40000, n=1000, residual=False, group=128, strided=True, name="rms_8bit_40000x1000_f16"),
        # the backward pass of a full batch of the widest net, with the gradient that the residual stream brings
        dict(kind="rms", back=True, dtype="f32", rows=65536, n=1536, residual=True, group=None, strided=False, name="rms_bwd_65536x1536"),
        # a full batch's two buckets of nine
        dict(kind="order", rows=65536, k=2, experts=9, align=1, padding=0.0, name="order_65536x2_of_9"),
        # a wide mixture with padding rows, experts on boundaries of tiles of 128 rows
        dict(kind="order", rows=40000, k=8, experts=256, align=128, padding=0.1, name="order_40000x8_of_256"),
        # the full batch's rows to their buckets
        dict(kind="send", dtype="bf16", rows=65536, n=1536, k=2, experts=9, align=1, padding=0.0, name="send_65536x1536_k2_bf16"),
        # a ragged batch back from a wide mixture
        dict(kind="join", back=False, dtype="f16", rows=30011, n=1000, k=8, experts=256, align=1, padding=0.05, gates=True, name="join_30011x1000_k8_f16"),
        # the gradients of rows and gates of a mid-size net's batch
        dict(kind="join", back=True, dtype="f32", rows=40000, n=768, k=2, experts=9, align=1, padding=0.0, gates=True, name="join_bwd_40000x768_k2"),
        # a table row for each of a batch's features, the frequent ones over and over
        dict(kind="look", dtype="bf16", count=262144, table=FEATURES, n=512, padding=0.05, scale=22.627417, name="look_262144x512_bf16"),
        # the gradient of a row for each of 81 king squares, a small batch: every row has many tokens
        dict(kind="learn", dtype="f32", count=1000, table=81, n=256, padding=0.0, scale=1.0, name="learn_1000x256_of_81"),
        # the gradient of a feature table
        dict(kind="learn", dtype="f32", count=131072, table=FEATURES, n=768, padding=0.05, scale=1.0, name="learn_131072x768"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rms", "rms", "order", "send", "join", "join", "look", "learn", "learn"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "rms":
        n = _log(rng, 8, 12288)
        back = rng.random() < 0.4
        return dict(kind=kind, back=back, dtype=dtype, rows=_log(rng, 1, min(65536, 65536 * 1536 // n)), n=n, residual=rng.random() < 0.5,
                    group=None if back else rng.choice([None, None, 32, 64, 128, n]), strided=rng.random() < 0.3)
    if kind in ("look", "learn"):
        table, n = _log(rng, 2, 200000), _log(rng, 4, 2048)
        while table * n > FEATURES * 1536:
            table //= 2
        return dict(kind=kind, dtype=dtype, count=_log(rng, 1, min(262144, 262144 * 384 // n)), table=table, n=n, padding=rng.choice([0.0, 0.05, 0.5]),
                    scale=rng.choice([1.0, math.sqrt(n)]))
    k = rng.randint(1, 8)
    case = dict(kind=kind, k=k, experts=_log(rng, max(2, k), 1024), align=rng.choice([1, 1, 16, 128]), padding=rng.choice([0.0, 0.05, 0.5]))
    if kind == "order":
        return dict(case, rows=_log(rng, 1, 131072))
    n = _log(rng, 8, 4096)
    case = dict(case, dtype=dtype, n=n, rows=_log(rng, 1, min(65536, 65536 * 1536 // (n * k))))
    return dict(case, back=rng.random() < 0.4, gates=True) if kind == "join" and rng.random() < 0.7 else dict(case, back=False, gates=False) if kind == "join" else case


# ---- inputs ------------------------------------------------------------------------------------------------------
def _shares(table):
    """How often each of a table's rows is asked for, most frequent first: the first few make up a good part of all tokens."""
    i = np.arange(table, dtype=np.float64)
    return np.log((i + 2) / (i + 1)) / math.log(table + 1)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    uniform = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    kind, s = case["kind"], dict(case=case)
    if kind == "rms":
        rows, n, t = case["rows"], case["n"], TYPES[case["dtype"]]
        # rows of a scale of their own with a few large columns; strided: the first columns of a wider buffer
        columns = torch.where(uniform(n) < 0.01, 8.0, 1.0)
        wide = 2 * n if case["strided"] else n
        x = (rand(rows, wide) * (uniform(rows, 1) + 0.2)).to(t)[:, :n]
        x.mul_(columns.to(t))
        s["weight"] = 1 + 0.1 * rand(n)
        if case["back"]:
            s["h"], s["rstd"] = x, _rms(x.float())
            s["dy"] = (1e-2 * rand(rows, n)).to(t)
            s["dresidual"] = (1e-2 * rand(rows, n)).to(t) if case["residual"] else None
        else:
            s["x"], s["residual"] = x, rand(rows, n).to(t) if case["residual"] else None
        return s
    if kind in ("look", "learn"):
        count, table, n, t = case["count"], case["table"], case["n"], TYPES[case["dtype"]]
        place = torch.randperm(table, generator=g, device="cuda")
        rank = (torch.exp(uniform(count).double() * math.log(table + 1)) - 1).long().clamp(0, table - 1)
        s["tokens"] = torch.where(uniform(count) < case["padding"], -1, place[rank])
        if kind == "look":
            s["table"] = (0.02 * rand(table, n)).to(t)
        else:
            s["dy"] = (1e-2 * rand(count, n)).to(t)
        return s
    rows, k, experts = case["rows"], case["k"], case["experts"]
    # distinct experts of every row, some of them in demand; a row of padding has none
    score = uniform(rows, experts).log_().neg_().log_().neg_() + 0.5 * rand(experts)
    index = score.topk(k, dim=1).indices.to(torch.int32)
    del score
    s["index"] = torch.where(uniform(rows, 1) < case["padding"], -1, index)
    if kind == "order":
        return s
    n, t = case["n"], TYPES[case["dtype"]]
    s["order"] = _plain_order(s["index"], experts, case["align"])
    slots = s["order"]["source"].shape[0]
    if kind == "send":
        s["x"] = rand(rows, n).to(t)
        return s
    s["y"] = rand(slots, n).to(t)
    s["gate"] = torch.softmax(rand(rows, k), 1) if case["gates"] else None
    if case["back"]:
        s["dout"] = (1e-2 * rand(rows, n)).to(t)
    return s


def _slots(case):
    entries = case["rows"] * case["k"]
    return (entries + min(case["experts"], entries) * (case["align"] - 1)) // case["align"] * case["align"]


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _rms(h):
    return 1 / (h.square().mean(1) + RMS_EPS).sqrt()


def _plain_rms(s):
    case, t = s["case"], s["x"].dtype
    h = s["x"].float()
    if case["residual"]:
        h = h + s["residual"].float()
    rstd = _rms(h)
    y = h * rstd[:, None] * s["weight"]
    out = {"rstd": rstd}
    if case["residual"]:
        out["h"] = h.to(t)
    if case["group"] is None:
        return dict(out, y=y.to(t))
    rows, n, group = case["rows"], case["n"], case["group"]
    groups = -(-n // group)
    padded = torch.nn.functional.pad(y, (0, groups * group - n)).view(rows, groups, group)
    scale = (padded.abs().amax(2) / E4M3_MOST).clamp(min=LEAST_SCALE)
    q = (padded / scale[:, :, None]).view(rows, groups * group)[:, :n]
    return dict(out, q=q.to(torch.float8_e4m3fn), scale=scale)


def _plain_rms_backward(s):
    h, rstd, dy = s["h"].float(), s["rstd"][:, None], s["dy"].float()
    xh, t = h * rstd, dy * s["weight"]
    dx = rstd * (t - xh * (t * xh).mean(1, keepdim=True))
    if s["dresidual"] is not None:
        dx = dx + s["dresidual"].float()
    return {"dx": dx.to(s["h"].dtype), "dweight": (dy * xh).sum(0)}


def _plain_order(index, experts, align):
    rows, k = index.shape
    entries = rows * k
    flat = index.flatten().long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    by = key.sort(stable=True)
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.long, device=index.device)
    offsets[1:] = ((counts + align - 1) // align * align).cumsum(0)
    begins = torch.zeros(experts + 1, dtype=torch.long, device=index.device)  # of the experts in the sorted entries
    begins[1:] = counts.cumsum(0)
    ok = by.values < experts
    place = torch.where(ok, offsets[by.values] + torch.arange(entries, device=index.device) - begins[by.values], -1)
    position = torch.empty(entries, dtype=torch.long, device=index.device)
    position[by.indices] = place
    slots = (entries + min(experts, entries) * (align - 1)) // align * align
    source = torch.full((slots + 1,), -1, dtype=torch.long, device=index.device)  # the last one takes the entries without a place
    source[torch.where(ok, place, slots)] = torch.where(ok, by.indices, -1)
    return {"position": position.view(rows, k).to(torch.int32), "source": source[:slots].to(torch.int32), "offsets": offsets.to(torch.int32)}


def _plain_send(s):
    source = s["order"]["source"].long()
    x = s["x"][source.clamp(min=0) // s["case"]["k"]]
    return torch.where(source[:, None] >= 0, x, 0)


def _plain_join(s):
    position = s["order"]["position"].long()
    y = torch.where(position[:, :, None] >= 0, s["y"][position.clamp(min=0)].float(), 0)
    if s["gate"] is not None:
        y = y * s["gate"][:, :, None]
    return y.sum(1).to(s["y"].dtype)


def _plain_join_backward(s):
    source, position = s["order"]["source"].long(), s["order"]["position"].long()
    dout, at = s["dout"].float(), source.clamp(min=0)
    dy = torch.where(source[:, None] >= 0, dout[at // s["case"]["k"]] * s["gate"].flatten()[at][:, None], 0)
    y = s["y"][position.clamp(min=0)].float()
    dgate = torch.where(position >= 0, (y * dout[:, None]).sum(2), 0)
    return {"dy": dy.to(s["y"].dtype), "dgate": dgate}


def _plain_look(s):
    tokens, table = s["tokens"], s["table"]
    ok = (tokens >= 0) & (tokens < len(table))
    rows = table[torch.where(ok, tokens, 0)].float() * s["case"]["scale"]
    return torch.where(ok[:, None], rows, 0).to(table.dtype)


def _plain_learn(s):
    case, tokens = s["case"], s["tokens"]
    ok = (tokens >= 0) & (tokens < case["table"])
    total = torch.zeros(case["table"] + 1, case["n"], device=tokens.device)  # the last row takes what has no token
    total.index_add_(0, torch.where(ok, tokens, case["table"]), s["dy"].float())
    return (total[:-1] * case["scale"]).to(s["dy"].dtype)


# ---- one pass ----------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "rms":
            return _plain_rms_backward(s) if case["back"] else _plain_rms(s)
        if kind == "order":
            return _plain_order(s["index"], case["experts"], case["align"])
        if kind == "send":
            return {"places": _plain_send(s)}
        if kind == "join":
            return _plain_join_backward(s) if case["back"] else {"out": _plain_join(s)}
        return {"rows": _plain_look(s)} if kind == "look" else {"dtable": _plain_learn(s)}
    from tatara_b200 import ops
    if kind == "rms":
        if case["back"]:
            dx, dweight = ops.rms_norm_backward(s["dy"], s["h"], s["rstd"], s["weight"], dresidual=s["dresidual"])
            return {"dx": dx, "dweight": dweight}
        if case["group"] is None:
            y, h, rstd = ops.rms_norm_forward(s["x"], s["weight"], residual=s["residual"], eps=RMS_EPS)
            out = {"y": y, "rstd": rstd}
        else:
            q, scale, h, rstd = ops.rms_norm_quantised(s["x"], s["weight"], residual=s["residual"], eps=RMS_EPS, group=case["group"])
            out = {"q": q, "scale": scale, "rstd": rstd}
        return dict(out, h=h) if case["residual"] else out
    if kind == "order":
        return ops.expert_order(s["index"], case["experts"], align=case["align"])._asdict()
    if kind in ("send", "join"):
        order = ops.Order(s["order"]["position"], s["order"]["source"], s["order"]["offsets"])
        if kind == "send":
            return {"places": ops.dispatch_forward(s["x"], order)}
        if case["back"]:
            dy, dgate = ops.combine_backward(s["dout"], s["y"], order, s["gate"])
            return {"dy": dy, "dgate": dgate}
        return {"out": ops.combine_forward(s["y"], order, s["gate"]) if case["gates"] else ops.dispatch_backward(s["y"], order)}
    if kind == "look":
        return {"rows": ops.embedding_forward(s["tokens"], s["table"], scale=case["scale"])}
    return {"dtable": ops.embedding_backward(s["dy"], s["tokens"], case["table"], scale=case["scale"])}


# ---- in 64 bits --------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "order":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "rms":
        n, weight = case["n"], s["weight"].double()
        if case["back"]:
            dy, r = s["dy"].double(), s["rstd"].double()
            xh = torch.einsum("ij,i->ij", s["h"].double(), r)
            along = torch.einsum("ij,j,ij->i", dy, weight, xh) / n
            dx = torch.einsum("i,ij->ij", r, torch.addcmul(dy * weight, xh, along[:, None], value=-1))
            return {"dx": dx if s["dresidual"] is None else dx + s["dresidual"], "dweight": torch.einsum("ij,ij->j", dy, xh)}
        h = s["x"].double() if s["residual"] is None else torch.add(s["residual"].double(), s["x"])
        r = (torch.linalg.vector_norm(h, dim=1).square() / n + RMS_EPS).rsqrt()
        y = torch.einsum("ij,i,j->ij", h, r, weight)
        out = {"rstd": r} if s["residual"] is None else {"rstd": r, "h": h}
        if case["group"] is None:
            return dict(out, y=y)
        column = torch.arange(n, device=y.device) // case["group"]
        most = torch.zeros(case["rows"], int(column[-1]) + 1, dtype=torch.float64, device=y.device).index_reduce_(1, column, y.abs(), "amax")
        scale = torch.clamp(most / E4M3_MOST, min=LEAST_SCALE)
        return dict(out, q=y / scale[:, column], scale=scale)
    if case["kind"] in ("send", "join"):
        rows, k, position = case["rows"], case["k"], s["order"]["position"].long()
        slots = s["order"]["source"].shape[0]
        row, j = (position >= 0).nonzero(as_tuple=True)
        at = position[row, j]
        places = torch.zeros(slots, case["n"], dtype=torch.float64, device=position.device)
        if case["kind"] == "send":
            return {"places": places.index_copy_(0, at, s["x"].double()[row])}
        gate = s["gate"].double() if case["gates"] else torch.ones(rows, k, dtype=torch.float64, device=position.device)
        if case["back"]:
            dout, y = s["dout"].double(), s["y"].double()
            places.index_copy_(0, at, dout[row] * gate[row, j][:, None])
            dgate = torch.zeros(rows, k, dtype=torch.float64, device=position.device)
            dgate[row, j] = torch.einsum("ij,ij->i", y[at], dout[row])
            return {"dy": places, "dgate": dgate}
        out = torch.zeros(rows, case["n"], dtype=torch.float64, device=position.device)
        for c in range(k):
            of = (position[:, c] >= 0).nonzero()[:, 0]
            out[of] += torch.einsum("ij,i->ij", s["y"][position[of, c]].double(), gate[of, c])
        return {"out": out}
    tokens, n = s["tokens"], case["n"]
    ok = (0 <= tokens) & (tokens < case["table"])
    if case["kind"] == "look":
        out = torch.zeros(case["count"], n, dtype=torch.float64, device=tokens.device)
        out[ok] = s["table"].double().index_select(0, tokens[ok]) * case["scale"]
        return {"rows": out}
    # the tokens' rows in order of their tokens, summed along, and the sums' differences
    by = tokens[ok].sort()
    sums = torch.zeros(len(by.values) + 1, n, dtype=torch.float64, device=tokens.device)
    torch.cumsum(s["dy"][ok][by.indices].double(), 0, out=sums[1:])
    ends = torch.searchsorted(by.values, torch.arange(case["table"] + 1, device=tokens.device))
    return {"dtable": (sums[ends[1:]] - sums[ends[:-1]]) * case["scale"]}


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "order":  # choices in; their places, the places' choices and the experts' begins out
        entries = case["rows"] * case["k"]
        return {"bytes": 8 * entries + 4 * _slots(case) + 4 * (case["experts"] + 1), "flops": 0}
    size, n = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size(), case["n"]
    if kind == "rms":
        rows, more = case["rows"], 1 if case["residual"] else 0
        if case["back"]:  # dy, h, 1 / rms and the stream's gradient in, dx out; weight in, its gradient out
            return {"bytes": (3 + more) * rows * n * size + 4 * rows + 8 * n, "flops": (9 + more) * rows * n}
        if case["group"] is None:  # x and the residual in, y and the sum out
            return {"bytes": (2 + 2 * more) * rows * n * size + 4 * rows + 4 * n, "flops": (4 + more) * rows * n}
        groups = -(-n // case["group"])
        return {"bytes": rows * n * ((1 + 2 * more) * size + 1) + 4 * rows * (groups + 1) + 4 * n, "flops": (7 + more) * rows * n}
    if kind in ("send", "join"):
        rows, slots = case["rows"], _slots(case)
        entries = case["rows"] * case["k"] * (1 - case["padding"])
        if kind == "send":  # rows in, all places out
            return {"bytes": (rows * (1 - case["padding"]) + slots) * n * size + 4 * rows * case["k"], "flops": 0}
        gates = (8 if case["gates"] else 4) * rows * case["k"]
        if case["back"]:  # the rows' gradients and the places' rows in, the places' and the gates' gradients out
            return {"bytes": (rows * (1 - case["padding"]) + entries + slots) * n * size + gates + 4 * rows * case["k"], "flops": 3 * entries * n}
        return {"bytes": (entries + rows) * n * size + gates, "flops": 2 * entries * n}
    live = case["count"] * (1 - case["padding"])
    if kind == "look":  # the rows that are asked for in, every one once; a row for each token out
        distinct = float((1 - (1 - _shares(case["table"])) ** live).sum())
        return {"bytes": (distinct + case["count"]) * n * size + 8 * case["count"], "flops": live * n}
    return {"bytes": (live + case["table"]) * n * size + 8 * case["count"], "flops": live * n}
