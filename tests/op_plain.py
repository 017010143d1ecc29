"""Plain 64-bit forms of the operators on device tensors, written from their definitions, and the units of rounding the tests count in."""
import math

import torch

U32 = 2.0 ** -24                                                                        # half a unit in the last place, fp32
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # ... of a result rounded to the type
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # ... of its smallest numbers


def norm_forward(x, weight, bias, eps):
    x = x.double()
    mean = x.mean(1)
    rstd = 1 / torch.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)
    y = (x - mean[:, None]) * rstd[:, None]
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    return y, mean, rstd


def norm_backward(dy, x, mean, rstd, weight):
    x, g = x.double(), dy.double()
    xh = (x - mean.double()[:, None]) * rstd.double()[:, None]
    t = g * weight.double() if weight is not None else g
    dx = rstd.double()[:, None] * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))
    return dx, (g * xh).sum(0), g.sum(0), xh, t


def route_forward(logits, k, renormalise, mask=None):
    """Row by row, as the definition reads."""
    rows, experts = logits.shape
    x = logits.double().cpu()
    index = torch.full((rows, k), -1, dtype=torch.int32)
    gate = torch.zeros(rows, k, dtype=torch.float64)
    counts = torch.zeros(experts, dtype=torch.int32)
    p_sum, z_sum, n = torch.zeros(experts, dtype=torch.float64), 0.0, 0
    for r in range(rows):
        row = x[r].tolist()
        if (mask is not None and not bool(mask[r])) or all(v == -math.inf for v in row):
            continue
        order = sorted((e for e in range(experts) if row[e] != -math.inf), key=lambda e: (-row[e], e))[:k]
        top = max(row)
        p = [math.exp(v - top) for v in row]
        total = sum(p)
        n += 1
        z_sum += (top + math.log(total)) ** 2
        p_sum += torch.tensor([v / total for v in p], dtype=torch.float64)
        below = sum(p[e] for e in order) if renormalise else total
        for j, e in enumerate(order):
            index[r, j], gate[r, j] = e, p[e] / below
            counts[e] += 1
    n1 = max(n, 1)
    mean = p_sum / n1
    return dict(index=index, gate=gate, counts=counts, rows=n, prob_mean=mean,
                losses=torch.tensor([experts / (n1 * k) * float((counts.double() * mean).sum()), z_sum / n1], dtype=torch.float64))


def route_objective(x, index, counts, n, k, renormalise, live, dgate, dlosses):
    """What `route_backward` is the gradient of, for a 64-bit x with the choice and the counts held."""
    x = torch.where(live[:, None], x, torch.zeros_like(x))
    p = torch.softmax(x, 1) * live[:, None]
    lse = torch.logsumexp(x, 1) * live
    ok = index >= 0
    chosen = p.gather(1, index.clamp(min=0).long()) * ok
    gate = chosen / chosen.sum(1, keepdim=True).clamp(min=1e-300) if renormalise else chosen
    n1 = max(n, 1)
    balance = x.shape[1] / (n1 * k) * (counts.double() * p.sum(0) / n1).sum()
    return (gate * dgate * ok).sum() + dlosses[0] * balance + dlosses[1] * (lse ** 2).sum() / n1


COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalise(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The definition, matrix by matrix."""
    x = x.double()
    if x.dim() == 2:
        return orthogonalise(x[None], steps, coefficients, eps)[0]
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + eps)
    a, b, c = coefficients
    for _ in range(steps):
        g = x @ x.transpose(1, 2)
        x = a * x + (b * g + c * g @ g) @ x
    return x.transpose(1, 2) if tall else x


def muon_step(w, m, g, lr, beta, nesterov, weight_decay, scale, clip, steps=5):
    w, m, g = w.double(), m.double(), g.double()
    m = beta * m + g
    o = orthogonalise(g + beta * m if nesterov else m, steps)
    return (w * (1 - lr * weight_decay) - lr * scale * o).clamp(-clip, clip), m
