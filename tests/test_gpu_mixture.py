"""The operators run together as a mixture's layer uses them: token rows onto a residual stream -> root-mean-square norm -> router -> rows by expert -> experts' products -> back,
and all of it backward.  Gradients against automatic differentiation in 64 bits; the same bits with the device idle between the calls, without, on another stream, from two
threads and in a graph."""
import threading

import pytest

import tatara_b200 as tb

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
SCALE, EPS, K, EXPERTS, TABLE = 3.0, 1e-6, 2, 9, 50


def ops():
    from tatara_b200 import ops as o
    return o


def state(rows, n, seed, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    tokens = torch.randint(-1, TABLE, (rows,), generator=g, device="cuda")
    return dict(tokens=tokens, table=(0.3 * r(TABLE, n)).to(dtype), stream=r(rows, n).to(dtype), weight=1 + 0.1 * r(n), gate=(r(EXPERTS, n) / n ** 0.5).to(dtype),
                experts=(r(EXPERTS, n, n) / n ** 0.5).to(dtype), dout=r(rows, n).to(dtype), dlosses=torch.tensor([0.3, 0.01], device="cuda"))


def layer(s, between=lambda: None, align=16):
    """Forward and backward; the stream and the gradients."""
    o, rows = ops(), len(s["tokens"])
    x = o.embedding_forward(s["tokens"], s["table"], scale=SCALE)
    between()
    y, h, rstd = o.rms_norm_forward(x, s["weight"], residual=s["stream"], eps=EPS, out=x)
    between()
    r = o.route_forward(y @ s["gate"].t(), K)
    between()
    order = o.expert_order(r.index, EXPERTS, align=align)
    between()
    xs = o.dispatch_forward(y, order)
    between()
    of = torch.searchsorted(order.offsets[1:], torch.arange(len(order.source), device="cuda", dtype=torch.int32), right=True).clamp(max=EXPERTS - 1)
    w = s["experts"][of]                                  # every place's expert: small products, without waiting for the device
    z = torch.bmm(w, xs[:, :, None])[:, :, 0]
    out = h + o.combine_forward(z, order, r.gate)
    between()
    dz, dgate = o.combine_backward(s["dout"], z, order, r.gate)
    between()
    dxs = torch.bmm(w.transpose(1, 2), dz[:, :, None])[:, :, 0]
    logits = y @ s["gate"].t()
    dlogits = o.route_backward(logits, r, dgate, s["dlosses"])
    between()
    dy = o.dispatch_backward(dxs, order) + dlogits @ s["gate"]
    between()
    dx, dweight = o.rms_norm_backward(dy, h, rstd, s["weight"], dresidual=s["dout"])
    between()
    dtable = o.embedding_backward(dx, s["tokens"], TABLE, scale=SCALE)
    between()
    member = torch.nn.functional.one_hot(of.long(), EXPERTS).to(dz.dtype)
    return dict(out=out, stream=dx, weight=dweight, table=dtable, gate=dlogits.t() @ y, experts=torch.einsum("se,si,sj->eij", member, dz, xs), index=r.index, counts=r.counts,
                position=order.position, rows=rows)


def test_gradients():
    rows, n = 600, 48
    s = state(rows, n, 3)
    got = layer(s)
    p = {k: s[k].double().requires_grad_() for k in ("table", "stream", "weight", "gate", "experts")}
    ok = (s["tokens"] >= 0)[:, None]
    h = p["stream"] + torch.where(ok, SCALE * p["table"][s["tokens"].clamp(min=0)], 0.0)
    y = h / (h.square().mean(1, keepdim=True) + EPS).sqrt() * p["weight"]
    logits = y @ p["gate"].t()
    index = got["index"].long()
    chosen = torch.softmax(logits.gather(1, index), 1)
    z = torch.einsum("rkij,rj->rki", p["experts"][index], y)
    out = h + (chosen[:, :, None] * z).sum(1)
    balance = EXPERTS / (rows * K) * (got["counts"].double() * torch.softmax(logits, 1).mean(0)).sum()
    value = (out * s["dout"].double()).sum() + 0.3 * balance + 0.01 * torch.logsumexp(logits, 1).square().mean()
    value.backward()
    # fp32 throughout: sums of at most 600 tokens' and 48 columns' terms, five of them in a row at worst: (600 + 5 * 48) 2^-24 = 5e-5 of the norm
    assert (got["out"].double() - out).norm() <= 5e-5 * out.norm()
    for name, t in p.items():
        assert (got[name].double() - t.grad).norm() <= 5e-5 * t.grad.norm(), name


def chain(s, turns, between=lambda: None):
    """Every turn works on what the one before has left, in place where it can."""
    results = []
    for _ in range(turns):
        got = layer(s, between)
        s["stream"].copy_(ops().rms_norm_forward(got["out"], eps=EPS)[0])
        s["table"].add_(got["table"], alpha=-0.01)
        s["experts"].add_(got["experts"], alpha=-0.01 / len(s["tokens"]))
        results.append(got["position"].clone())
    return results


KEPT = ("stream", "table", "experts")


@pytest.mark.parametrize("rows,n,dtype", [(700, 40, torch.float32), (3000, 24, torch.bfloat16), (513, 33, torch.float16)])
def test_calls_in_a_row(rows, n, dtype):
    want = state(rows, n, 1, dtype)
    places = chain(want, 4, torch.cuda.synchronize)
    torch.cuda.synchronize()
    for _ in range(3):
        s = state(rows, n, 1, dtype)
        again = chain(s, 4)
        assert all(torch.equal(s[k], want[k]) for k in KEPT) and all(torch.equal(a, b) for a, b in zip(again, places)) and s["stream"].isfinite().all()


def test_on_another_stream_and_in_a_graph():
    want = state(900, 40, 2)
    chain(want, 3, torch.cuda.synchronize)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    s = state(900, 40, 2)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        chain(s, 3)
    stream.synchronize()
    assert all(torch.equal(s[k], want[k]) for k in KEPT)
    s = state(900, 40, 2)
    keep = {k: v.clone() for k, v in s.items()}
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        chain(s, 1)                      # whatever is set up once, before the capture
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            chain(s, 1)
        for k, v in keep.items():
            s[k].copy_(v)
        for _ in range(3):
            graph.replay()
    stream.synchronize()
    assert all(torch.equal(s[k], want[k]) for k in KEPT)


def test_two_threads_on_two_streams():
    want = [state(1500, 40, 5), state(1200, 64, 6)]
    for s in want:
        chain(s, 6, torch.cuda.synchronize)
    got, errors = [state(1500, 40, 5), state(1200, 64, 6)], []
    torch.cuda.synchronize()

    def run(s):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                chain(s, 6)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(s,)) for s in got]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for s, w in zip(got, want):
        assert all(torch.equal(s[k], w[k]) for k in KEPT)


def test_larger_sorts_on_two_streams():
    """Sorts of several launches and table gradients with long lists beside one another: workspaces and counters are a call's own."""
    g = torch.Generator("cuda").manual_seed(8)
    tokens = [torch.randint(0, v, (60000,), generator=g, device="cuda") ** 2 // v for v in (3000, 40)]
    dy = [torch.randn(60000, 96, generator=g, device="cuda") for _ in tokens]
    index = torch.randint(-1, 256, (30000, 4), generator=g, device="cuda", dtype=torch.int32)
    want = [ops().embedding_backward(d, t, 3000) for d, t in zip(dy, tokens)] + list(ops().expert_order(index, 256, align=8))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = [[], [], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append([ops().embedding_backward(dy[i], tokens[i], 3000)] if i < 2 else list(ops().expert_order(index, 256, align=8)))
    torch.cuda.synchronize()
    for r in results[0]:
        assert torch.equal(r[0], want[0])
    for r in results[1]:
        assert torch.equal(r[0], want[1])
    for r in results[2]:
        assert all(torch.equal(a, b) for a, b in zip(r, want[2:]))


def test_results_written_over_tensors_are_marked():
    x, r = torch.randn(8, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    before = x._version, r._version
    ops().rms_norm_forward(x, residual=r, out=x, residual_out=r)
    assert (x._version, r._version) == (before[0] + 1, before[1] + 1)
    ops().rms_norm_quantised(x, residual=r, residual_out=r)
    ops().rms_norm_backward(x, r, torch.ones(8, device="cuda"), out=x)
    out = torch.empty(4, 16, device="cuda")
    v = out._version
    ops().embedding_forward(torch.arange(4, device="cuda"), x, out=out)
    assert (x._version, r._version, out._version) == (before[0] + 2, before[1] + 2, v + 1)


def test_an_order_s_results_are_tensors_of_their_own():
    order = ops().expert_order(torch.randint(0, 5, (37, 3), dtype=torch.int32, device="cuda"), 5, align=4)
    keep = [t.clone() for t in order]
    for i, t in enumerate(order):
        assert t.is_contiguous() and t.data_ptr() % 128 == 0 and t.dtype == torch.int32
        t.fill_(7)
        assert all(torch.equal(u, keep[j]) for j, u in enumerate(order) if j != i)
        t.copy_(keep[i])


def test_the_stream_and_its_rstd_are_tensors_of_their_own():
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(7, 33, device="cuda").to(dtype)
        y, h, rstd = ops().rms_norm_forward(x, residual=x)
        q, scale, h8, rstd8 = ops().rms_norm_quantised(x, residual=x)
        for a, b in ((h, rstd), (h8, rstd8)):
            keep = a.clone(), b.clone()
            assert a.is_contiguous() and b.is_contiguous() and a.dtype == dtype and b.dtype == torch.float32 and torch.equal(keep[0], (2 * x.float()).to(dtype))
            a.fill_(3)
            assert torch.equal(b, keep[1])
            b.fill_(4)
            assert (a == 3).all()


def test_tensors_of_another_device_are_refused():
    x = torch.zeros(4, 8, device="cuda")
    for bad in (lambda: ops().rms_norm_forward(x, torch.zeros(8)), lambda: ops().dispatch_forward(x, ops().Order(torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), None)),
                lambda: ops().embedding_forward(torch.zeros(3, dtype=torch.int64), x)):
        with pytest.raises(tb.TrainerError):
            bad()
