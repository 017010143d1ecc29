"""Calls that follow one another on a stream overlap at their ends; what one writes, the next one reads.  The same chains with the device idle between the calls,
on another stream and in a graph give the same bits."""
import pytest

import tatara_b200 as tb  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def ops():
    from tatara_b200 import ops as o
    return o


def state(rows, n, experts, side, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(x=r(rows, n), gate=0.05 * r(experts, n), m=torch.zeros(experts, n, device="cuda"), w=r(side, n), wm=torch.zeros(side, n, device="cuda"), scale=1 + 0.1 * r(n), k=2)


def chain(s, turns, between=lambda: None):
    """Every call reads what the one before it has written, in place where it can; workspaces and outputs are freed and given out again along the way."""
    for _ in range(turns):
        y, mean, rstd = ops().layer_norm_forward(s["x"], s["scale"])
        between()
        logits = y @ s["gate"].t()
        r = ops().route_forward(logits, s["k"])
        between()
        d = ops().route_backward(logits, r, r.gate, r.losses)
        between()
        dx, dw, _ = ops().layer_norm_backward(d @ s["gate"], s["x"], mean, rstd, s["scale"])
        between()
        ops().layer_norm_forward(dx, out=dx)
        between()
        ops().muon_step(s["gate"], s["m"], d.t() @ y, lr=0.01)
        between()
        ops().orthogonalise(s["w"], out=s["w"])
        between()
        ops().muon_step(s["w"], s["wm"], s["w"] * dw, lr=0.05)
        between()
        ops().layer_norm_forward(s["w"], out=s["w"])
        between()
        s["x"].add_(dx, alpha=0.1)
    return s


SHAPES = [(4000, 40, 9, 6), (300, 256, 16, 100), (5000, 1001, 33, 70), (64, 9000, 8, 3)]


@pytest.mark.parametrize("rows,n,experts,side", SHAPES)
def test_calls_in_a_row(rows, n, experts, side):
    want = chain(state(rows, n, experts, side, 1), 12, torch.cuda.synchronize)
    torch.cuda.synchronize()
    for _ in range(3):
        got = chain(state(rows, n, experts, side, 1), 12)
        assert all(torch.equal(got[k], want[k]) for k in ("x", "gate", "m", "w", "wm")) and got["x"].isfinite().all()


@pytest.mark.parametrize("rows,n,experts,side", SHAPES[:2])
def test_calls_in_a_row_on_another_stream_and_in_a_graph(rows, n, experts, side):
    want = chain(state(rows, n, experts, side, 2), 4, torch.cuda.synchronize)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    s = state(rows, n, experts, side, 2)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        chain(s, 4)
    stream.synchronize()
    assert all(torch.equal(s[k], want[k]) for k in ("x", "gate", "m", "w", "wm"))
    s = state(rows, n, experts, side, 2)
    keep = {k: v.clone() for k, v in s.items() if torch.is_tensor(v)}
    with torch.cuda.stream(stream):
        chain(s, 1)                      # whatever is set up once, before the capture
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            chain(s, 1)
        for k, v in keep.items():
            s[k].copy_(v)
        for _ in range(4):
            graph.replay()
    stream.synchronize()
    assert all(torch.equal(s[k], want[k]) for k in ("x", "gate", "m", "w", "wm"))


def test_results_of_one_call_are_tensors_of_their_own():
    x = torch.randn(37, 19, device="cuda")
    y, mean, rstd = ops().layer_norm_forward(x)
    dx, dw, db = ops().layer_norm_backward(y, x, mean, rstd)
    r = ops().route_forward(x, 3)
    for group in ((mean, rstd), (dw, db), (r.counts, r.rows, r.prob_mean, r.losses)):
        keep = [t.clone() for t in group]
        for i, t in enumerate(group):
            assert t.is_contiguous() and not t.requires_grad and t.data_ptr() % 128 == 0 and t.device == x.device
            t.fill_(7)   # touches no other result
            for j, u in enumerate(group):
                assert j == i or torch.equal(u, keep[j])
            t.copy_(keep[i])
            assert torch.equal((t * 2).cpu(), (keep[i] * 2).cpu()) and torch.equal(t.view(-1)[:1], keep[i][:1])
    assert r.rows.dtype == r.counts.dtype == torch.int32 and r.losses.dtype == torch.float32 and r.losses.shape == (2,)
    # a leaf of its own, as any new tensor
    leaf = dw.requires_grad_()
    (leaf * leaf).sum().backward()
    assert torch.equal(leaf.grad, 2 * dw.detach()) and not db.requires_grad


def test_an_error_that_an_earlier_call_left_is_not_this_call_s():
    """A call of another part of the library that failed (no such device) leaves its error on the thread; the operators' launches did not fail."""
    import ctypes as C
    lib = tb.load_library()
    x = torch.randn(70, 90, device="cuda")
    want = [ops().layer_norm_forward(x)[0], ops().route_forward(x, 2).gate, ops().orthogonalise(x), ops().orthogonalise(x[:40])]
    zero, result = (C.c_int32 * 8)(), tb._lib.MicrobenchResult()
    for call, w in ((lambda: ops().layer_norm_forward(x)[0], want[0]), (lambda: ops().route_forward(x, 2).gate, want[1]), (lambda: ops().orthogonalise(x), want[2]),
                    (lambda: ops().orthogonalise(x[:40]), want[3])):
        assert lib.tb_ft_microbench(99, zero, zero, 1, 128, 4, 0, 8, 1, 0, C.byref(result)) != 0
        assert torch.equal(call(), w)


def writes():
    """A call, the tensors it writes and those it only reads."""
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    x, dy, v, one = r(6, 40), r(6, 40), torch.zeros(6, device="cuda"), torch.ones(6, device="cuda")
    w, m, g, w2, m2 = r(12, 40), r(12, 40), r(12, 40), r(12, 40), r(12, 40)
    yield lambda: ops().layer_norm_forward(x, out=x), [x], []
    yield lambda: ops().layer_norm_forward(x, out=dy), [dy], [x]
    yield lambda: ops().layer_norm_backward(dy, x, v, one, out=dy), [dy], [x, v, one]
    yield lambda: ops().orthogonalise(g, out=g), [g], []
    yield lambda: ops().orthogonalise(g[:3], out=w2[4:7]), [w2], [g]  # a view's memory is its base's
    yield lambda: ops().muon_step(w, m, g, lr=0.1), [w, m], [g]
    yield lambda: ops().muon_step(w, m, g, lr=0.1, weight_out=w2, momentum_out=m2), [w2, m2], [w, m, g]
    yield lambda: ops().muon_step(w, m, g, lr=0.1, weight_out=w2), [w2, m], [w, g]
    yield lambda: (ops().layer_norm_forward(x, one.new_ones(40)), ops().layer_norm_backward(dy, x, v, one), ops().orthogonalise(x), ops().route_forward(x, 2)), [], [x, dy, v, one]


def test_tensors_that_were_written_are_known_to_be():
    for call, written, read in writes():
        before = [t._version for t in written + read]
        call()
        after = [t._version for t in written + read]
        assert all(b > a for a, b in zip(before, after[:len(written)])) and before[len(written):] == after[len(written):]
    # a gradient through values that a step has replaced since is refused, not computed from the new ones
    w = torch.randn(20, 30, device="cuda", requires_grad=True)
    value = (w * w).sum()
    ops().muon_step(w, torch.zeros(20, 30, device="cuda"), torch.randn(20, 30, device="cuda"), lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        value.backward()
    with torch.inference_mode():  # tensors without such a count
        x = torch.randn(6, 40, device="cuda")
        want = ops().layer_norm_forward(x.clone())[0]
        assert torch.equal(ops().layer_norm_forward(x, out=x)[0], want)
    x = torch.ones(3, 8, device="cuda")
    with pytest.raises(tb.TrainerError):
        ops().layer_norm_forward(x, eps=-1.0, out=x)
    assert x._version == torch.ones(3, 8, device="cuda")._version  # nothing was written


def test_arguments_without_a_truth_value():
    x, w = torch.randn(6, 9, device="cuda"), torch.randn(6, 9, device="cuda")
    r, neither = ops().route_forward(x, 2), torch.ones(2)
    for bad in (lambda: ops().route_forward(x, 2, renormalise=neither), lambda: ops().route_backward(x, r, renormalise=neither),
                lambda: ops().muon_step(w, torch.zeros_like(w), x, lr=0.1, nesterov=neither)):
        with pytest.raises(tb.TrainerError, match="truth value"):
            bad()
    assert torch.equal(ops().route_forward(x, 2, renormalise=torch.tensor(True)).gate, r.gate)


def test_tensors_whose_memory_does_not_hold_their_values():
    x, v = torch.randn(6, 9, device="cuda"), torch.randn(9, device="cuda")
    for t, u in ((torch._neg_view(x), torch._neg_view(v)), (torch._efficientzerotensor((6, 9), device="cuda"), torch._efficientzerotensor((9,), device="cuda"))):
        for bad in (lambda: ops().layer_norm_forward(t), lambda: ops().layer_norm_forward(x, u), lambda: ops().layer_norm_forward(x, out=t), lambda: ops().route_forward(t, 2),
                    lambda: ops().orthogonalise(t), lambda: ops().muon_step(x, torch.zeros_like(x), t, lr=0.1)):
            with pytest.raises(tb.TrainerError, match="in memory"):
                bad()
    assert torch.equal(ops().orthogonalise(torch._neg_view(x).resolve_neg()), ops().orthogonalise(-x))


def test_two_threads_with_a_stream_each():
    """Chains on two streams at once, fed by two threads: the bits of each by itself."""
    import threading
    shapes = [(4000, 40, 9, 6), (300, 256, 16, 100)]
    want = [chain(state(*s, 3 + i), 20) for i, s in enumerate(shapes)]
    got = [state(*s, 3 + i) for i, s in enumerate(shapes)]
    streams = [torch.cuda.Stream() for _ in shapes]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(streams[i]):
                chain(got[i], 20)
            streams[i].synchronize()
        except Exception as e:  # shown by the assertion below
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for g, w in zip(got, want):
        assert all(torch.equal(g[k], w[k]) for k in ("x", "gate", "m", "w", "wm"))
