"""What mc_log_probs, mc_log_probs_grad and the gradient-norm entry points refuse (argument checks run before any device work), how
gradient lists are cut into spans, and the 64-bit oracle of the log probabilities against its own differences."""
import ctypes

import numpy as np
import pytest

from oracle import golden as G

P = 1 << 20      # stands for a device pointer; never read


def lib():
    import mckernels
    return mckernels.lib()


def last():
    return lib().mc_last_error().decode()


def forward(logits=P, type=0, cs=1, ns=100, labels=P, label_type=3, N=4, V=100, logp=P, H=P, stats=P, classes=None, top=None, k=0, work=None, size=0):
    return lib().mc_log_probs(logits, type, cs, ns, labels, label_type, N, V, logp, H, stats, classes, top, k, work, size, None)


@pytest.mark.parametrize("kw,text", [
    (dict(V=0), "classes"), (dict(V=(1 << 30) + 1, ns=1 << 31), "classes"), (dict(N=-1), "cases"), (dict(type=3), "element type"), (dict(type=-1), "element type"), (dict(logits=None), "logits"),
    (dict(logits=P + 2), "aligned"), (dict(type=2, logits=P + 1), "aligned"), (dict(cs=2, ns=100), "stride"), (dict(cs=1, ns=99), "stride"),
    (dict(cs=3, ns=1), "stride"), (dict(cs=0, ns=1), "positive"), (dict(cs=1, ns=-100), "positive"), (dict(cs=1, ns=1 << 62), "large"),
    (dict(labels=None), "labels"), (dict(labels=P + 2), "labels"), (dict(label_type=1), "MC_I32"), (dict(k=-1), "numTop"), (dict(k=33, classes=P, top=P), "numTop"),
    (dict(k=2), "topClasses"), (dict(k=2, classes=P), "topClasses"), (dict(classes=P, top=P), "topClasses"), (dict(logp=None, H=None, stats=None), "no output"),
    (dict(V=(1 << 24) + 1, ns=1 << 25, label_type=0), "float32 labels"),
])
def test_forward_refusals(kw, text):
    assert forward(**kw) == -1 and text in last()


def test_no_cases_is_no_work():
    assert forward(N=0) == 0 and forward(N=0, logits=None) == 0
    assert grad(N=0) == 0


def grad(logits=P, type=0, cs=1, ns=100, labels=P, label_type=3, N=4, V=100, stats=P, H=P, sl=1.0, sh=1.0, sz=1.0, target=P, tcs=1, tns=100):
    return lib().mc_log_probs_grad(logits, type, cs, ns, labels, label_type, N, V, stats, H, None, sl, None, sh, None, sz, target, tcs, tns, 0, None)


@pytest.mark.parametrize("kw,text", [
    (dict(V=0), "classes"), (dict(type=5), "element type"), (dict(logits=None), "logits"), (dict(target=None), "target"), (dict(target=P + 1), "aligned"),
    (dict(stats=None), "maxAndLogSum"), (dict(H=None), "entropy"), (dict(labels=None), "labels"), (dict(ns=99), "stride"), (dict(tns=99), "target"),
    (dict(tcs=100, tns=1), "order"), (dict(tns=101), "overlap"), (dict(target=P + 400), "overlap"), (dict(target=P + 4 * 399), "overlap"),
])
def test_gradient_refusals(kw, text):
    assert grad(**kw) == -1 and text in last()


def test_matrices_that_no_grid_covers_are_refused():
    assert forward(N=(1 << 26) - 3, V=10, ns=10) == -1 and "too many cases" in last()
    assert grad(N=(1 << 26) - 3, V=10, ns=10, tns=10, target=1 << 50) == -1 and "too many cases" in last()
    assert grad(N=1 << 24, V=1 << 15, ns=1 << 15, tns=1 << 15, target=1 << 50) == -1 and "too many cases" in last()
    assert grad(N=(1 << 31) - 1, V=1 << 20, cs=1 << 31, ns=1, tcs=1 << 31, tns=1, target=1 << 60) == -1 and "too many cases" in last()
    assert lib().mc_clip_grads(P, 1 << 23, P, None) == -1 and "too many spans" in last()
    assert lib().mc_weights_update_spans_clipped(P, P, P, P, 1 << 24, P, None) == -1 and "too many spans" in last()
    import mckernels as m
    with pytest.raises(m.McError, match="too many elements"):
        m.grad_spans([(P, 0, 1 << 48, 1.0, 2, 2)])


def test_workspace_refusals():
    L = lib()
    assert L.mc_grad_norm(P, 3, 1.0, P, None, 0, None) == -3 and "workspace" in last()
    assert L.mc_grad_norm(P, 3, 1.0, P, P, 8, None) == -3
    assert L.mc_grad_norm(P, 3, 1.0, P, P + 8, 1 << 20, None) == -3


def test_workspace_of_split_cases():
    L = lib()
    size = L.mc_log_probs_workspace_bytes(2, 1, 131072, 1, 131072, 20)
    assert size > 0
    kw = dict(type=2, ns=131072, N=1, V=131072, classes=P, top=P, k=20)
    assert forward(**kw) == -3 and "workspace" in last()
    assert forward(work=P, size=size - 1, **kw) == -3 and forward(work=P + 8, size=size, **kw) == -3
    assert L.mc_log_probs_workspace_bytes(0, 128, 1, 128, 10, 5) == 0               # short cases take one launch and no workspace
    for bad in ((3, 1, 10, 4, 10, 0), (0, 2, 2, 4, 10, 0), (0, 1, 10, -1, 10, 0), (0, 1, 10, 4, 0, 0), (0, 1, 10, 4, 10, 33)):
        assert L.mc_log_probs_workspace_bytes(*bad) == 0


@pytest.mark.parametrize("args", [(None, 3, 1.0, P), (P, -1, 1.0, P), (P, 3, 0.0, P), (P, 3, -1.0, P), (P, 3, float("nan"), P), (P, 3, 1.0, None)])
def test_norm_refusals(args):
    assert lib().mc_grad_norm(*args, P, 1 << 20, None) == -1
    if args[2] == 1.0:
        assert lib().mc_clip_grads(args[0], args[1], args[3], None) == -1


def test_update_refusals():
    L = lib()
    assert L.mc_weights_update_spans_clipped(P, P, P, P, 3, None, None) == -1 and "null" in last()
    assert L.mc_weights_update_spans_clipped(P + 4, P, P, P, 3, P, None) == -1 and "aligned" in last()
    assert L.mc_weights_update_spans_clipped(P, P, P, P, 0, P, None) == 0


def test_spans_cover_every_tensor_once():
    import mckernels as m
    rng = np.random.default_rng(0)
    for big in (1, 1000, 70_000_000):
        sizes = [int(v) for v in rng.integers(0, 20000, 40)] + [big, 0, 4096]
        at, tensors = P, []
        for i, n in enumerate(sizes):
            tensors.append((at, (1 << 40) + 2 * at if i % 2 else 0, n, float(i + 1), m.BF16, m.F32))
            at += 2 * n
        spans = m.grad_spans(tensors)
        got = iter(spans)
        for g, o, n, s, gt, ot in tensors:
            done = 0
            while done < n:
                sp = next(got)
                assert sp.grad == g + 2 * done and (sp.out or 0) == (o + 4 * done if o else 0)
                assert sp.scale == s and (sp.gradType, sp.outType) == (gt, ot) and 0 < sp.count <= 65536
                done += sp.count
            assert done == n
        assert next(got, None) is None


def test_span_refusals():
    import mckernels as m
    ok = (P, P + 4096, 10, 1.0, 0, 0)
    assert len(m.grad_spans([])) == 0 and len(m.grad_spans([(0, 0, 0, 1.0, 0, 0)])) == 0
    assert len(m.grad_spans([ok, (P, 0, 10, 1.0, 0, 0)])) == 2                  # a shared gradient may be listed twice
    assert len(m.grad_spans([(P, P, 10, 1.0, 0, 0)])) == 1
    for bad, text in [([(P, P + 4096, 10, 1.0, 3, 0)], "type"), ([(P, 0, 10, 1.0, 0, 7)], "type"), ([(0, 0, 10, 1.0, 0, 0)], "null"),
                      ([(P + 2, 0, 10, 1.0, 0, 0)], "aligned"), ([(P, P + 4097, 10, 1.0, 1, 1)], "aligned"), ([(P, 0, 10, float("nan"), 0, 0)], "finite"),
                      ([(P, P, 10, 1.0, 1, 2)], "in place"), ([(P, P + 4, 10, 1.0, 0, 0)], "overlap"), ([ok, ok], "overlap"),
                      ([(P, P, 10, 1.0, 0, 0)] * 2, "overlap"), ([ok, (P + 4096 + 36, 0, 1, 1.0, 0, 0)], "overlap"), ([ok, (1 << 30, P + 8, 2, 1.0, 0, 0)], "overlap"),
                      ([(P, 0, 1 << 60, 1.0, 0, 0)], "elements")]:
        with pytest.raises(m.McError, match=text):
            m.grad_spans(bad)
    list_ = (m.GradTensor * 1)(m.GradTensor(P, None, 10000, 1.0, 0, 0, 0))
    spans, n = (m.GradSpan * 1)(), ctypes.c_int(0)
    assert lib().mc_grad_spans(list_, 1, spans, 1, ctypes.byref(n)) == -1 and n.value == 3
    assert lib().mc_grad_spans(None, 1, spans, 1, ctypes.byref(n)) == -1 and lib().mc_grad_spans(list_, 1, spans, 1, None) == -1


def test_oracle_gradient_against_differences():
    """Central differences of the oracle's own outputs in 64 bits: truncation h^2 (third derivatives are below 8 here) and rounding 1e-16 / h."""
    rng = np.random.default_rng(1)
    N, V, h = 5, 9, 1e-5
    x = rng.standard_normal((N, V)) * 2
    x[2, 3] = -np.inf
    y = np.array([0, 8, 1, -1, 9])
    g, he, z = rng.standard_normal((3, N))
    e = G.log_probs(x, y)
    grad = G.log_probs_grad(x, y, np.stack([e["max"], e["logSum"]]), e["entropy"], g=g, h=he, z=z)

    def value(v):
        q = G.log_probs(v, y)
        return g * q["logp"] + he * q["entropy"] + z * (q["max"] + q["logSum"])
    for j in range(V):
        d = np.zeros((N, V))
        d[:, j] = h
        num = (value(x + d) - value(x - d)) / (2 * h)
        assert np.abs(num - grad[:, j]).max() < 8 * h * h * 10 + 1e-14 / h


def test_oracle_forward():
    x = np.log(np.array([[0.5, 0.25, 0.125, 0.125]]))
    e = G.log_probs(x, np.array([1]), 6)
    assert abs(e["logp"][0] - np.log(0.25)) < 1e-15 and abs(e["entropy"][0] - 1.75 * np.log(2)) < 1e-15
    assert list(e["classes"][:, 0]) == [0, 1, 2, 3, -1, -1] and e["top"][5, 0] == -np.inf
    e = G.log_probs(np.array([[-np.inf] * 3, [np.nan, 1.0, 2.0], [np.inf, 0.0, 1.0]]), np.array([0, 1, -1]), 2)
    assert e["logp"][0] == -np.inf and np.isnan(e["logp"][1]) and e["logp"][2] == 0.0 and e["entropy"][0] == 0.0
    assert list(e["classes"][:, 0]) == [-1, -1] and list(e["classes"][:, 1]) == [2, 1] and list(e["classes"][:, 2]) == [0, 2]
