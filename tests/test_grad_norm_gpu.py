"""mc_grad_norm, mc_clip_grads and mc_weights_update_spans_clipped against 64-bit arithmetic.  Squares are summed in double, 16-bit
ones after sums of 8 in float32 (a tree: 3 roundings, so 3 u of the norm's square and 1.5 u of the norm, u = 2^-24); the norm's own rounding
adds u and the double sum n 2^-53.  The factor has the same error and its rounding.  A clipped gradient adds the roundings of factor * scale
and of the product, 6 u in all, and one rounding to its type."""
import ctypes

import numpy as np
import pytest

from oracle import golden as G

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def mc():
    import mckernels
    return mckernels


def torch_():
    import torch
    return torch


KINDS = {"f32": 0, "f16": 1, "bf16": 2}


def dtype(kind):
    t = torch_()
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16}[kind]


def upload(array):
    t = torch_()
    return t.from_numpy(np.frombuffer(bytes(array), dtype=np.uint8).copy()).cuda()


class Run(object):
    """A list of (gradient, output or None, scale) on the device, its spans and workspace."""

    def __init__(self, tensors):
        t, m = torch_(), mc()
        code = {t.float32: 0, t.float16: 1, t.bfloat16: 2}
        self.tensors = tensors
        spans = m.grad_spans([(g.data_ptr(), o.data_ptr() if o is not None else 0, g.numel(), s, code[g.dtype], code[(o if o is not None else g).dtype])
                              for g, o, s in tensors])
        self.n = len(spans)
        self.spans = upload(spans) if self.n else None
        self.size = m.lib().mc_grad_norm_workspace_bytes(self.n)
        self.work = t.full((self.size,), 255, dtype=t.uint8, device="cuda")
        self.stats = t.full((2,), -1.0, device="cuda")

    def norm(self, max_norm, stream=None):
        mc().call("mc_grad_norm", self.spans.data_ptr() if self.n else None, self.n, max_norm, self.stats.data_ptr(), self.work.data_ptr(), self.size, stream)

    def clip(self, stream=None):
        mc().call("mc_clip_grads", self.spans.data_ptr() if self.n else None, self.n, self.stats.data_ptr(), stream)

    def values(self):
        torch_().cuda.synchronize()
        return self.stats.cpu().numpy()


def grads(sizes, kind, seed=0, scale=0.01, packed=True):
    """Tensors of one store, side by side (so most are not aligned to 16 bytes) or 64 elements apart."""
    t = torch_()
    unit = 1 if packed else 64
    offs = np.cumsum([0] + [-(-n // unit) * unit for n in sizes])
    store = (t.randn(int(offs[-1]) + 1, generator=t.Generator().manual_seed(seed)) * scale).to(dtype(kind)).cuda()
    return [store[o:o + n] for o, n in zip(offs, sizes)]


def f64(ts):
    torch_().cuda.synchronize()
    return [x.double().cpu().numpy() for x in ts]


SIZES = [[1], [7], [4096], [4097, 1, 4095], [100003], [0, 5, 0], [65536 * 3 + 1, 17, 31, 1 << 20], [3] * 700, [40_000_001]]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "bf16"), ("f32", "f16")])
def test_norm_and_clip(sizes, kind, out):
    t = torch_()
    gs, outs = grads(sizes, kind, len(sizes)), grads(sizes, out, 5)
    scales = [1.0 if i % 3 else 0.25 for i in range(len(sizes))]
    exact = f64(gs)
    true, _ = G.grad_norm(exact, scales, 1.0)
    run = Run(list(zip(gs, outs, scales)))
    for share in (0.25, 4.0):
        run.norm(max(true * share, 1e-30))
        norm, factor = run.values()
        want = min(1.0, np.float64(np.float32(max(true * share, 1e-30))) / true)
        off = U * (1.01 if kind == "f32" else 2.51) + sum(sizes) * 2.0 ** -52
        assert abs(norm - true) <= true * off
        assert abs(factor - want) <= want * off
        run.clip()
        half = float(t.finfo(dtype(out)).eps) / 2 if out != "f32" else 0.0
        small = float(t.finfo(dtype(out)).tiny) * float(t.finfo(dtype(out)).eps)
        for g, o, s in zip(exact, f64(outs), scales):
            exp = g * (want * s)
            assert (np.abs(o - exp) <= np.abs(exp) * (4 * U + half) * 1.01 + small).all()
    for g, e in zip(f64(gs), exact):
        assert np.array_equal(g, e)                                 # out of place: the gradients stay


def test_in_place_and_without_output():
    gs = grads([1000, 33, 5000], "f32", 2)
    exact = f64(gs)
    true, _ = G.grad_norm(exact, [1, 1, 1], 1)
    run = Run([(gs[0], gs[0], 1.0), (gs[1], None, 1.0), (gs[2], gs[2], 1.0)])
    run.norm(float(np.float32(true * 2)))
    run.clip()
    assert run.values()[1] == 1.0
    assert all(np.array_equal(a, b) for a, b in zip(f64(gs), exact))  # factor 1: not a bit changes
    run.norm(float(np.float32(true / 2)))
    run.clip()
    got = f64(gs)
    for i in (0, 2):
        assert (np.abs(got[i] - exact[i] / 2) <= np.abs(exact[i]) * 3 * U).all()
    assert np.array_equal(got[1], exact[1])


def test_empty_lists_and_zero_gradients():
    t = torch_()
    run = Run([])
    run.norm(1.0)
    run.clip()
    assert list(run.values()) == [0.0, 1.0]
    z = t.zeros(5000, device="cuda")
    run = Run([(z, z, 1.0)])
    run.norm(1.0)
    run.clip()
    assert list(run.values()) == [0.0, 1.0] and not z.any()


def test_a_norm_that_is_not_finite_drops_the_step():
    t, m = torch_(), mc()
    for kind, bad in (("f32", float("nan")), ("f32", float("inf")), ("f16", float("-inf")), ("bf16", float("nan"))):
        gs, outs = grads([5000, 300], kind, 3), grads([5000, 300], kind, 4)
        gs[1][17] = bad
        run = Run([(g, o, 1.0) for g, o in zip(gs, outs)])
        run.norm(1.0)
        run.clip()
        norm, factor = run.values()
        assert not np.isfinite(norm) and factor == 0.0
        assert not any(o.any() for o in outs)
    w, inc, g = (t.randn(256, device="cuda") for _ in range(3))
    before = w.clone(), inc.clone()
    spans = update_spans([(0, 256, 0.9, -0.1)])
    m.call("mc_weights_update_spans_clipped", w.data_ptr(), inc.data_ptr(), g.data_ptr(), spans.data_ptr(), 1, run.stats.data_ptr(), None)
    assert t.equal(w, before[0]) and t.equal(inc, before[1])


def test_large_and_small_gradients():
    """Squares that float32 cannot hold, and a norm that only just fits or does not."""
    t = torch_()
    g = t.full((100,), 3e37, device="cuda")
    run = Run([(g, None, 1.0)])
    run.norm(1.0)
    norm, factor = run.values()
    true = 10 * float(np.float32(3e37))
    assert abs(norm - true) <= true * 2 * U and abs(factor - 1 / true) <= 2.0 ** -149
    g = t.full((10000,), 3e37, device="cuda")
    run = Run([(g, None, 1.0)])
    run.norm(float("inf"))
    assert list(run.values()) == [float("inf"), 0.0]
    g = t.full((100,), 1e-30, device="cuda")
    run = Run([(g, None, 1.0)])
    run.norm(float("inf"))
    norm, factor = run.values()
    true = 10 * float(np.float32(1e-30))
    assert abs(norm - true) <= true * 2 * U and factor == 1.0


@pytest.mark.parametrize("size", [1e-30, 3e-25, 1e-18, 1e15, 1e25])
def test_bf16_gradients_beyond_the_range_of_float32_squares(size):
    """The same accuracy where a float32 square would overflow or vanish, alone and beside zeros."""
    t = torch_()
    g = (t.randn(50_000, generator=t.Generator().manual_seed(1)) * size).to(t.bfloat16).cuda()
    g[1000:9000] = 0
    true = float(np.sqrt((f64([g])[0] ** 2).sum()))
    run = Run([(g, None, 1.0)])
    run.norm(float("inf"))
    assert abs(run.values()[0] - true) <= true * 2.51 * U


def test_bits_do_not_depend_on_the_run():
    gs = grads([3_000_001, 7, 500_000], "bf16", 9)
    run = Run([(g, None, 1.0) for g in gs])
    run.norm(1.0)
    first = run.values().copy()
    for _ in range(5):
        run.work.fill_(3)
        run.norm(1.0)
        assert np.array_equal(run.values(), first)


def update_spans(entries, step=4096):
    rows = [(o + at, min(step, n - at), mom, wceps, 0) for o, n, mom, wceps in entries for at in range(0, n, step)]
    dt = [("start", "<u8"), ("count", "<u4"), ("mom", "<f4"), ("wceps", "<f4"), ("pad", "<u4")]
    spans = upload(np.array(rows, dtype=dt).tobytes())
    spans.rows = len(rows)
    return spans


@pytest.mark.parametrize("sizes", [[10], [4096, 1, 4097], [1000, 192, 100003, 10], [9_000_000]])
def test_clipped_update(sizes):
    t, m = torch_(), mc()
    offs = np.cumsum([0] + [-(-n // 64) * 64 for n in sizes])
    whole = int(offs[-1])
    gen = t.Generator().manual_seed(len(sizes))
    w, inc, g = ((t.randn(whole, generator=gen) * s).cuda() for s in (0.1, 1e-3, 1e-2))
    spans = update_spans([(int(o), n, 0.9 if i % 2 == 0 else 0.5, -0.01 if i % 2 == 0 else 0.0) for i, (o, n) in enumerate(zip(offs, sizes))])
    stats = t.tensor([1.0, 1.0], device="cuda")
    w1, i1, w2, i2 = w.clone(), inc.clone(), w.clone(), inc.clone()
    m.call("mc_weights_update_spans", w1.data_ptr(), i1.data_ptr(), g.data_ptr(), spans.data_ptr(), spans.rows, None)
    m.call("mc_weights_update_spans_clipped", w2.data_ptr(), i2.data_ptr(), g.data_ptr(), spans.data_ptr(), spans.rows, stats.data_ptr(), None)
    assert t.equal(w1, w2) and t.equal(i1, i2)                       # factor 1: the unclipped update's bits
    stats = t.tensor([1.0, 0.3], device="cuda")
    w2, i2 = w.clone(), inc.clone()
    m.call("mc_weights_update_spans_clipped", w2.data_ptr(), i2.data_ptr(), g.data_ptr(), spans.data_ptr(), spans.rows, stats.data_ptr(), None)
    f = float(np.float32(0.3))
    W, I, D, W2, I2 = f64([w, inc, g, w2, i2])
    for i, (o, n) in enumerate(zip(offs, sizes)):
        s = slice(int(o), int(o) + n)
        mom, wceps = (float(np.float32(0.9)), float(np.float32(-0.01))) if i % 2 == 0 else (0.5, 0.0)
        terms = np.abs(mom * I[s]) + np.abs(f * D[s]) + np.abs(wceps * W[s])
        exp = mom * I[s] + f * D[s] + wceps * W[s]
        assert (np.abs(I2[s] - exp) <= terms * 3 * U).all()
        assert (np.abs(W2[s] - (W[s] + exp)) <= terms * 3 * U + np.abs(W[s] + exp) * 2 * U).all()


def test_other_streams_and_graphs():
    t, m = torch_(), mc()
    sizes = [100, 4097, 300_000]
    gs, outs = grads(sizes, "bf16", 1), grads(sizes, "f32", 2)
    run = Run([(g, o, 0.5) for g, o in zip(gs, outs)])
    stream = t.cuda.Stream()
    stream.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(stream):
        run.norm(0.5, stream.cuda_stream)
        run.clip(stream.cuda_stream)
    stream.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph, stream=stream):
        run.norm(0.5, stream.cuda_stream)
        run.clip(stream.cuda_stream)
    for i in range(4):
        for g in gs:
            g.copy_((t.randn(g.shape, generator=t.Generator().manual_seed(i)) * 0.01 * (i + 1)).to(g.dtype))
        graph.replay()
        t.cuda.synchronize()
        got = run.stats.clone(), [o.clone() for o in outs]
        run.norm(0.5)
        run.clip()
        t.cuda.synchronize()
        assert t.equal(got[0], run.stats) and all(t.equal(a, b) for a, b in zip(got[1], outs))


def test_together_as_a_training_step_uses_them():
    """logits -> log probabilities -> their gradient -> dense weight gradient -> norm -> clipped update, against the same step in 64 bits."""
    t, m = torch_(), mc()
    N, D, V = 96, 64, 1000
    rng = np.random.default_rng(4)
    xv, wv = rng.standard_normal((D, N)).astype(np.float32), (rng.standard_normal((V, D)) * 0.3).astype(np.float32)
    y = rng.integers(0, V, N)
    x, w = t.from_numpy(xv).cuda(), t.from_numpy(wv).cuda()
    inc, dw, logits, dlogits = t.zeros(V, D, device="cuda"), t.zeros(V, D, device="cuda"), t.zeros(V, N, device="cuda"), t.zeros(V, N, device="cuda")
    lab = t.as_tensor(y, dtype=t.float32).cuda()
    lp, stats = t.zeros(N, device="cuda"), t.zeros(2, N, device="cuda")
    run = Run([(dw.view(-1), None, 1.0)])
    spans = update_spans([(0, V * D, 0.9, 0.0)])
    size = m.lib().mc_log_probs_workspace_bytes(0, N, 1, N, V, 0)
    work = t.zeros(max(size, 16), dtype=t.uint8, device="cuda")
    W, INC = wv.astype(np.float64), np.zeros((V, D))
    rate, max_norm = 0.5, 0.05
    for _ in range(3):
        m.call("mc_gemm", w.data_ptr(), x.data_ptr(), logits.data_ptr(), V, N, D, 0, 0, D, N, N, 0.0, 1.0, None, 0, None, 0, None)
        m.call("mc_log_probs", logits.data_ptr(), 0, N, 1, lab.data_ptr(), 0, N, V, lp.data_ptr(), None, stats.data_ptr(), None, None, 0, work.data_ptr(), size, None)
        m.call("mc_log_probs_grad", logits.data_ptr(), 0, N, 1, lab.data_ptr(), 0, N, V, stats.data_ptr(), None, None, rate / N, None, 0.0, None, 0.0,
               dlogits.data_ptr(), N, 1, 0, None)
        m.call("mc_gemm", dlogits.data_ptr(), x.data_ptr(), dw.data_ptr(), V, D, N, 0, 1, N, N, D, 0.0, 1.0, None, 0, None, 0, None)
        run.norm(max_norm)
        m.call("mc_weights_update_spans_clipped", w.data_ptr(), inc.data_ptr(), dw.data_ptr(), spans.data_ptr(), spans.rows, run.stats.data_ptr(), None)
        L = (W @ xv.astype(np.float64)).T
        e = G.log_probs(L, y)
        g = G.log_probs_grad(L, y, np.stack([e["max"], e["logSum"]]), None, g=np.full(N, rate / N))
        dW = g.T @ xv.astype(np.float64).T
        norm, factor = G.grad_norm([dW], [1.0], max_norm)
        assert factor < 1.0
        # a logit sums D = 64 products of size <= 4 * 1: off by 64 u * 16 at most, and p by that relative; the weight gradient sums N = 96 more
        assert np.abs(lp.cpu().numpy() - e["logp"]).max() <= 64 * 16 * U + 400 * U
        assert abs(run.values()[0] - norm) <= norm * (64 * 16 + 400) * U * 2
        INC = 0.9 * INC + factor * dW
        W = W + INC
        tol = (64 * 16 + 400 + N) * U * 8
        assert np.abs(w.cpu().numpy() - W).max() <= tol * np.abs(INC).max() + 4 * U * np.abs(W).max()
