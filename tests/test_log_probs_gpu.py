"""mc_log_probs / mc_log_probs_grad against the 64-bit oracle: element types, both layouts, strides and alignments, lengths from one
class to long ones, ruled-out classes and empty cases, ties, extremes, streams and captured graphs.

Tolerances, with u = 2^-24 (half a float32 step): a lane adds at most V / 32 + 64 terms one after the other in any variant, and each
term exp(t) is off by (|t| + 8) u relative, |t| <= 52 wherever exp(t) matters beside exp(0) = 1.  So a sum over the classes is off
by D u relative, D = V / 32 + 124.  The log sum inherits D u absolute and its own rounding; a log probability adds the rounding of
x - m; the entropy log s - w / s has 2 D u relative on w / s.  p in the gradient is off by (|ln p| + 8) u relative."""
import numpy as np
import pytest

from oracle import golden as G

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")


def mc():
    import mckernels
    return mckernels


def torch_():
    import torch
    return torch


def dtypes():
    t = torch_()
    return {"f32": (t.float32, 0), "f16": (t.float16, 1), "bf16": (t.bfloat16, 2)}


class Matrix(object):
    """Logits on the device from a (numCases, numOut) array: `layout` "class" (the library's own) or "case", rows `pad` elements apart
    and the first element `shift` elements off alignment."""

    def __init__(self, values, kind, layout, pad=0, shift=0):
        t = torch_()
        dtype, self.code = dtypes()[kind]
        v = t.from_numpy(np.ascontiguousarray(values, dtype=np.float32)).to(dtype)
        self.N, self.V = values.shape
        rows, cols = (self.V, self.N) if layout == "class" else (self.N, self.V)
        self.store = t.full((shift + rows * (cols + pad) + 8,), 7.0, dtype=dtype).cuda()
        self.view = self.store[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
        self.view.copy_(v.t() if layout == "class" else v)
        self.layout, ld = layout, cols + pad
        self.cs, self.ns = (ld, 1) if layout == "class" else (1, ld)
        self.exact = v.double().numpy()          # what the kernel is given, to the bit

    def rows(self):
        x = self.view.t() if self.layout == "class" else self.view
        return x.double().cpu().numpy()


def forward(x, labels, top=0, entropy=True, label_type=3, stream=None, outs=None):
    t, m = torch_(), mc()
    N, V = x.N, x.V
    y = t.as_tensor(np.asarray(labels), dtype=t.int32 if label_type == 3 else t.float32).cuda()
    size = m.lib().mc_log_probs_workspace_bytes(x.code, x.cs, x.ns, N, V, top)
    work = t.full((max(16, size),), 255, dtype=t.uint8, device="cuda")
    o = dict(logp=t.full((N,), 9.0, device="cuda"), H=t.full((N,), 9.0, device="cuda"), stats=t.full((2, N), 9.0, device="cuda"),
             classes=t.full((max(top, 1), N), 9, dtype=t.int32, device="cuda"), top=t.full((max(top, 1), N), 9.0, device="cuda"))
    m.call("mc_log_probs", x.view.data_ptr(), x.code, x.cs, x.ns, y.data_ptr(), label_type, N, V, o["logp"].data_ptr(),
           o["H"].data_ptr() if entropy else None, o["stats"].data_ptr(), o["classes"].data_ptr() if top else None,
           o["top"].data_ptr() if top else None, top, work.data_ptr(), size, stream)
    if outs is not None:
        outs.update(o, y=y, work=work)
        return None
    t.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in o.items()}


def same(got, exp, tol):
    """|got - exp| <= tol where exp is finite; the same infinities and NaN elsewhere."""
    got, exp = got.astype(np.float64), np.asarray(exp, np.float64)
    fine = np.isfinite(exp)
    assert np.array_equal(np.isnan(got), np.isnan(exp)), (got, exp)
    rest = ~fine & ~np.isnan(exp)
    assert np.array_equal(got[rest], exp[rest]), (got[rest], exp[rest])
    err, tol = np.abs(got - exp)[fine], np.broadcast_to(tol, exp.shape)[fine]
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()))


def check(x, labels, top, got, entropy=True):
    e = G.log_probs(x.exact, labels, top)
    D = x.V / 32.0 + 124.0
    with np.errstate(invalid="ignore", over="ignore"):
        same(got["stats"][0], e["max"], 0.0)
        tol_sum = U * (D + np.abs(e["logSum"]) + 2)
        same(got["stats"][1], e["logSum"], tol_sum)
        same(got["logp"], e["logp"], tol_sum + U * 3 * np.abs(e["logp"]))
        if entropy:
            same(got["H"], e["entropy"], tol_sum + U * (2 * D + 2) * np.abs(e["meanShift"]) + U * np.abs(e["entropy"]))
        if top:
            assert np.array_equal(got["classes"], e["classes"])
            same(got["top"], e["top"], tol_sum + U * 3 * np.where(np.isfinite(e["top"]), np.abs(e["top"]), 0.0))


def logits(rng, N, V, spread=2.5):
    x = rng.standard_normal((N, V)) * spread
    y = rng.integers(0, V, N)
    x[np.arange(N), y] = rng.random(N) * 16
    return x, y


# numCases, numOut, layout, pad, shift, top: both sides of every rule that picks a variant, odd sizes, a single class, a single case
SHAPES = [
    (1, 1, "class", 0, 0, 1), (1, 1, "case", 0, 0, 5), (128, 10, "class", 0, 0, 5), (22, 10, "class", 0, 0, 10), (5, 3, "case", 0, 0, 5),
    (128, 1000, "class", 0, 0, 5), (130, 999, "class", 3, 1, 20), (7, 1000, "class", 0, 0, 32), (1, 1000, "class", 5, 0, 3), (33, 257, "class", 0, 0, 0),
    (1, 50021, "case", 0, 0, 20), (3, 131072, "case", 0, 0, 20), (64, 8191, "case", 1, 1, 5), (700, 2049, "case", 0, 0, 32), (1030, 515, "case", 13, 3, 1),
    (2, 70001, "class", 0, 0, 32), (257, 4096, "class", 0, 2, 8), (2100, 40, "case", 0, 0, 4), (2500, 70, "class", 1, 0, 3), (300, 30011, "case", 0, 0, 0),
    (1, 200000, "class", 0, 0, 20),
]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V,layout,pad,shift,top", SHAPES)
def test_forward(N, V, layout, pad, shift, top, kind):
    rng = np.random.default_rng(N * 7 + V)
    v, y = logits(rng, N, V)
    y[rng.random(N) < 0.1] = -1
    x = Matrix(v, kind, layout, pad, shift)
    check(x, y, top, forward(x, y, top))
    assert np.array_equal(x.rows(), x.exact)                      # the logits are read only


def test_outputs_that_are_not_asked_for_and_float_labels():
    rng = np.random.default_rng(3)
    for layout in ("class", "case"):
        v, y = logits(rng, 40, 300)
        x = Matrix(v, "f32", layout)
        check(x, y, 0, forward(x, y, 0, entropy=False), entropy=False)
        y[:5] = [-1, 300, 10 ** 6, 299, 0]
        check(x, y, 3, forward(x, y, 3, label_type=0))            # float32 class indices, as cost.logreg has them
        t, m = torch_(), mc()
        H = t.zeros(40, device="cuda")
        size = m.lib().mc_log_probs_workspace_bytes(x.code, x.cs, x.ns, 40, 300, 0)
        work = t.zeros(max(16, size), dtype=t.uint8, device="cuda")
        m.call("mc_log_probs", x.view.data_ptr(), x.code, x.cs, x.ns, None, 0, 40, 300, None, H.data_ptr(), None, None, None, 0, work.data_ptr(), size, None)
        assert np.array_equal(H.cpu().numpy(), forward(x, y, 3)["H"])


MASK_SHAPES = [(6, 10), (9, 1000), (6, 40000)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["class", "case"])
@pytest.mark.parametrize("N,V", MASK_SHAPES)
def test_ruled_out_classes_and_extremes(N, V, layout, kind):
    """Rows of -inf; one class left; labels that are ruled out; the type's lowest and largest values; NaN and +inf."""
    rng = np.random.default_rng(V)
    v, y = logits(rng, N, V)
    top_value = float(torch_().finfo(dtypes()[kind][0]).max)
    v[0] = -INF                                                    # nothing left
    v[1] = -INF
    v[1, V // 2] = 1.5                                             # one class left, and it is not the label
    y[1] = V // 2 - 1
    v[2] = -top_value                                              # a mask of the lowest value over everything: uniform
    v[3] = -top_value
    v[3, [0, V - 1]] = [2.0, 2.0]                                  # two classes left by such a mask
    v[4, ::2] = -INF
    v[5, 1], v[5, V - 1] = top_value, -top_value                   # x - m overflows
    x = Matrix(v, kind, layout)
    check(x, y, 5, forward(x, y, 5))
    v[0, 0] = np.nan
    v[1, 2] = INF
    v[2, V - 1] = np.nan
    v[3] = np.nan
    x = Matrix(v, kind, layout)
    check(x, y, 5, forward(x, y, 5))


@pytest.mark.parametrize("layout", ["class", "case"])
@pytest.mark.parametrize("N,V", [(3, 50), (3, 5000), (2, 150000)])
def test_ties_and_orders(N, V, layout):
    """Equal logits go by class; rising, falling and periodic rows fill the candidate lists in the worst orders; -0 equals 0."""
    rows = [np.zeros(V), np.arange(V) / 1000.0, -np.arange(V) / 1000.0, (np.arange(V) % 7).astype(float), np.where(np.arange(V) % 2, -0.0, 0.0),
            np.floor(np.arange(V) / 300.0), np.where(np.arange(V) % 256 < 3, 5.0, 0.0), np.where(np.arange(V) % 64 == 9, np.arange(V) / 1e4, -3.0)]
    for kind in ("f32", "bf16"):
        for i in range(0, len(rows), N):
            v = np.stack((rows + rows)[i:i + N])
            for top in (1, 20, 32):
                x = Matrix(v, kind, layout)
                y = np.arange(N) % V
                check(x, y, top, forward(x, y, top))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("N,V", [(2, 3000), (2, 16384), (2, 24000), (2, 33000), (2, 40000), (2, 300000), (300, 33000)])
def test_joined_parts(N, V, kind):
    """Cases split into few parts and many: more parts than alternatives and fewer, ties beyond the joining kernels' lists, one part that holds
    all of the best, parts that hold nothing."""
    rng = np.random.default_rng(V)
    rows = [np.zeros(V), np.arange(V) // 64 * 1.0, np.where(np.arange(V) % 5 == 0, 1.0, -2.0), np.where(np.arange(V) < 40, 9.0 + np.arange(V) / 64.0, 0.0),
            np.where(np.arange(V) >= V - 3, 2.0, -INF), np.where(np.arange(V) % 1000 == 7, np.arange(V) % 7.0, -INF), rng.standard_normal(V), np.floor(3 * rng.standard_normal(V))]
    for i in range(0, len(rows), min(N, len(rows))):
        v = np.resize(np.stack(rows[i:i + N]), (N, V))
        for top in (1, 5, 20, 32) if N == 2 else (20,):
            x = Matrix(v, kind, "case")
            y = np.arange(N) % V
            check(x, y, top, forward(x, y, top))


@pytest.mark.parametrize("layout", ["class", "case"])
def test_offsets_beyond_32_bits(layout):
    """Lines further apart than 2^32 bytes (and elements)."""
    t, m = torch_(), mc()
    N, V, ld = (3, 2, (1 << 32) + 3) if layout == "class" else (2, 300, (1 << 32) + 5)
    lines = V if layout == "class" else N
    store = t.empty((lines - 1) * ld + 512, dtype=t.bfloat16, device="cuda")
    rng = np.random.default_rng(5)
    v, y = logits(rng, N, V)
    x = Matrix(v, "bf16", layout)
    x.view, x.cs, x.ns = store, (ld if layout == "class" else 1), (1 if layout == "class" else ld)
    src = t.from_numpy(x.exact).to(t.bfloat16).cuda()
    for i in range(lines):
        store[i * ld:i * ld + (N if layout == "class" else V)] = src[:, i] if layout == "class" else src[i]
    got = forward(x, y, 2)
    check(x, y, 2, got)
    g = t.full((N,), -0.25, device="cuda")
    stats = t.from_numpy(got["stats"]).cuda()
    yy = t.as_tensor(y, dtype=t.int32).cuda()
    m.call("mc_log_probs_grad", store.data_ptr(), x.code, x.cs, x.ns, yy.data_ptr(), 3, N, V, stats.data_ptr(), None, g.data_ptr(), 1.0, None, 0.0,
           None, 0.0, store.data_ptr(), x.cs, x.ns, 0, None)
    exp = G.log_probs_grad(x.exact, y, got["stats"], None, g=np.full(N, -0.25))
    for i in range(lines):
        line = store[i * ld:i * ld + (N if layout == "class" else V)].double().cpu().numpy()
        same(line, exp[:, i] if layout == "class" else exp[i], 2.0 ** -8 * np.abs(exp[:, i] if layout == "class" else exp[i]) + 1e-6)
    del store
    t.cuda.empty_cache()


def grad_case(x, y, rng, target_pad=0, in_place=False, add=False, terms="lhz", scales=(0.5, 0.25, 2.0), arrays=True):
    t, m = torch_(), mc()
    N, V = x.N, x.V
    e = G.log_probs(x.exact, y, 0)
    stats = np.stack([e["max"], e["logSum"]]).astype(np.float32)
    H = e["entropy"].astype(np.float32)
    gs = [rng.standard_normal(N).astype(np.float32) for _ in range(3)]
    d = [t.from_numpy(g).cuda() for g in gs]
    scale = [s if c in terms else 0.0 for s, c in zip(scales, "lhz")]
    target = x if in_place else Matrix(rng.standard_normal((N, V)), {0: "f32", 1: "f16", 2: "bf16"}[x.code], x.layout, target_pad, 1)
    before = target.exact
    dstats, dH, yy = t.from_numpy(stats).cuda(), t.from_numpy(H).cuda(), t.as_tensor(np.asarray(y), dtype=t.int32).cuda()
    pt = [p.data_ptr() if arrays else None for p in d]
    m.call("mc_log_probs_grad", x.view.data_ptr(), x.code, x.cs, x.ns, yy.data_ptr() if "l" in terms else None, 3, N, V, dstats.data_ptr(),
           dH.data_ptr() if "h" in terms else None, pt[0], scale[0], pt[1], scale[1], pt[2], scale[2], target.view.data_ptr(), target.cs, target.ns, int(add), None)
    if not arrays:
        gs = [np.ones(N, np.float32)] * 3
    w = [s * g.astype(np.float64) for s, g in zip(scale, gs)]
    exp = G.log_probs_grad(x.exact, y, stats, H, g=w[0], h=w[1], z=w[2])
    size = G.log_probs_grad_size(x.exact, y, stats, H, g=w[0], h=w[1], z=w[2])
    half = float(t.finfo(x.view.dtype).eps) / 2
    total = exp + (before if add else 0.0)
    # ln p is off by (2 |ln p| + 13) u, exp and the products and sums around it add 8 u: 32 u (1 + |ln p| / 8) of the terms; then one
    # rounding to the type (or its smallest step; float32 results may flush below 1.2e-38 times a weight)
    tol = size * U * 32 + U * 2 * np.abs(total) + (half * np.abs(total) if x.code else 0.0) + float(t.finfo(x.view.dtype).tiny) * float(t.finfo(x.view.dtype).eps) + 1e-35
    with np.errstate(invalid="ignore"):
        same(target.rows(), total, np.where(np.isfinite(tol), tol, 0.0))
    t.cuda.synchronize()
    if not in_place and target_pad:
        flat = target.store.float().cpu().numpy()
        rows, cols = target.view.shape
        pads = flat[1:1 + rows * (cols + target_pad)].reshape(rows, cols + target_pad)[:, cols:]
        assert (pads == 7.0).all() and flat[0] == 7.0                # nothing is written beside the matrix
    return target


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V,layout,pad,shift,top", SHAPES)
def test_gradient(N, V, layout, pad, shift, top, kind):
    rng = np.random.default_rng(N * 5 + V)
    v, y = logits(rng, N, V)
    y[rng.random(N) < 0.1] = V + 3
    for terms, add, in_place, target_pad in (("lhz", False, False, 3), ("l", False, True, 0), ("hz", True, False, 0)):
        grad_case(Matrix(v, kind, layout, pad, shift), y, rng, target_pad, in_place, add, terms)


def test_gradient_without_arrays_and_in_place_sum():
    rng = np.random.default_rng(8)
    v, y = logits(rng, 9, 77)
    for layout in ("class", "case"):
        grad_case(Matrix(v, "f32", layout), y, rng, arrays=False, terms="lz")
        grad_case(Matrix(v, "f32", layout), y, rng, in_place=True, add=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["class", "case"])
@pytest.mark.parametrize("N,V", MASK_SHAPES)
def test_gradient_of_ruled_out_classes_and_extremes(N, V, layout, kind):
    rng = np.random.default_rng(V + 1)
    v, y = logits(rng, N, V)
    top_value = float(torch_().finfo(dtypes()[kind][0]).max)
    v[0] = -INF
    v[1] = -INF
    v[1, V // 2] = 1.5
    y[1] = V // 2 - 1
    v[2] = -top_value
    v[3] = -top_value
    v[3, [0, V - 1]] = [2.0, 2.0]
    v[4, ::2] = -INF
    v[5, 1], v[5, V - 1] = top_value, -top_value
    grad_case(Matrix(v, kind, layout), y, rng)
    v[1, 2] = INF
    v[2, V - 1] = np.nan
    x = Matrix(v, kind, layout)
    got = grad_case(x, y, rng, terms="l").rows()
    assert np.isnan(got[[1, 2]]).all() and np.isfinite(got[[0, 3, 4, 5]]).all()


def test_other_streams_and_graphs():
    """On a stream of its own, and captured: every replay gives the eager call's bits, with work of the program's own in between."""
    t, m = torch_(), mc()
    rng = np.random.default_rng(11)
    for N, V, layout, top in ((128, 10, "class", 5), (128, 1000, "class", 5), (1, 131072, "case", 20), (600, 5000, "case", 20)):
        v, y = logits(rng, N, V)
        x = Matrix(v, "bf16", layout)
        want = forward(x, y, top)
        stream = t.cuda.Stream()
        stream.wait_stream(t.cuda.current_stream())
        outs = {}
        with t.cuda.stream(stream):
            forward(x, y, top, stream=stream.cuda_stream, outs=outs)
        stream.synchronize()
        for k in want:
            assert np.array_equal(outs[k].cpu().numpy(), want[k], equal_nan=True)
        size = m.lib().mc_log_probs_workspace_bytes(x.code, x.cs, x.ns, N, V, top)
        target = t.zeros_like(x.view)
        target = t.empty_strided(x.view.shape, x.view.stride(), dtype=x.view.dtype, device="cuda").zero_()

        def calls(s):
            m.call("mc_log_probs", x.view.data_ptr(), x.code, x.cs, x.ns, outs["y"].data_ptr(), 3, N, V, outs["logp"].data_ptr(), outs["H"].data_ptr(),
                   outs["stats"].data_ptr(), outs["classes"].data_ptr(), outs["top"].data_ptr(), top, outs["work"].data_ptr(), size, s)
            m.call("mc_log_probs_grad", x.view.data_ptr(), x.code, x.cs, x.ns, outs["y"].data_ptr(), 3, N, V, outs["stats"].data_ptr(), outs["H"].data_ptr(),
                   None, -1.0, None, 0.1, None, 0.01, target.data_ptr(), x.cs, x.ns, 0, s)
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph, stream=stream):
            calls(stream.cuda_stream)
        for i in range(4):
            other = t.from_numpy(rng.standard_normal((N, V)).astype(np.float32)).cuda().to(t.bfloat16)
            x.view.copy_(other.t() if layout == "class" else other)
            outs["work"].fill_(i)
            graph.replay()
            t.cuda.synchronize()
            got = {k: outs[k].clone() for k in want}
            got["grad"] = target.clone()
            calls(t.cuda.current_stream().cuda_stream)
            t.cuda.synchronize()
            for k in want:
                assert t.equal(got[k], outs[k]), (k, i)
            assert t.equal(got["grad"], target)


def test_two_calls_at_once():
    """Two streams, two workspaces: neither sees the other."""
    t = torch_()
    rng = np.random.default_rng(12)
    v, y = logits(rng, 4, 100003)
    w, z = logits(rng, 4, 100003)
    a, b = Matrix(v, "f32", "case"), Matrix(w, "f32", "case")
    want = forward(a, y, 20), forward(b, z, 20)
    s1, s2 = t.cuda.Stream(), t.cuda.Stream()
    t.cuda.synchronize()
    for _ in range(5):
        o1, o2 = {}, {}
        with t.cuda.stream(s1):
            forward(a, y, 20, stream=s1.cuda_stream, outs=o1)
        with t.cuda.stream(s2):
            forward(b, z, 20, stream=s2.cuda_stream, outs=o2)
        t.cuda.synchronize()
        for o, e in ((o1, want[0]), (o2, want[1])):
            for k in e:
                assert np.array_equal(o[k].cpu().numpy(), e[k])


def test_agrees_with_the_softmax_and_logreg_kernels():
    """The same numbers as mc_softmax + mc_compute_logreg_cost + mc_compute_logreg_softmax_grad, for the framework's own layout and labels."""
    t, m = torch_(), mc()
    rng = np.random.default_rng(13)
    for N, V in ((128, 10), (128, 1000)):
        v, y = logits(rng, N, V)
        x = Matrix(v, "f32", "class")
        yy = t.as_tensor(y, dtype=t.float32).cuda()
        probs, lp, correct, grad, mine = (t.zeros(s, device="cuda") for s in ((V, N), (N,), (N,), (V, N), (V, N)))
        m.call("mc_softmax", x.view.data_ptr(), probs.data_ptr(), N, V, None)
        m.call("mc_compute_logreg_cost", yy.data_ptr(), probs.data_ptr(), lp.data_ptr(), correct.data_ptr(), N, V, None)
        m.call("mc_compute_logreg_softmax_grad", yy.data_ptr(), probs.data_ptr(), grad.data_ptr(), 0, 0.5, N, V, None)
        got = forward(x, y, 0, label_type=0)
        D = V + 200.0                                             # one lane adds a case's classes there
        assert np.abs(got["logp"] - lp.cpu().numpy()).max() <= U * 4 * D + U * 8 * np.abs(got["logp"]).max()
        stats = t.from_numpy(got["stats"]).cuda()
        m.call("mc_log_probs_grad", x.view.data_ptr(), 0, x.cs, x.ns, yy.data_ptr(), 0, N, V, stats.data_ptr(), None, None, 0.5, None, 0.0, None, 0.0,
               mine.data_ptr(), N, 1, 0, None)
        assert (mine - grad).abs().max().item() <= U * 4 * D
