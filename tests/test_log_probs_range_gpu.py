"""mc_log_probs / mc_log_probs_grad where the largest logit of a case is far from zero: finite masks of -1e10 or -1e30 over whole cases
and over single parts of them, maxima up to the type's largest value, neighbours one step apart.

The bounds are test_log_probs_gpu's.  They hold here too: a term exp(x - m) is off by (|t| + 8) u relative whatever m is, because
x - m has no rounding where exp(x - m) matters beside 1 (x and m within a factor of 2 of one another: the difference is exact), and the largest
logit itself has t = 0 exactly or a residue of |m| 2^-24 < 0.1 that is known and taken back."""
import numpy as np
import pytest

from oracle import golden as G
from test_log_probs_gpu import INF, Matrix, check, dtypes, forward, grad_case, logits, mc, same, torch_

pytestmark = pytest.mark.gpu

SIZES = [1.0, 5e4, 1e6, 1048575.0, 2.0 ** 20, 3e7, 1e9, 1.5e9, 2.0 ** 30, 3e9, 1e10, 1e20, 1e30, 1e37, 9.9e37, 1e38, 3e38]


def rounded(values, kind):
    t = torch_()
    return t.from_numpy(np.atleast_1d(np.asarray(values, np.float32))).to(dtypes()[kind][0]).double().numpy()


def below(m, kind):
    """The next smaller value of the type."""
    t = torch_()
    dtype = dtypes()[kind][0]
    v = t.tensor([m], dtype=dtype)
    bits = v.view(t.int32 if kind == "f32" else t.int16)
    bits += -1 if m > 0 else 1
    return float(v.double()[0])


def cases_of(rng, V, kind):
    """One case of every sort for every size that the type holds."""
    rows = []
    most = float(torch_().finfo(dtypes()[kind][0]).max)
    for size in SIZES:
        for sign in (-1.0, 1.0):
            m = float(rounded(sign * size, kind)[0]) if size <= most else INF
            if not abs(m) < most:
                continue
            ordinary, lower = rng.standard_normal(V) * 2.5, below(m, kind)
            rows.append(np.full(V, m))                                            # uniform: ln V whatever m is
            rows.append(np.where(rng.random(V) < 0.5, m, lower))                  # neighbours
            rows.append(np.where(np.arange(V) == V // 3, m, np.where(np.arange(V) % 3 == 1, lower, -INF)))
            rows.append(np.where(np.arange(V) < V // 2, m, ordinary))             # parts of one, parts of the other
            rows.append(np.where(rng.random(V) < 0.5, m, ordinary))
    return np.stack(rows)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["class", "case"])
@pytest.mark.parametrize("V", [1, 3, 50, 1000, 5000, 40000])
def test_maxima_of_every_size(V, layout, kind):
    rng = np.random.default_rng(V)
    v = cases_of(rng, V, kind)
    y = rng.integers(0, V, len(v))
    x = Matrix(v, kind, layout)
    for top, entropy in ((5, True), (0, True), (0, False)):
        check(x, y, top, forward(x, y, top, entropy=entropy), entropy=entropy)
    grad_case(x, y, rng)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("N,V,top", [(1, 131072, 20), (3, 131072, 20), (2, 40000, 0)])
def test_one_masked_part(N, V, top, kind):
    """Few cases, split into many parts: a mask over the tail, over a stretch in the middle, over everything but a few classes."""
    rng = np.random.default_rng(N)
    for mask in (-1e9, -1e10, -1e30, -1e37, float(rounded(-3e38, kind)[0])):
        for a, b in ((V - 20000, V), (4096, 16384), (3, V), (0, V - 2), (0, V)):
            v, y = logits(rng, N, V)
            v[:, a:b] = mask
            x = Matrix(v, kind, "case")
            check(x, y, top, forward(x, y, top))


def test_a_step_under_a_finite_mask_is_finite():
    """Masks of -1e30 over whole cases and parts of others: log probabilities, gradient and its norm, one after the other."""
    t, m = torch_(), mc()
    rng = np.random.default_rng(7)
    for layout in ("class", "case"):
        for kind in ("f32", "bf16"):
            v, y = logits(rng, 40, 1000)
            v[::4] = -1e30
            v[1::4, 300:] = -1e30
            y[1::4] = rng.integers(0, 300, len(y[1::4]))
            x = Matrix(v, kind, layout)
            got = forward(x, y)
            check(x, y, 0, got)
            stats, yy = t.from_numpy(got["stats"]).cuda(), t.as_tensor(y, dtype=t.int32).cuda()
            target = t.zeros(x.view.shape, dtype=x.view.dtype, device="cuda")
            cs, ns = (target.stride(0), 1) if layout == "class" else (1, target.stride(0))
            m.call("mc_log_probs_grad", x.view.data_ptr(), x.code, x.cs, x.ns, yy.data_ptr(), 3, 40, 1000, stats.data_ptr(), None, None, 1.0, None, 0.0,
                   None, 0.0, target.data_ptr(), cs, ns, 0, None)
            exact = target.double().cpu().numpy()
            spans = m.grad_spans([(target.data_ptr(), 0, target.numel(), 1.0, x.code, x.code)])
            dev = t.from_numpy(np.frombuffer(bytes(spans), dtype=np.uint8).copy()).cuda()
            nf, work = t.zeros(2, device="cuda"), t.zeros(m.lib().mc_grad_norm_workspace_bytes(len(spans)), dtype=t.uint8, device="cuda")
            m.call("mc_grad_norm", dev.data_ptr(), len(spans), 1.0, nf.data_ptr(), work.data_ptr(), work.numel(), None)
            norm, factor = nf.cpu().numpy()
            true, share = G.grad_norm([exact], [1.0], 1.0)
            assert np.isfinite(true) and abs(norm - true) <= true * 2.51 * 2.0 ** -24 and factor > 0
