"""mc_log_probs with signalling NaN among the logits: bit patterns that arithmetic never gives, but memory that was never written and damaged
files do."""
import numpy as np
import pytest

from test_log_probs_gpu import INF, Matrix, check, forward, logits, torch_

pytestmark = pytest.mark.gpu

PATTERNS = {"f32": (0x7f800001, -0x7fffff), "f16": (0x7c01, -0x3ff), "bf16": (0x7f81, -0x7f)}     # both signs, as signed integers


def signal(x, where):
    """NaN that signal, at `where` (numCases, numOut), in the matrix and in what the oracle is given."""
    t = torch_()
    bits = x.store.view(t.int32 if x.code == 0 else t.int16)
    kind = {0: "f32", 1: "f16", 2: "bf16"}[x.code]
    cases, classes = np.nonzero(where)
    at = t.as_tensor(x.view.storage_offset() + classes * x.cs + cases * x.ns, dtype=t.int64, device="cuda")
    pattern = t.as_tensor(np.resize(PATTERNS[kind], len(cases)), dtype=bits.dtype, device="cuda")
    bits[at] = pattern
    x.exact = np.where(where, np.nan, x.exact)
    assert np.array_equal(np.isnan(x.rows()), where)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["class", "case"])
@pytest.mark.parametrize("N,V", [(9, 3), (9, 10), (9, 60), (9, 1000), (40, 1000), (9, 5000), (9, 40000), (2, 131072)])
def test_signalling_nan(N, V, layout, kind):
    """A NaN of either sort is never named and hides nobody: the maximum and the best classes are those of the numbers, all the rest is NaN."""
    rng = np.random.default_rng(V)
    v, y = logits(rng, N, V)
    where = rng.random((N, V)) < 0.3
    best = rng.integers(0, V, N)
    v[np.arange(N), best] = 30.0
    where[np.arange(N), best] = False
    where[0] = False                                     # none here,
    where[0, (best[0] + 1) % V] = True                   # but beside the best
    where[1] = False
    where[1, best[1] - 1] = True
    if N > 4:
        where[2] = True                                  # nothing else
        where[3] = False
        v[4] = -INF                                      # nothing else but ruled-out classes
    x = Matrix(v, kind, layout)
    signal(x, where)
    for top in (5, 1, 0):
        check(x, y, top, forward(x, y, top))
    got = forward(x, y, 0, entropy=False)
    check(x, y, 0, got, entropy=False)
