"""How mc_grad_spans cuts: the kernels take spans of at most 4096 elements (mc_clip_grads leaves out what lies beyond), and every span but a
tensor's first begins on a 128-byte line of what is written, or of what is read where nothing is."""
import numpy as np
import pytest

BASE = 1 << 20
SIZE = {0: 4, 1: 2, 2: 2}


@pytest.mark.parametrize("grad_type,out_type", [(0, 0), (1, 1), (2, 2), (2, 0), (0, 1), (1, 0), (0, None), (2, None)])
def test_spans_are_short_and_cut_at_lines(grad_type, out_type):
    import mckernels as m
    rng = np.random.default_rng(3)
    tensors, at, to = [], BASE, BASE << 20
    written = grad_type if out_type is None else out_type
    for n in [1, 31, 4064, 4095, 4096, 4097, 8192, 12289, 100003, 0, 1 << 20] + [int(v) for v in rng.integers(1, 30000, 60)]:
        at += int(rng.integers(0, 64)) * SIZE[grad_type]
        to += int(rng.integers(0, 64)) * SIZE[written]
        tensors.append((at, 0 if out_type is None else to, n, 1.0, grad_type, written))
        at += n * SIZE[grad_type]
        to += n * SIZE[written]
    spans = iter(m.grad_spans(tensors))
    for grad, out, n, *_ in tensors:
        done = 0
        while done < n:
            sp = next(spans)
            assert 0 < sp.count <= 4096 and sp.grad == grad + done * SIZE[grad_type]
            assert (sp.out or 0) == (out + done * SIZE[written] if out else 0)
            assert done == 0 or (sp.out or sp.grad) % 128 == 0
            done += sp.count
        assert done == n
    assert next(spans, None) is None


def test_spans_of_the_largest_single_tensors():
    """A tensor that begins off a line: the first span is the shorter one, all that follow but the last are whole."""
    import mckernels as m
    for shift in (0, 4, 60, 124):
        counts = [s.count for s in m.grad_spans([(BASE + shift, 0, 1 << 22, 1.0, 0, 0)])]
        assert counts[0] == 4096 - shift // 4 and set(counts[1:-1]) == {4096} and sum(counts) == 1 << 22
