"""libkernel.startPredictions with a layer that has more outputs than the net has classes: labels that its cost layer would read beyond the
probabilities with are refused, the others are predicted."""
import os
import subprocess
import sys

import numpy as np
import pytest

from oracle import golden as G

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
U = 2.0 ** -24


def test_labels_beyond_the_classes_of_the_cost_layer(tmp_path):
    path = str(tmp_path / "res.npz")
    r = subprocess.run([sys.executable, "-u", os.path.join(HERE, "run_predict_labels.py"), "--layer=fc64", "--out=" + path], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, "child failed:\n" + r.stdout[-3000:] + "\n" + r.stderr[-3000:]
    r = dict(np.load(path))
    assert len(r["refused"]) == 3
    assert all("logprob" in str(m) for m in r["refused"][:2]) and "fc64" in str(r["refused"][2])
    assert int(r["numCases"]) == 50
    e = G.log_probs(r["ftrs"].astype(np.float64), r["labels"][0].astype(np.int64), 3)
    # the bounds of test_predictions, for 64 outputs
    D = 64 / 32.0 + 124.0
    tol = U * (D + np.abs(e["logSum"]) + 2)
    assert (abs(r["out"][:, 0] - e["logp"]) <= tol + 3 * U * abs(e["logp"])).all()
    assert (abs(r["out"][:, 1] - e["entropy"]) <= tol + U * (2 * D + 2) * abs(e["meanShift"]) + U * abs(e["entropy"])).all()
    assert np.array_equal(r["out"][:, 2:5], e["classes"].T)
