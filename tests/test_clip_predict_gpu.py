"""Gradient clipping in the training step (libkernel.setGradClip / getGradNorm, convnet.py --clip-norm) and predictions of a test pass
(libkernel.startPredictions): eager, forked and captured steps, data parallelism of one rank, and the two used together with training."""
import os
import re
import subprocess
import sys
import tempfile

import numpy as np
import pytest

import modelutil
from oracle import golden as G

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "cuda-convnet_amd")
U = 2.0 ** -24     # half a step of float32, relative


def run(_env=None, **kw):
    out = os.path.join(tempfile.mkdtemp(prefix="cp_"), "res.npz")
    cmd = [sys.executable, "-u", os.path.join(HERE, "run_clip_predict.py"), "--out", out]
    for k, v in kw.items():
        cmd += ["--%s=%s" % (k.replace("_", "-"), v)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300, env=dict(os.environ, **(_env or {})))
    assert r.returncode == 0, "child failed:\n" + r.stdout[-3000:] + "\n" + r.stderr[-3000:]
    return dict(np.load(out))


def same_weights(a, b, tag_a, tag_b):
    n = 0
    for k in a:
        if k.startswith(tag_a + ":"):
            assert np.array_equal(a[k], b[tag_b + k[len(tag_a):]]), k
            n += 1
    assert n


def rates(net):
    """{weight key: (learning rate, weight decay)}"""
    layers = modelutil.load_net(net, seed=42, init_w=0.05)[0]
    out = {}
    for l in layers:
        for i in range(len(l.get("weights", []))):
            out["%s:%d" % (l["name"], i)] = (l["epsW"][i], l["wc"][i])
        if "weights" in l:
            out[l["name"] + ":b"] = (l["epsB"], 0.0)
    return out


@pytest.mark.parametrize("net", ["nin-tiny", "80sec", "conv-local"])
def test_one_step_is_scaled_by_its_norm(net):
    """A first step (increments 0) leaves inc = g - wc*eps*W, g being eps times the gradient.  Every float32 operation on the way errs by
    at most U times |g| + |d|, d = wc*eps*W: four of them (the product wc*eps, its product with W, the sum, the stored value) before g
    is back in 64 bits, which moves the norm by at most the norm of those errors over eps; scale and the norm's own rounding: 3 U."""
    plain = run(net=net, cases=32, mini=32, clips="keep")
    free = run(net=net, cases=32, mini=32, clips="inf")
    same_weights(plain, free, "0", "0")                    # measuring alone changes nothing
    norm, factor = free["norms"][0]
    assert factor == 1.0 and norm > 0
    g, d, sq, err = {}, {}, 0.0, 0.0
    for k, (eps, wc) in rates(net).items():
        inc, w0 = plain["0:I:" + k].astype(np.float64), plain["start:W:" + k].astype(np.float64)
        assert not plain["start:I:" + k].any()
        if eps <= 0:
            continue
        d[k] = np.float64(np.float32(wc)) * np.float32(eps) * w0
        g[k] = inc + d[k]
        sq += ((g[k] / np.float32(eps)) ** 2).sum()
        err += ((4 * U * (abs(g[k]) + abs(d[k])) / np.float32(eps)) ** 2).sum()
    assert abs(norm - np.sqrt(sq)) <= 3 * U * norm + np.sqrt(err)
    bound = np.float32(norm / 3)
    tight = run(net=net, cases=32, mini=32, clips=repr(float(bound)))
    assert tight["norms"][0][0] == norm and abs(tight["norms"][0][1] - bound / norm) <= 2 * U * bound / norm
    f = tight["norms"][0][1]
    for k in g:                                            # errors of g as above, then the same operations again and the product with f
        want = f * g[k] - d[k]
        tol = 10 * U * (abs(g[k]) + abs(d[k]))
        got = tight["0:I:" + k].astype(np.float64)
        assert (abs(got - want) <= tol).all(), k
        w = plain["start:W:" + k].astype(np.float64) + want
        assert (abs(tight["0:W:" + k] - w) <= tol + U * abs(w) + 1e-45).all(), k


def test_captured_and_eager_steps_clip_alike():
    """Replayed graphs take the norm anew in every step, and a bound that is changed, turned off or set again takes effect with the next
    step, not with the setting that a graph was captured under."""
    kw = dict(net="80sec", cases=6 * 32 + 7, mini=32, clips="0.05,inf,0.02,0,0.02")
    graph = run(_env={"MC_STEP_GRAPH": "1"}, **kw)
    eager = run(_env={"MC_NO_STEP_GRAPH": "1", "MC_NO_STEP_FORK": "1"}, **kw)
    mixed = run(**kw)
    assert int(graph["replays"]) >= 5 * 3 and int(eager["replays"]) == 0 and int(eager["forked"]) == 0
    for b in range(5):
        for other in (graph, mixed):
            same_weights(other, eager, str(b), str(b))
            assert np.array_equal(other["norms"][b], eager["norms"][b])
    assert eager["norms"][0][1] < 1 and eager["norms"][1][1] == 1 and eager["norms"][2][1] < 1
    loose = run(net="80sec", cases=6 * 32 + 7, mini=32, clips="keep")
    assert not np.array_equal(loose["0:W:fc10:0"], eager["0:W:fc10:0"])


@pytest.mark.parametrize("env", [{"MC_NO_STEP_GRAPH": "1"}, {"MC_STEP_GRAPH": "1"}])
def test_a_step_without_a_finite_norm_is_dropped(env):
    """One case of NaN in one minibatch a batch: that step changes nothing, and the next batch trains on."""
    r = run(_env=env, net="80sec", cases=32, mini=32, clips="1,1,1,1", poison=2)
    same_weights(r, r, "1", "2")
    assert np.isnan(r["norms"][2][0]) and r["norms"][2][1] == 0
    assert r["norms"][3][1] > 0 and not np.array_equal(r["2:W:fc10:0"], r["3:W:fc10:0"])
    for k in r:
        if k.startswith("3:"):
            assert np.isfinite(r[k]).all(), k


def test_single_rank_group_clips_alike():
    kw = dict(net="nin-tiny", cases=6 * 32, mini=32, clips="0.5")
    a, b = run(_env={"MC_NO_STEP_GRAPH": "1"}, **kw), run(single_rank_comm=1, **kw)
    same_weights(a, b, "0", "0")
    assert np.array_equal(a["norms"], b["norms"]) and int(b["forked"]) > 0


@pytest.mark.parametrize("net,layer,top", [("nin-tiny", "poolg", 5), ("80sec", "fc10", 0), ("80sec", "fc10", 10), ("80sec", "fc10", 32)])
def test_predictions(net, layer, top):
    """Against the 64-bit oracle on the features that the device computed; a ragged tail, more alternatives than
    classes.  The bounds count roundings: of the shift, of each of the V terms and their sum, of the logarithm and the products."""
    cases = 150
    r = run(net=net, cases=cases, mini=64, predict=layer, top=top)
    x = r["ftrs"].astype(np.float64)
    V = x.shape[1]
    e = G.log_probs(x, r["labels"][0].astype(np.int64), min(top, V))
    assert np.array_equal(r["out"], r["again"]) and int(r["numCases"]) == cases
    tol = U * (V / 32.0 + 124.0 + np.abs(e["logSum"]) + 2)
    assert (abs(r["out"][:, 0] - e["logp"]) <= tol + 3 * U * abs(e["logp"])).all()
    D = V / 32.0 + 124.0
    assert (abs(r["out"][:, 1] - e["entropy"]) <= tol + U * (2 * D + 2) * abs(e["meanShift"]) + U * abs(e["entropy"])).all()
    k = min(top, V)
    assert np.array_equal(r["out"][:, 2:2 + k], e["classes"].T.reshape(cases, k))
    assert (abs(r["out"][:, 2 + top:2 + top + k] - e["top"].T.reshape(cases, k)) <= (tol[:, None] + 3 * U * abs(e["top"].T.reshape(cases, k)))).all()
    assert (r["out"][:, 2 + k:2 + top] == -1).all() and (r["out"][:, 2 + top + k:] == -np.inf).all()


@pytest.mark.parametrize("env", [{"MC_NO_STEP_GRAPH": "1"}, {"MC_STEP_GRAPH": "1"}])
def test_predictions_between_training_batches(env):
    """Training goes on to the same bits whether or not the net predicts in between (another number of cases, so that matrices change
    shape under captured steps), and what it predicts is what the cost layer of the same pass saw: the log probabilities add up to its
    cost. A case's bound: 156 U for the log probability (test_predictions' for 10 classes, |ln p| < 5); for the cost a probability off by 100 U
    (a float32 exp of |x - m| < 16 as x and m are rounded, a sum of 10, a division) and a logarithm off by 2 U of 5: below 280 U. Sums are in double."""
    kw = dict(net="80sec", cases=5 * 32, mini=32, clips="0.05,0.05,0.05")
    a, b = run(_env=env, **kw), run(_env=env, between=75, **kw)
    for i in range(3):
        same_weights(a, b, str(i), str(i))
        out, cost = b["out:%d" % i].astype(np.float64), b["cost:%d" % i]
        assert (out[:, 0] > np.log(0.01)).all()
        assert abs(-out[:, 0].sum() - cost[0]) <= 75 * 280 * U
        assert (np.diff(out[:, 5:], axis=1) <= 0).all() and ((out[:, 1] >= 0) & (out[:, 1] <= np.log(10) + 1e-5)).all()
    assert np.array_equal(a["norms"], b["norms"])


def test_clip_norm_option(tmp_path):
    """--clip-norm on the command line, saved with the checkpoint and changed when resuming from it."""
    cfg = ["--layer-def=" + os.path.join(modelutil.CONFIGS, "layers-80sec.cfg"), "--layer-params=" + os.path.join(modelutil.CONFIGS, "layer-params-80sec.cfg")]
    base = ["--data-path=" + str(tmp_path), "--save-path=" + str(tmp_path), "--train-range=1", "--test-range=1", "--test-freq=1",
            "--data-provider=dummy-cn-%d" % (32 * 32 * 3)]

    def driver(args):
        r = subprocess.run([sys.executable, "-u", os.path.join(PKG, "convnet.py")] + args, capture_output=True, text=True, timeout=300, cwd=PKG,
                           env=dict(os.environ, CONVNET_SEED="7"))
        return r.returncode, r.stdout + r.stderr
    rc, out = driver(base + cfg + ["--epochs=1", "--clip-norm=0.25"])
    assert rc == 0 and re.search(r"Largest global norm.*: 0.25", out), out[-3000:]
    ckpt = [d for d in os.listdir(tmp_path) if d.startswith("ConvNet__")][0]
    rc, out = driver(["-f", str(tmp_path / ckpt), "--epochs=2"])
    assert rc == 0 and re.search(r"Largest global norm.*: 0.25", out), out[-3000:]
    rc, out = driver(["-f", str(tmp_path / ckpt), "--epochs=3", "--clip-norm=-1"])
    assert rc != 0 and "maxNorm must be positive" in out, out[-3000:]
