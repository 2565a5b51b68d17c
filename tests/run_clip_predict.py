"""Child process of test_clip_predict_gpu.py (one model per process): trains one net, one synthetic batch per entry of --clips with
that gradient bound set before it, records norm and factor after each, or writes a layer's features and predictions."""
import argparse
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "cuda-convnet_amd"))
import modelutil  # noqa: E402


def refused(kind, fn, *args):
    try:
        fn(*args)
    except kind:
        return
    raise AssertionError("%s%r was not refused" % (fn.__name__, args))


def weights(layers, res, tag):
    for l in layers:
        for i, w in enumerate(l.get("weights", [])):
            res["%s:W:%s:%d" % (tag, l["name"], i)] = np.array(w)
            res["%s:I:%s:%d" % (tag, l["name"], i)] = np.array(l["weightsInc"][i])
        if "weights" in l:
            res["%s:W:%s:b" % (tag, l["name"])] = np.array(l["biases"])
            res["%s:I:%s:b" % (tag, l["name"])] = np.array(l["biasesInc"])


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--net", required=True)
    ap.add_argument("--cases", type=int, required=True)
    ap.add_argument("--mini", type=int, required=True)
    ap.add_argument("--clips", default="", help="gradient bounds, one batch each; 'keep' sets none")
    ap.add_argument("--poison", type=int, default=-1, help="the batch of --clips whose first case holds a NaN")
    ap.add_argument("--single-rank-comm", type=int, default=0)
    ap.add_argument("--predict", default="", help="layer name: its features, and predictions from it with --top alternatives")
    ap.add_argument("--top", type=int, default=0)
    ap.add_argument("--between", type=int, default=0, help="predictions of that many cases after each batch of --clips")
    ap.add_argument("--out", required=True)
    a = ap.parse_args()
    import libkernel
    layers, dims, classes = modelutil.load_net(a.net, seed=42, init_w=0.05)
    data = modelutil.synthetic_batch(dims, classes, a.cases)
    libkernel.initModel(layers, a.mini, 0)
    libkernel.setSeed(77)
    if a.single_rank_comm:
        libkernel.initComm(0, 1, libkernel.commUniqueId(), 1)
    res = {}
    if a.predict:
        idx = [i for i, l in enumerate(layers) if l["name"] == a.predict][0]
        ftrs = np.full((a.cases, layers[idx]["outputs"]), np.nan, np.float32)
        libkernel.startFeatureWriter(data + [ftrs], idx)
        fcosts = libkernel.finishBatch()
        out = np.full((a.cases, 2 + 2 * a.top), np.nan, np.float32)
        refused(ValueError, libkernel.startPredictions, data + [out], len(layers), a.top)
        refused(ValueError, libkernel.startPredictions, data + [out], idx, 33)
        refused(ValueError, libkernel.startPredictions, data + [out], idx, -1)
        refused(ValueError, libkernel.startPredictions, [data[0], out], idx, a.top)
        for wrong in (np.zeros((a.cases, 3 + 2 * a.top), np.float32), np.zeros((a.cases + 1, 2 + 2 * a.top), np.float32),
                      np.zeros((a.cases, 2 + 2 * a.top), np.float32, order="F")):
            libkernel.startPredictions(data + [wrong], idx, a.top)
            refused(RuntimeError, libkernel.finishBatch)
        for label in (-1, layers[idx]["outputs"], float("nan")):
            bad = data[1].copy()
            bad[0, 77] = label
            libkernel.startPredictions([data[0], bad, out], idx, a.top)
            refused(RuntimeError, libkernel.finishBatch)
        libkernel.startPredictions(data + [out], idx, a.top)
        n = libkernel.finishBatch()[1]
        above = [i for i, l in enumerate(layers) if l["type"] == "softmax" and idx in l["inputs"]]
        again = np.full_like(out, np.nan)
        libkernel.startPredictions(data + [again], above[0], a.top)
        libkernel.finishBatch()
        np.savez(a.out, ftrs=ftrs, out=out, again=again, labels=data[1], numCases=n, cost=fcosts[0]["logprob"])
        return
    refused(ValueError, libkernel.setGradClip, -1.0)
    refused(ValueError, libkernel.setGradClip, float("nan"))
    refused(RuntimeError, libkernel.getGradNorm)
    libkernel.syncWithHost()
    weights(layers, res, "start")
    norms = []
    for b, c in enumerate(a.clips.split(",")):
        if c != "keep":
            libkernel.setGradClip(float(c))
        d = [x.copy() for x in data]
        if b == a.poison:
            d[0][:, 0] = np.nan
        libkernel.startBatch(d, 0)
        refused(RuntimeError, libkernel.setGradClip, 7.0)       # a batch is under way
        res["case:%d" % b] = libkernel.finishBatch()[1]
        if c in ("keep", "0"):
            refused(RuntimeError, libkernel.getGradNorm)
            norms.append((0.0, 1.0))
        else:
            norms.append(libkernel.getGradNorm())
        libkernel.syncWithHost()
        weights(layers, res, str(b))
        if a.between:
            out = np.full((a.between, 2 + 2 * 3), np.nan, np.float32)
            soft = [i for i, l in enumerate(layers) if l["type"] == "softmax"][0]
            libkernel.startPredictions([np.ascontiguousarray(x[:, :a.between]) for x in data] + [out], soft, 3)
            res["cost:%d" % b] = libkernel.finishBatch()[0]["logprob"]
            res["out:%d" % b] = out
    prof = libkernel.getProfile()
    np.savez(a.out, norms=np.array(norms), replays=prof["net/step_graph:replays"][0], forked=prof["net/step_fork:steps"][0], **res)


if __name__ == "__main__":
    main()
