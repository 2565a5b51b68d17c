"""Child process of test_predict_labels_gpu.py (one model per process): predictions from a layer with more outputs than the net has classes."""
import argparse
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "cuda-convnet_amd"))
import modelutil  # noqa: E402


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--layer", required=True)
    ap.add_argument("--out", required=True)
    a = ap.parse_args()
    import libkernel
    layers, dims, classes = modelutil.load_net("80sec", seed=42, init_w=0.05)
    data = modelutil.synthetic_batch(dims, classes, 50)
    libkernel.initModel(layers, 32, 0)
    idx = [i for i, l in enumerate(layers) if l["name"] == a.layer][0]
    wide = layers[idx]["outputs"]
    assert wide > classes
    refused = []
    for label in (classes, wide - 1, wide):
        bad = data[1].copy()
        bad[0, 41] = label
        out = np.full((50, 8), np.nan, np.float32)
        libkernel.startPredictions([data[0], bad, out], idx, 3)
        try:
            libkernel.finishBatch()
        except RuntimeError as e:
            refused.append(str(e))
        assert np.isnan(out).all()
    ftrs, out = np.full((50, wide), np.nan, np.float32), np.full((50, 8), np.nan, np.float32)
    libkernel.startFeatureWriter(data + [ftrs], idx)
    libkernel.finishBatch()
    libkernel.startPredictions(data + [out], idx, 3)
    n = libkernel.finishBatch()[1]
    np.savez(a.out, refused=np.array(refused), ftrs=ftrs, out=out, labels=data[1], numCases=n)


if __name__ == "__main__":
    main()
