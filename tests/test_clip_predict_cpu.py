"""The clipping option of the driver and what libkernel's clipping and prediction calls answer before there is a model."""
import numpy as np
import pytest


def test_clip_norm_option_parses():
    import convnet
    op = convnet.ConvNet.get_options_parser()
    assert op.options["clip_norm"].default == 0.0 and type(op.options["clip_norm"].default) is float
    op.set_value("clip_norm", "2.5")
    assert op.get_value("clip_norm") == 2.5
    with pytest.raises(Exception, match="float"):
        op.set_value("clip_norm", "much")


def test_calls_without_a_model_are_refused():
    import libkernel
    for fn, args in ((libkernel.setGradClip, (1.0,)), (libkernel.getGradNorm, ()), (libkernel.startPredictions, ([np.zeros((1, 1), np.float32)] * 3, 0, 1))):
        with pytest.raises(RuntimeError):
            fn(*args)
