"""The check that a call's stream belongs to the current device: where the runtime cannot tell, its answer is not taken for the launch's."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
MC_OK, MC_ELAUNCH = 0, -2


def test_a_query_that_fails_is_not_the_launchs_error(tmp_path):
    exe = str(tmp_path / "stream_check")
    subprocess.check_call(["hipcc", "--offload-arch=gfx950", "--cuda-host-only", "-x", "hip", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"),
                           "-I", os.path.join(ROOT, "cuda-convnet_amd", "csrc", "kernels"), os.path.join(HERE, "stream_check_main.cpp"), "-o", exe])
    rows = dict((line.split()[0], tuple(map(int, line.split()[1:]))) for line in subprocess.check_output([exe], text=True).splitlines())
    assert rows["same"] == (1, MC_OK) and rows["null"] == (1, MC_OK)
    assert rows["other"] == (0, MC_OK)
    assert rows["stream-unknown"] == (1, MC_OK)
    assert rows["device-unknown"] == (1, MC_OK)
    assert rows["failed-before"] == (1, MC_ELAUNCH)          # an error that was there before is still reported
