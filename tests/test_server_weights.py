"""The server executable's --weights option, without a GPU."""
import os
import subprocess

import pytest

SERVER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "opure-voxelengine_b200", "opure_server")
pytestmark = pytest.mark.skipif(not os.path.exists(SERVER), reason="opure_server not built")


def run(*args):
    return subprocess.run([SERVER, *args], capture_output=True, text=True, timeout=60)


def test_weights_option(tmp_path):
    """mxfp4 is taken (and the model then asked for); anything else is a usage error."""
    for bad in (("--weights", "int3"), ("--weights",)):
        r = run("--model", str(tmp_path / "none"), *bad)
        assert r.returncode == 2 and "[--weights mxfp4]" in r.stdout
    r = run("--model", str(tmp_path / "none"), "--weights", "mxfp4")
    assert r.returncode == 1 and r.stderr.startswith("opure_server:") and "usage" not in r.stdout
