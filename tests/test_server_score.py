"""POST /score and --kv, as far as they need no GPU."""
import os
import subprocess

import pytest

from test_server import request
from voxelengine import engine as ve

SERVER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "opure-voxelengine_b200", "opure_server")


def test_route_without_engine():
    with ve.Server() as s:
        assert request(s.port, "POST", "/score", b'{"tokens":[1]}')[0] == 503
        assert request(s.port, "GET", "/score")[0] == 405
        assert request(s.port, "POST", "/scores", b'{"tokens":[1]}')[0] == 404


@pytest.mark.skipif(not os.path.exists(SERVER), reason="opure_server not built")
def test_kv_option(tmp_path):
    """fp4 is taken (and the model then asked for); anything else is a usage error."""
    def run(*args):
        return subprocess.run([SERVER, "--model", str(tmp_path / "none"), *args], capture_output=True, text=True, timeout=60)

    for bad in (("--kv", "fp8"), ("--kv",)):
        r = run(*bad)
        assert r.returncode == 2 and "[--kv fp4]" in r.stdout
    r = run("--kv", "fp4", "--weights", "mxfp4")
    assert r.returncode == 1 and r.stderr.startswith("opure_server:") and "usage" not in r.stdout
