"""The Node host where only the first of its two addons was built: a program of one sequence runs, and one of many is told what is missing."""
import json
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
PACKAGE = os.path.join(os.path.dirname(HERE), "webllm_amd")
NODE = shutil.which("node")


@pytest.mark.skipif(NODE is None, reason="node not installed")
def test_first_addon_alone(tmp_path):
    os.makedirs(tmp_path / "js"), os.makedirs(tmp_path / "lib")
    shutil.copy(os.path.join(PACKAGE, "js", "index.js"), tmp_path / "js")
    for name in ("qlinear_napi.node", "libqlinear.so"):
        os.symlink(os.path.join(PACKAGE, "lib", name), tmp_path / "lib" / name)
    r = subprocess.run([NODE, os.path.join(HERE, "js", "addons_check.js"), str(tmp_path / "js" / "index.js")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    got = json.loads(r.stdout.strip().splitlines()[-1])
    assert got["functions"] > 10 and got["names"] and got["config"] == 128
    for said in (got["attend"], got["addon"]):
        assert "not built" in said and "qlinear_batch_napi.node" in said and "__graft_entry__" in said, said
