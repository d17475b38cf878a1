"""bench.py where the reference's CPU graph is not built: the reference arm says so in one
line and ends well, and the framework's own line has the reason in its place."""
import importlib
import json
import os
import subprocess
import sys

import pytest

from conftest import ROOT


@pytest.mark.parametrize("extra", [[], ["--gpus", "1", "--steps", "20", "--warmup", "5"], ["--config", "3"],
                                   ["--config", "3", "--http"]])
def test_reference_arm_says_that_it_is_unavailable(tmp_path, extra):
    code = ("import sys, oracle, bench; oracle.REF_SO = bench.SERVER_CPU_BIN = bench.os.path.join(bench.ROOT, 'none.so'); "
            "bench.main()")
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([ROOT, os.path.join(ROOT, "oracle")]))
    r = subprocess.run([sys.executable, "-c", code, "--impl", "reference", *extra], cwd=tmp_path, env=env,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = r.stdout.strip().splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert line["impl"] == "reference" and "none.so is not built" in line["unavailable"]


def test_own_line_has_the_reason(monkeypatch):
    oracle, bench = importlib.import_module("oracle"), importlib.import_module("bench")
    monkeypatch.setattr(oracle, "REF_SO", os.path.join(ROOT, "none.so"))
    res = bench.cpu_baseline_run("no model is opened", (4,), 1, 1, seed=1)
    assert set(res) == {"unavailable"} and "none.so" in res["unavailable"]
