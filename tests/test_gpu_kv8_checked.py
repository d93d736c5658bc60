"""The 8-bit paged cache's small cases through the checked build of the library, which holds every pointer
argument against the allocation it lies in."""
from __future__ import annotations

import json
import os
import subprocess
import sys

import pytest

from conftest import ROOT
from test_gpu_bounds import _env, bounds_lib  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def test_kv8_cases_run_clean_under_the_checked_build(gpu, bounds_lib):  # noqa: F811
    cmd = [sys.executable, "-m", "pytest", os.path.join(ROOT, "tests", "test_gpu_kv8.py"),
           os.path.join(ROOT, "tests", "test_gpu_kv8_edges.py"), "-m", "gpu", "-q", "-x", "-p", "no:cacheprovider",
           "-k", "not fill_the_gpu and not four and not many and not 32_bits and not 20000 and not heads"]
    r = subprocess.run(cmd, env=_env(bounds_lib), capture_output=True, text=True, cwd=ROOT)
    tail = (r.stdout + r.stderr)[-3000:]
    assert r.returncode == 0, tail
    line = [l for l in r.stdout.splitlines() if l.startswith("[bounds]")]
    assert line, tail
    rec = json.loads(line[-1][len("[bounds]"):])
    assert rec["enabled"] == 1 and rec["violations"] == 0 and rec["checked_spans"] > 1000, rec
