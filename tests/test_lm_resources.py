"""Static resources of libnsparse_lm's kernels, compiled for gfx950 (no GPU): none uses scratch, none asks for more LDS than there is."""
import os
import shutil
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))

import kernel_resources as kr  # noqa: E402

pytestmark = pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc") and shutil.which("hipcc") is None, reason="no hipcc on this box")
UNITS = ("attend_bwd", "attend_fwd", "select", "route")


def test_kernels_fit():
    with ThreadPoolExecutor(max_workers=4) as ex:
        tables = list(ex.map(lambda u: kr.unit_resources("s", "lm/" + u), UNITS))
    for unit, rows in zip(UNITS, tables):
        assert rows, unit
        for r in rows:
            assert r["scratch"] == 0 and r["vspill"] == 0, r["name"]
            assert r["lds"] <= 160 * 1024 and r["occ"] >= 1, r["name"]
