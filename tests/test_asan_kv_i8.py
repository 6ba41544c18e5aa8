"""Host-side AddressSanitizer run of the int8 cache's entry points: tests/asan/kv_i8_driver.cpp against the library whose
host-only sources are compiled with ASan (built by __graft_entry__.build()).  No GPU is used."""

import os
import subprocess
from pathlib import Path

import pytest

DRIVER = Path(__file__).resolve().parents[1] / "wrinklefree-monorepo_amd" / "_build" / "asan" / "kv_i8_driver"


@pytest.mark.skipif(not DRIVER.exists(), reason="ASan driver not built (run __graft_entry__.build())")
def test_entry_points_under_asan():
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1:halt_on_error=1")
    res = subprocess.run([str(DRIVER)], capture_output=True, text=True, env=env, timeout=300)
    out = res.stdout + res.stderr
    assert "AddressSanitizer" not in out, out[-4000:]
    assert res.returncode == 0 and "kv_i8: 0 failures" in res.stdout, out[-4000:]
