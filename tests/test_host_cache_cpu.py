"""What launchers keep per device: tests/c/host_cache.cc compiled against the header and
run, and the launchers' sources, which hold no table of their own beside it."""

from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parents[1]
CSRC = REPO / "inference-kernel_b200" / "csrc"


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_device_cache(tmp_path):
    exe = tmp_path / "host_cache"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-pthread", f"-I{CSRC}",
                    str(REPO / "tests" / "c" / "host_cache.cc"), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr
    assert run.stdout.count("ok ") == 4


def test_launchers_keep_no_table_for_all_devices():
    for path in sorted(CSRC.glob("*.cu")):
        text = path.read_text()
        assert not re.search(r"if \((g_\w+_)?count < \d+\)", text), path.name
    users = {p.name for p in CSRC.glob("*.cu") if "DeviceCache<" in p.read_text()}
    assert users == {"gemm_dispatch.cu", "gemm_skinny.cu", "activation.cu"}
