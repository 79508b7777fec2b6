"""The single-token attention kernel's ring of page copies (bitnetrs_b200/csrc/kvq_ring.h) on the host: a warp whose wait
runs out waits for every copy that it still has in flight, a full ring's among them (tests/kvq_ring.cpp)."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_copy_in_flight_is_waited_for(tmp_path):
    exe = tmp_path / "kvq_ring"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", str(HERE / "kvq_ring.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and int(r.stdout.split()[1]) > 10000, r.stdout
