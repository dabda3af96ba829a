"""Units of work of the cache attention (csrc/q8_ragged.h) on the CPU under the
sanitizers: runs and records of well-formed calls, and offsets that hold nonsense,
whose sums stay at 2^30 and whose row tiles, columns and rows lie inside their
sequences."""

import os
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_units_and_sums(tmp_path):
    gxx = shutil.which("g++")
    assert gxx, "g++ is needed"
    out = str(tmp_path / "sums")
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
                        "-fno-sanitize-recover=all", os.path.join(ROOT, "tests", "ragged_sums_driver.cpp"),
                        "-o", out], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([out], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.stdout, r.stderr[-3000:])
