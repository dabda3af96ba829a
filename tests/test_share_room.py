"""Space of the attention over shared prefixes (csrc/q8_ragged.h) on the CPU under the
sanitizers: records fit beside a block of the sequences' own parts, for every number of KV
heads, and a call's groups keep to their blocks."""

import os
import shutil
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_room(tmp_path):
    gxx = shutil.which("g++")
    assert gxx, "g++ is needed"
    out = str(tmp_path / "room")
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
                        "-fno-sanitize-recover=all", os.path.join(ROOT, "tests", "share_room_driver.cpp"),
                        "-o", out], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([out], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.stdout, r.stderr[-3000:])
