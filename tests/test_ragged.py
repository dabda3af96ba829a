"""Index arithmetic of the calls over several sequences (csrc/q8_ragged.h) and
the page-state oracle, on the CPU.  The driver, built with g++ under the
sanitizers, checks over random ragged calls that every row, touched page and
unit of work belongs to exactly one block, that split records are written where
the merge reads them, and that arrays of nonsense keep every index in range."""

import os
import shutil
import subprocess

import numpy as np

from oracle import batch_oracle as bo

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_index_arithmetic(tmp_path):
    gxx = shutil.which("g++")
    assert gxx, "g++ is needed"
    out = str(tmp_path / "ragged")
    r = subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined",
                        "-fno-sanitize-recover=all", os.path.join(ROOT, "tests", "ragged_driver.cpp"),
                        "-o", out], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([out], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout == "ok\n", (r.stdout, r.stderr[-3000:])


def test_oracle_block_codes():
    """The oracle's scale and codes at their borders: ties to even, a grown
    scale, zeros, denormal scales, non-finite values."""
    c = bo.Cache(1, 16, 1, 64)
    codes = np.zeros((16, 64), np.int8)
    x = np.zeros((2, 64), np.float32)
    x[0, :5] = [127.0, 0.5, 1.5, -2.5, 63.49]
    assert c._block(codes, x, np.array([0, 1]), 0, np.nan) == 1.0
    assert codes[0, :5].tolist() == [127, 0, 2, -2, 63] and not codes[1].any()
    # twice the scale: old codes halved, ties to even
    assert c._block(codes, np.full((1, 64), 254, np.float32), np.array([2]), 2, 1.0) == 2.0
    assert codes[0, :5].tolist() == [64, 0, 1, -1, 32] and (codes[2] == 127).all()
    assert c._block(codes, np.zeros((1, 64), np.float32), np.array([0]), 0, 5.0) == 0.0
    assert np.isnan(c._block(codes, np.full((1, 64), np.inf, np.float32), np.array([3]), 3, 2.0))
    assert codes[0, 0] == 0 and not codes[3].any()


def test_oracle_pages():
    p = bo.Pages(3, 4, 8, 16)
    assert p.reserve([20, 0, 1]) == [] and p.rows == [[0, 1], [], [2]]
    p.set_len([20, -1, 1])
    p.fork([0, 0, -1])
    assert p.refs()[:3] == [2, 2, 1]
    # both sharers of the partly filled page grow: both get copies, page 1 is free again
    assert p.reserve([21, 21, 1]) == [(1, 3), (1, 4)] and p.refs()[1] == 0
    p.set_len([0, 21, 1])
    assert p.refs() == [1, 0, 1, 0, 1, 0, 0, 0]
    assert p.compact() == (3, [(4, 1)]) and p.rows[1] == [0, 1]
    # too few pages: the slots from the first that does not fit on get nothing
    assert p.reserve([64, 64, 64]) == [] and [len(r) for r in p.rows] == [4, 2, 1]
    # pages reserved ahead that a fork shares: replaced when their slots write to them
    p = bo.Pages(2, 6, 12, 16)
    p.reserve([60, 0])
    p.set_len([0, -1])
    p.reserve([60, 0])
    p.len[0] = 20
    p.fork([-1, 0])
    assert p.rows == [[0, 1, 2, 3]] * 2
    assert p.reserve([33, 20]) == [(1, 4)] and p.rows == [[0, 4, 5, 3], [0, 1, 2, 3]]
    assert p.reserve([33, 70]) == [] and p.rows[1] == [0, 1, 2, 6, 7]
