"""Which launches of attention run every other round of row tiles backwards, on the host.  No GPU needed."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    exe = tmp_path_factory.mktemp("order") / "attention_order_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", os.path.join(ROOT, "ratchet_amd", "csrc"), os.path.join(ROOT, "tests", "attention_order_check.cpp"), "-o", str(exe)], check=True)
    return exe


@pytest.mark.parametrize("tiles, per, held, rounds", [
    (256, 32, 2, 0), (257, 1, 2, 256), (512, 32, 2, 8), (512, 32, 3, 8),
    (544, 32, 2, 8), (552, 8, 2, 32), (640, 32, 2, 8), (736, 32, 2, 8), (768, 32, 2, 8), (769, 1, 2, 0),      # two blocks to a CU: a third round is turned as well
    (544, 32, 3, 8), (768, 32, 3, 8), (800, 32, 3, 0),
    (300, 1, 1, 0), (512, 32, 1, 0), (544, 32, 1, 0)])                                                        # one block to a CU: the longest first
def test_rounds(check, tiles, per, held, rounds):
    run = subprocess.run([str(check), str(tiles), str(per), "256", str(held)], capture_output=True, text=True, check=True)
    assert int(run.stdout) == rounds
