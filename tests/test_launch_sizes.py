"""The launches of the largest calls that the operators on a paged cache take stay
within the runtime's limits (c/host_hip_sizes.cpp): no GPU."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from conftest import ROOT
from host_runtime import START


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    lib = os.path.join(tmp_path_factory.mktemp("sizes"), "libhost_hip_sizes.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I/opt/rocm/include", "-w",
                    os.path.join(ROOT, "tests", "c", "host_hip_sizes.cpp"), "-o", lib], check=True)

    def go(body):
        r = subprocess.run([sys.executable, "-c", START.format(stub=lib) + body], cwd=ROOT, capture_output=True, text=True,
                           timeout=300)
        assert r.returncode == 0, r.stdout + r.stderr

    return go


@pytest.mark.parametrize("batch, beams, vocab", [(2 ** 23, 1, 1), (2 ** 22, 2, 1), (2 ** 22 + 5, 1, 900), (8192, 1024, 2), (1, 1, 2 ** 30),
                                                 (1, 1024, 2 ** 20), (4, 1, 2 ** 29)])
def test_the_largest_selections(run, batch, beams, vocab):
    run(f"""
net = ra.Network(0)
B, R, V = {batch}, {beams}, {vocab}
net.beam_select_device(device(8 * B * R * V), device(8 * B * R), B, R, V, 1, device(4 * B), device(4 * B), device(8 * B))
assert launches("k_beam_pick") >= 1 and launches("k_beam_pieces") == 1
""")
