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


@pytest.mark.parametrize("batch, rows, heads, dh, page_rows, max_pages, kv", [
    (256, 65536, 1, 1, 1024, 2 ** 20, 2 ** 30 - 65536),  # 2^44 steps of work: more than 32 bits for each block
    (4, 65536, 12, 64, 16, 2 ** 14, 2 ** 18 - 65536), (65535, 1, 4, 1, 16, 1, 3), (65535, 2, 4, 1, 16, 1, 3), (8, 1, 32768, 1, 16, 4, 60),
    (1, 65536, 4, 256, 1024, 64, 0)])
def test_the_largest_chunks(run, batch, rows, heads, dh, page_rows, max_pages, kv):
    run(f"""
net = ra.Network(0)
B, n, H, dh, ps, P = {batch}, {rows}, {heads}, {dh}, {page_rows}, {max_pages}
q, k, v, o = (device(16 * B * n * H * dh) for _ in range(4))
net.paged_attention_device(q, k, v, device(16 * H * ps * dh), device(16 * H * ps * dh), device(4 * B * P), [{kv}] * B, n, H, dh, ps, 1, P, o)
assert launches("k_paged_tile") + launches("k_paged_split") + launches("k_paged_beams") == 1
""")


@pytest.mark.parametrize("old, new, pages, max_pages, layers", [(65535, 65535, 2 ** 24, 4, 1), (1, 65535, 8, 4096, 16384), (65535, 1, 8, 1, 1)])
def test_the_largest_forks(run, old, new, pages, max_pages, layers):
    run(f"""
net = ra.Network(0)
old, new, pages, P, layers = {old}, {new}, {pages}, {max_pages}, {layers}
k, v = (device(16 * 16 * layers * pages) for _ in range(2))
net.fork_pages_device(k, v, layers, pages, 1, 16, 1, device(4 * old * P), device(4 * old), old, P, device(4 * new), new, device(4 * new * P),
                      device(4 * new))
assert launches("k_fork_commit") == 1
""")
