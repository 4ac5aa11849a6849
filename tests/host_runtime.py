"""The library's host code on a HIP runtime of host memory that launches nothing
(c/host_hip.cpp): states, refusals and failing calls, without a GPU.  The
numbers that come out have no meaning."""
from __future__ import annotations

import functools
import os
import subprocess
import sys
import tempfile

from conftest import ROOT

START = """
import ctypes, numpy as np, pytest
hip = ctypes.CDLL({stub!r}, mode=ctypes.RTLD_GLOBAL)  # before the library looks its names up
hip.host_hip_calls.restype = hip.host_hip_launches.restype = ctypes.c_long
calls, launches = (lambda f: lambda name: f(name.encode()))(hip.host_hip_calls), lambda part: hip.host_hip_launches(part.encode())
fail = lambda name, k=1: hip.host_hip_fail(name.encode(), ctypes.c_long(k))
hip.host_hip_pinned.restype = ctypes.c_void_p
pinned = lambda words: (ctypes.c_uint32 * words).from_address(hip.host_hip_pinned(ctypes.c_size_t(4 * words)))
import rustcrates_amd as ra

def device(nbytes):  # memory that the library takes for the device's
    p = ctypes.c_void_p()
    assert hip.hipMalloc(ctypes.byref(p), ctypes.c_size_t(nbytes)) == 0
    return p.value

def refused(code, match, f):
    with pytest.raises(ra.MitokError, match=match) as e:
        f()
    assert e.value.code == code, e.value

def stack(max_ctx=40, rope=False, d=16, layers=1, vocab=50):
    net = ra.Network(0)
    net.add_embedding(vocab, d)
    if rope:
        net.add_positional_encoding(d, 1250.0)
    for _ in range(layers):
        net.add_norm(d, 1e-5)
        net.add_self_attention(2, d, max_ctx, 1e-12)
        net.add_feed_forward(d, 24)
    net.add_linear(d, vocab)
    net.add_softmax(1)
    net.init_seeded(1)
    return net
"""


@functools.lru_cache
def stub() -> str:
    lib = os.path.join(tempfile.mkdtemp(), "libhost_hip.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I/opt/rocm/include", "-w",
                    os.path.join(ROOT, "tests", "c", "host_hip.cpp"), "-o", lib], check=True)
    return lib


def run(body: str):
    """Runs `body` in a process of its own, after START."""
    r = subprocess.run([sys.executable, "-c", START.format(stub=stub()) + body], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
