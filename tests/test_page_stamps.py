"""What a paged attention remembers of its pages where a runtime call fails
(host_runtime.py): no GPU."""
from __future__ import annotations

from host_runtime import run


def test_stamps_that_were_not_cleared_are_cleared_by_the_next_call():
    """A page's last call and sequence start at zero: filled once when made, and again after a call that failed."""
    run("""
net = ra.Network(0)
a = [device(1 << 22) for _ in range(7)]
def paged(pages=4):
    net.paged_attention_device(*a[:6], [20], 2, 2, 8, 16, pages, 4, a[6])
fills = launches("k_fill")
fail("launch", 1)
refused(2, "launch", paged)
paged()
assert launches("k_fill") == fills + 1
paged()
assert launches("k_fill") == fills + 1
paged(64)  # a larger pool
assert launches("k_fill") == fills + 2
fail("hipMalloc", 1)
refused(5, "hipMalloc", lambda: paged(1024))
paged(64)
assert launches("k_fill") == fills + 3
""")
