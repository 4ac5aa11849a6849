"""Which form one new token of many sequences takes (paged_plan), on a HIP runtime
of host memory (host_runtime.py): no GPU."""
from __future__ import annotations

import pytest

from host_runtime import run


@pytest.mark.parametrize("lens, heads, bunched", [
    ([200] * 4 * 64, 12, True),                                   # beams of one length
    ([x for k in range(32) for x in [200 + k] * 4], 8, True),     # of about one
    ([x for k in range(16) for x in [100 + 25 * k] * 16], 12, True),
    ([2000] * 16 + [x for k in range(42) for x in [100 + k] * 2], 12, False),  # 16 long ones would be one block's
    ([2000] * 4 + [x for k in range(42) for x in [100 + k] * 2], 12, False),
    ([1000] * 16 + [x for k in range(8) for x in [250 + 30 * k] * 16], 12, True),  # in smaller bunches
    ([200 + k for k in range(64)], 12, False),                    # no two of one length
])
def test_a_bunch_of_beams_holds_no_more_than_its_share(lens, heads, bunched):
    run(f"""
net = ra.Network(0)
lens, H = {lens}, {heads}
B, P = len(lens), 126
a = [device(1 << 22) for _ in range(6)]
net.paged_attention_device(*a[:5], device(4 * B * P), lens, 1, H, 8, 16, 100, P, a[5])
assert launches("k_paged_beams") == {int(bunched)} and launches("k_paged_split") == {int(not bunched)}
""")
