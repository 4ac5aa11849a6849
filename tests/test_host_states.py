"""What the serving calls do on caches that are gone, and where a runtime call
fails half way (host_runtime.py): no GPU."""
from __future__ import annotations

import pytest

from host_runtime import run

TREE = """
net = stack()
prompt = np.arange(2, 12, dtype=np.uint32).reshape(2, 5)
net.prefill(prompt)
net.tree_step([[3, 4, 5]] * 2, [[-1, 0, 0]] * 2, weigh_nodes=1)
"""


def test_the_host_runtime_stands_in_for_the_gpu():
    run(TREE + """
net.tree_accept([[0, 2]] * 2)  # a gap: rows move
assert launches("k_cache_pack") == 1 and launches("k_tree_split") == 1 and calls("hipMalloc") > 10
assert net.evict_rows(2, 4, 1, 1).tolist() == [4, 4]
""")


@pytest.mark.parametrize("drop", ["net.add_self_attention(2, 16, 40, 1e-12)", "net.init_seeded(2)"])
def test_dropped_caches_take_the_pending_tree_with_them(drop):
    run(TREE + drop + """
moved = launches("k_cache_pack")
refused(3, "without a tree_step", lambda: net.tree_accept([[0, 2]] * 2))
assert launches("k_cache_pack") == moved
refused(3, "no KV cache", lambda: net.evict_rows(2, 4))
refused(3, "no KV cache", lambda: net.decode_step())
""")


def test_an_error_of_the_threads_earlier_calls_is_not_a_calls_own():
    """The runtime keeps the last error of a thread, of whatever made the call, until it is read."""
    run(TREE + """
def stale(f):
    assert hip.hipSetDevice(5) != 0
    return f()
stale(lambda: net.tree_step([[3, 4, 5]] * 2, [[-1, 0, 0]] * 2, weigh_nodes=1))
stale(lambda: net.tree_accept([[0, 2]] * 2))
stale(lambda: net.decode_step())
stale(lambda: net.evict_rows(2, 4, 1, 1))
stale(lambda: net.process_logits(np.zeros((2, 50))))
stale(lambda: net.predict(prompt, forward_only=False))
stale(lambda: net.prefill(prompt))
a = [device(65536) for _ in range(4)]
stale(lambda: net.tree_attention_device(*a[:3], [3], [[-1]], 1, 4, 8, a[3]))
""")


MEND = """
def state():
    try:
        net.decode_step([3, 4])
    except ra.MitokError as e:
        assert e.code == 3, e  # dropped
        return "dropped"
    return "there"
"""


@pytest.mark.parametrize("name", ["hipMemcpyAsync", "launch", "hipMalloc", "hipStreamSynchronize"])
@pytest.mark.parametrize("call, moved", [
    ("net.tree_accept([[0, 2], [0, 1]])", "k_cache_pack"),
    ("net.evict_rows(2, 4, 1, 1)", "k_cache_pack"),
    ("net.tree_step([[5, 6]] * 2, [[-1, 0]] * 2, weigh_nodes=2)", "k_tree_split"),
])
def test_a_runtime_call_that_fails_half_way(name, call, moved):
    """Caches that a call may have touched are dropped where it fails, never half
    moved and still in use; where it finds no room before, they go on as they were."""
    run(MEND + f"""
for k in range(1, 60):
""" + "".join("    " + line + "\n" for line in TREE.strip().splitlines()) + f"""
    if "evict" in {call!r}:
        net.tree_accept([[0], [0]])
        net._lib.mitok_set_graph_mode(net._h, 0)
    before, lens = launches({moved!r}), calls({name!r})
    fail({name!r}, k)
    try:
        {call}
    except ra.MitokError as e:
        fail({name!r}, 0)
        assert e.code in (2, 5), e
        if launches({moved!r}) > before or "tree_step" in {call!r}:
            assert state() == "dropped", k
        elif {name!r} == "hipMalloc":
            {call}  # the same call again
            assert state() == "there"
        net.close()
        continue
    fail({name!r}, 0)
    assert calls({name!r}) - lens < k
    break
else:
    raise AssertionError("the call never ended well")
assert k > 1 or {name!r} == "hipMalloc"
""")


def test_a_path_array_wider_than_any_path():
    """Only the columns in use are staged: offsets into the table keep their 32 bits whatever max_path is."""
    run(TREE + """
path = np.zeros((2, 100000), np.uint32)
path[:, 1] = 2
host = calls("hipHostMalloc")
net.tree_accept(path, [2, 1])
assert calls("hipHostMalloc") == host and launches("k_cache_pack") == 1
""")


@pytest.mark.parametrize("step", ["net.decode_step([3])", "net.tree_step([[3]], [[-1]]); net.tree_accept([[0]])"])
def test_positions_past_the_rope_table(step):
    """A session that evicts and goes on: the table of angles grows a few times,
    not with every token, and the captured step with it."""
    run(f"""
net = stack(rope=True)
net.prefill(np.arange(2, 32, dtype=np.uint32)[None])
def evict():
    net.tree_step([[3]], [[-1]], weigh_nodes=1)
    net.tree_accept([[0]])
    net.evict_rows(1, 20, 2, 4)
pos, before, grown = 30, None, 0
while pos < 1300:
    evict()
    pos += 1
    for _ in range(15):
        if pos > 600:  # past the first growth
            now = calls("hipMalloc"), calls("hipGraphInstantiate")
            grown += before is not None and now != before
            before = now
        {step}
        pos += 1
assert 1 <= grown <= 2, grown
""")


@pytest.mark.parametrize("call", ["net.process_logits(np.zeros((2, 50)))", "net.tree_step([[3, 4, 5]] * 2, [[-1, 0, 0]] * 2)"])
def test_error_words_of_a_call_that_failed_otherwise(call):
    """What the kernels of a failing call found is not the next call's."""
    run(TREE + f"""
words = pinned(4)
for word in range(3):
    words[word] = 1  # as a kernel sets it
    fail("hipStreamSynchronize", 1)
    refused(2, "", lambda: {call})
    assert not any(words)
    net.prefill(prompt)
    {call}
    words[word] = 1
    refused(4 if word == 1 else 1, "", lambda: {call})
    net.prefill(prompt)
""")
