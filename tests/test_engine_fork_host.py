"""Forked sequences' pages, on the host, with a CUDA runtime of host memory (see test_engine_host.py): who holds which
pages, what is copied, and that nothing is lost when there is none left."""
import pytest

from test_engine_host import child  # noqa: F401  (a fixture)

KW = "context=64, max_batch=4, max_seqs=5, page_size=8"
TYPES = pytest.mark.parametrize("kv_type", [None, "f16", "e4m3", "e2m1"])


@TYPES
def test_a_fork_copies_the_page_it_ends_in(child, kv_type):  # noqa: F811
    child(f"""
e = Engine(cfg, weights, {KW}, kv_type={kv_type!r})
s = e.seq_open()
e.seq_prefill(s, list(range(20)))
ids = ("cudaMemcpyAsync", 2 * cfg.layers * 4)  # source and destination of one page in every layer
for length, copied in ((20, 1), (16, 0), (8, 0), (1, 1), (0, 0), (17, 1)):
    start, before = F.fake_calls(), e.lib.ijb_kernel_launches()
    t = e.seq_fork(s, length)
    assert t not in (0, s) and e.seq_length(t) == length and e.seq_length(s) == 20
    assert e.lib.ijb_kernel_launches() - before == copied
    calls = log(start)
    assert calls.count(ids) == copied and calls[-1][0] in ("cudaStreamSynchronize", "cudaMemcpy"), calls
    e.seq_close(t)
assert e.seq_length(e.seq_fork(s)) == 20
""")


@TYPES
def test_shared_pages_return_with_their_last_sequence(child, kv_type):  # noqa: F811
    child(f"""
e = Engine(cfg, weights, {KW}, kv_type={kv_type!r}, num_pages=8)
s = e.seq_open()
e.seq_prefill(s, list(range(32)))             # 4 of the 8 pages
forks = [e.seq_fork(s, 32) for _ in range(3)]  # none more
e.decode_step(forks, [1, 2, 3])               # one each: 7
e.seq_close(s)                                # its pages are still held
a = e.seq_open()
e.seq_prefill(a, list(range(8)))
try:
    e.decode_step([a], [1])
    raise SystemExit("there should be no page left")
except lib.IjbError as err:
    assert err.code == lib.ERR_CAPACITY
for t in forks:
    e.seq_close(t)
e.decode_step([a], [1])
b = e.seq_open()
e.seq_prefill(b, list(range(48)))             # all others
""")


def test_no_sequence_or_page_left_changes_nothing(child):  # noqa: F811
    child(f"""
e = Engine(cfg, weights, {KW}, num_pages=4)
s = e.seq_open()
e.seq_prefill(s, list(range(28)))             # all 4 pages
def refused(length, code):
    try:
        e.seq_fork(s, length)
        raise SystemExit("no error")
    except lib.IjbError as err:
        assert err.code == code, err
refused(28, lib.ERR_CAPACITY)                 # no page for the copy
refused(29, lib.ERR_INVALID)
refused(-1, lib.ERR_INVALID)
assert lib.load().ijb_seq_fork(e.h, 9, 0, ctypes.byref(ctypes.c_int())) == lib.ERR_INVALID
assert lib.load().ijb_seq_fork(e.h, 3, 0, ctypes.byref(ctypes.c_int())) == lib.ERR_INVALID  # not open
assert lib.load().ijb_seq_fork(e.h, s, 0, None) == lib.ERR_INVALID
assert lib.load().ijb_seq_fork(None, s, 0, ctypes.byref(ctypes.c_int())) == lib.ERR_INVALID
forks = [e.seq_fork(s, 24) for _ in range(3)]  # whole pages need none
refused(24, lib.ERR_CAPACITY)                 # the table is full
e.seq_close(s)                                # the page it ended in alone comes back
e.decode_step([forks[0]], [1])
try:
    e.decode_step([forks[1]], [1])
    raise SystemExit("no error")
except lib.IjbError as err:
    assert err.code == lib.ERR_CAPACITY
""")


@TYPES
def test_sequence_0_set_back_leaves_its_forks_alone(child, kv_type):  # noqa: F811
    """Writing to a shared page again takes a page of its own, with what stays of it."""
    child(f"""
e = Engine(cfg, weights, {KW}, kv_type={kv_type!r}, num_pages=8)
ids = ("cudaMemcpyAsync", 2 * cfg.layers * 4)
e.prefill(list(range(24)))                    # 3 pages
t = e.seq_fork(0, 24)
start = F.fake_calls()
e.forward(1, 11)                              # in the middle of the second page: copied
assert log(start).count(ids) == 1
start = F.fake_calls()
e.forward(1, 12)                              # its own by now
assert log(start).count(ids) == 0
e.reset()
start = F.fake_calls()
e.prefill(list(range(24)))                    # the first and the third from their start: replaced, not copied
assert log(start).count(ids) == 0
s = e.seq_open()
e.seq_prefill(s, list(range(16)))             # 3 + 3 + 2: all
try:
    e.decode_step([s], [1])
    raise SystemExit("no error")
except lib.IjbError as err:
    assert err.code == lib.ERR_CAPACITY
e.seq_close(t)
e.decode_step([s], [1])
""")


@pytest.mark.parametrize("fail", ["cudaMemcpyAsync", "cudaStreamSynchronize", "cudaMemcpy"])
def test_a_fork_that_fails_gives_its_pages_back(child, fail):  # noqa: F811
    child(f"""
e = Engine(cfg, weights, {KW}, num_pages=4)
s = e.seq_open()
e.seq_prefill(s, list(range(12)))             # 2 pages
e.seq_close(e.seq_fork(s, 12))                # (its buffers are there)
F.fake_fail(b"{fail}", b"cudaSetDevice")
try:
    e.seq_fork(s, 12)
    raise SystemExit("no error")
except lib.IjbError as err:
    assert "made by the test" in str(err), err
a, b = e.seq_fork(s, 12), e.seq_fork(s, 12)   # both pages that are left, both sequences' names
e.decode_step([a, b, s], [1, 2, 3])
""")

