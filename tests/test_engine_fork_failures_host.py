"""Calls that fail over shared pages, on the host, with a CUDA runtime of host memory (see test_engine_host.py): a sequence
that writes to a page which a fork shares keeps what it held, whichever call fails, and the device's page table follows the
host's."""
import pytest

from test_engine_host import child  # noqa: F401  (a fixture)

KW = "context=64, max_batch=4, max_seqs=5, page_size=8"
TYPES = pytest.mark.parametrize("kv_type", [None, "f16", "e4m3", "e2m1"])
CODE = """
ids = ("cudaMemcpyAsync", 2 * cfg.layers * 4)  # source and destination of one page in every layer
def fails(name, call):
    '''call() with its first call of name failing'''
    F.fake_fail(name.encode(), b"cudaSetDevice")
    F.cudaSetDevice(0)
    try:
        call()
    except lib.IjbError as err:
        assert "made by the test" in str(err), err
        return
    raise SystemExit("no error")
def copies(call):
    start = F.fake_calls()
    call()
    return log(start).count(ids)
"""


@TYPES
@pytest.mark.parametrize("fail", ["cudaMalloc", "cudaHostAlloc", "cudaStreamSynchronize", "cudaMemcpyAsync", "cudaGraphLaunch"])
def test_a_failed_write_to_a_shared_page_is_made_good(child, kv_type, fail):  # noqa: F811
    """The positions before the one that is written are copied by the failed call, and its copy stays, or by the next one."""
    child(f"""{CODE}
e = Engine(cfg, weights, {KW}, kv_type={kv_type!r})
e.prefill(list(range(24)))
t = e.seq_fork(0, 24)                         # whole pages: nothing has been copied
start = F.fake_calls()
fails({fail!r}, lambda: e.forward(1, 11))
done = [n for n, (name, size) in enumerate(log(start)) if (name, size) == ids]
if {fail!r} == "cudaMemcpyAsync":             # (the ids' own upload, which is logged all the same)
    assert len(done) == 1
    done = []
assert e.seq_length(0) == 24
assert len(done) + copies(lambda: e.forward(1, 11)) == 1
assert copies(lambda: e.forward(1, 12)) == 0
""")


@TYPES
def test_a_fork_after_a_failed_step_copies_its_own_page_only(child, kv_type):  # noqa: F811
    """A copy that was left for later would be in one call with one that reads its destination."""
    child(f"""{CODE}
e = Engine(cfg, weights, {KW}, kv_type={kv_type!r}, num_pages=6)
e.prefill(list(range(24)))                    # 3 pages
e.seq_fork(0, 24)
s = e.seq_open()
e.seq_prefill(s, list(range(16)))             # 2: one is left
try:
    e.decode_step([0, s], [1, 2])             # each needs one: sequence 0 goes on behind its shared pages
    raise SystemExit("no error")
except lib.IjbError as err:
    assert err.code == lib.ERR_CAPACITY
e.seq_close(s)
fails("cudaStreamSynchronize", lambda: e.forward(1, 11))
before = e.lib.ijb_kernel_launches()
assert copies(lambda: e.seq_fork(0, 10)) == 1 and e.lib.ijb_kernel_launches() - before == 1
""")


@TYPES
def test_the_page_table_is_sent_again(child, kv_type):  # noqa: F811
    """An upload of a sequence's row that failed, or that the call did not come to, is made up for by the next call."""
    child(f"""{CODE}
e = Engine(cfg, weights, {KW}, kv_type={kv_type!r}, num_pages=4)
s = e.seq_open()
fails("cudaMemcpyAsync", lambda: e.decode_step([s], [1]))
start = F.fake_calls()
e.decode_step([s], [1])
assert ("cudaMemcpyAsync", 4) in log(start)
try:
    e.generate(s, 1, 40)                      # 6 pages, of which there are 4
    raise SystemExit("no error")
except lib.IjbError as err:
    assert err.code == lib.ERR_CAPACITY
start = F.fake_calls()
e.decode_step([s], [1])                       # its page was there, the 3 others have been taken since
assert ("cudaMemcpyAsync", 16) in log(start)
start = F.fake_calls()
e.decode_step([s], [1])
assert ("cudaMemcpyAsync", 16) not in log(start)
""")


@TYPES
def test_the_page_table_is_sent_again_for_a_shared_page(child, kv_type):  # noqa: F811
    child(f"""{CODE}
e = Engine(cfg, weights, {KW}, kv_type={kv_type!r})
e.prefill(list(range(24)))
e.seq_fork(0, 24)
e.reset()
fails("cudaMemcpyAsync", lambda: e.forward(1, 0))  # no copy: the row's upload
start = F.fake_calls()
assert copies(lambda: e.forward(1, 0)) == 0
assert ("cudaMemcpyAsync", 12) in log(start)
""")


@TYPES
@pytest.mark.parametrize("fail", ["cudaMalloc", "cudaMemcpyAsync", "cudaGraphLaunch"])
def test_a_failed_write_to_a_page_s_start_keeps_what_is_behind_it(child, kv_type, fail):  # noqa: F811
    """The sequence is set back by a step that succeeds only: until then it may go on at any of its positions."""
    child(f"""{CODE}
e = Engine(cfg, weights, {KW}, kv_type={kv_type!r})
e.prefill(list(range(24)))
e.seq_fork(0, 24)
start = F.fake_calls()
fails({fail!r}, lambda: e.forward(1, 16))
done = log(start).count(ids) if {fail!r} == "cudaGraphLaunch" else 0
assert e.seq_length(0) == 24
assert done + copies(lambda: e.forward(1, 20)) == 1
""")


@TYPES
def test_generate_copies_no_page_that_it_writes_anew(child, kv_type):  # noqa: F811
    child(f"""{CODE}
def launches(fork):
    e = Engine(cfg, weights, {KW}, kv_type={kv_type!r})
    e.prefill(list(range(40)))                # 5 pages
    if fork:
        e.seq_fork(0, 40)
    e.forward(1, 11)                          # the second is sequence 0's own
    before = e.lib.ijb_kernel_launches()
    e.generate(0, 1, 29)                      # positions 12 to 39
    return e.lib.ijb_kernel_launches() - before
assert launches(True) == launches(False)
""")
