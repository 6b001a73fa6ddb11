"""Refusals of a cache in 4 bits: bad arguments come back as errors before any CUDA call."""
import ctypes

import pytest

from ijb200 import lib


def view(**kw):
    base = dict(type=4, kv_heads=2, head_dim=64, page_size=16, num_pages=4, data_dev=4096, scale_dev=8192,
                page_table_dev=256, n_seqs=1, max_pages=4)
    base.update(kw)
    return lib.KvView(**base)


BAD_VIEWS = [dict(type=3), dict(type=5), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=32), dict(page_size=4), dict(num_pages=0),
             dict(n_seqs=0), dict(max_pages=0), dict(data_dev=None), dict(data_dev=4104), dict(scale_dev=None),
             dict(page_table_dev=None)]


@pytest.mark.parametrize("bad", BAD_VIEWS)
@pytest.mark.parametrize("fn", ["ijb_kv_append", "ijb_kv_gather"])
def test_views_are_checked(fn, bad):
    L = lib.load()
    v = view(**bad)
    assert getattr(L, fn)(ctypes.byref(v), 0, 4096, 4096, 128, 1, 256, 256, None, None) == lib.ERR_INVALID
    assert fn in L.ijb_last_error(None).decode()


@pytest.mark.parametrize("bad", BAD_VIEWS + [dict(scale_dev=8196), dict(scale_dev=8200)])
def test_attention_views_are_checked(bad):
    L = lib.load()
    v = view(**bad)
    assert L.ijb_paged_attention(ctypes.byref(v), 4, 0, 4096, 256, 8192, 256, 2, 1, 256, None, 256, 1, 0.125, 4096,
                                 1 << 40, None, None) == lib.ERR_INVALID
    assert "ijb_paged_attention" in L.ijb_last_error(None).decode()


@pytest.mark.parametrize("bad", BAD_VIEWS)
def test_copied_pages_views_are_checked(bad):
    L = lib.load()
    v, w = view(**bad), view()
    for a, b in ((v, None), (w, v), (v, w)):
        rc = L.ijb_kv_copy_pages(ctypes.byref(a), None if b is None else ctypes.byref(b), 1, 256, 256, None, None)
        assert rc == lib.ERR_INVALID and "ijb_kv_copy_pages" in L.ijb_last_error(None).decode()


@pytest.mark.parametrize("other", [dict(type=2), dict(kv_heads=1), dict(head_dim=128), dict(page_size=32)])
def test_copies_between_pages_that_differ_are_refused(other):
    L = lib.load()
    v, w = view(), view(**other)
    assert L.ijb_kv_copy_pages(ctypes.byref(v), ctypes.byref(w), 1, 256, 256, None, None) == lib.ERR_INVALID


def test_copied_pages_arguments_are_checked():
    L = lib.load()
    v = view()
    for n, src, dst in ((-1, 256, 256), (1, None, 256), (1, 256, None)):
        assert L.ijb_kv_copy_pages(ctypes.byref(v), None, n, src, dst, None, None) == lib.ERR_INVALID
    assert L.ijb_kv_copy_pages(None, None, 1, 256, 256, None, None) == lib.ERR_INVALID
    before = L.ijb_kernel_launches()
    assert L.ijb_kv_copy_pages(ctypes.byref(v), None, 0, None, None, None, None) == lib.OK
    assert L.ijb_kernel_launches() == before
    wide = view(kv_heads=1024, page_size=256, head_dim=128)
    assert L.ijb_kv_copy_pages(ctypes.byref(wide), None, 0x7fffffff, 256, 256, None, None) == lib.ERR_INVALID


def test_a_torch_without_4_bit_tensors_keeps_the_other_caches():
    """Only the cache in 4 bits needs torch.float4_e2m1fn_x2."""
    import os
    import subprocess
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inferencer-jetson_b200")
    code = ("import sys, torch; sys.path.insert(0, sys.argv[1]); del torch.float4_e2m1fn_x2\n"
            "from ijb200 import ops\n"
            "assert torch.float16 in ops._KV and torch.float8_e4m3fn in ops._KV and len(ops._KV) == 2")
    r = subprocess.run([sys.executable, "-c", code, pkg], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
