"""Refusals of the stand-alone operators: bad arguments come back as errors before any CUDA call."""
import ctypes

import pytest

from ijb200 import lib


def view(**kw):
    base = dict(type=2, kv_heads=2, head_dim=64, page_size=16, num_pages=4, data_dev=4096, scale_dev=8192,
                page_table_dev=256, n_seqs=1, max_pages=4)
    base.update(kw)
    return lib.KvView(**base)


BAD_VIEWS = [dict(type=1), dict(kv_heads=0), dict(head_dim=96), dict(page_size=12), dict(page_size=4),
             dict(page_size=512), dict(num_pages=0), dict(n_seqs=0), dict(max_pages=0), dict(max_pages=1 << 30),
             dict(data_dev=None), dict(data_dev=4104), dict(scale_dev=None), dict(page_table_dev=None)]


@pytest.mark.parametrize("bad", BAD_VIEWS)
@pytest.mark.parametrize("fn", ["ijb_kv_append", "ijb_kv_gather"])
def test_cache_views_are_checked(fn, bad):
    L = lib.load()
    v = view(**bad)
    rc = getattr(L, fn)(ctypes.byref(v), 0, 4096, 4096, 128, 1, 256, 256, None, None)
    assert rc == lib.ERR_INVALID and fn in L.ijb_last_error(None).decode()


@pytest.mark.parametrize("fn", ["ijb_kv_append", "ijb_kv_gather"])
@pytest.mark.parametrize("args", [(30, 4096, 4096, 128, 1, 256, 256), (0, None, 4096, 128, 1, 256, 256),
                                  (0, 4096, None, 128, 1, 256, 256), (0, 4096, 4096, 127, 1, 256, 256),
                                  (0, 4096, 4096, 128, -1, 256, 256), (0, 4096, 4096, 128, 1, None, 256),
                                  (0, 4096, 4096, 128, 1, 256, None), (0, 4098, 4096, 128, 1, 256, 256),
                                  (1, 4096, 4097, 128, 1, 256, 256)])
def test_row_arguments_are_checked(fn, args):
    L = lib.load()
    v = view()
    assert getattr(L, fn)(ctypes.byref(v), *args, None, None) == lib.ERR_INVALID
    assert getattr(L, fn)(None, *args, None, None) == lib.ERR_INVALID


def test_no_rows_is_no_launch():
    L = lib.load()
    v = view()
    before = L.ijb_kernel_launches()
    assert L.ijb_kv_append(ctypes.byref(v), 0, None, None, 128, 0, None, None, None, None) == lib.OK
    assert L.ijb_sample(None, 10, 0, 10, None, None, None, None, None, None, None, None) == lib.OK
    assert L.ijb_kernel_launches() == before


@pytest.mark.parametrize("args", [(None, 10, 1, 10, 256, 256), (256, 9, 1, 10, 256, 256), (256, 10, -1, 10, 256, 256),
                                  (256, 131073, 1, 131073, 256, 256), (256, 10, 1, 0, 256, 256),
                                  (256, 10, 1, 10, None, 256), (256, 10, 1, 10, 256, None)])
def test_sample_arguments_are_checked(args):
    L = lib.load()
    x, stride, n, vocab, u, token = args
    assert L.ijb_sample(x, stride, n, vocab, u, None, None, None, None, token, None, None) == lib.ERR_INVALID
    assert "ijb_sample" in L.ijb_last_error(None).decode()


def attention(v, heads=4, type_=0, q=4096, qs=256, out=8192, os=256, n=2, e=1, start=256, kv_len=256, work=4096,
              size=1 << 40):
    return lib.load().ijb_paged_attention(ctypes.byref(v), heads, type_, q, qs, out, os, n, e, start, None, kv_len, 1,
                                          0.125, work, size, None, None)


@pytest.mark.parametrize("bad", BAD_VIEWS + [dict(scale_dev=8194)])
def test_attention_views_are_checked(bad):
    assert attention(view(**bad)) == lib.ERR_INVALID
    assert "ijb_paged_attention" in lib.load().ijb_last_error(None).decode()


@pytest.mark.parametrize("bad", [dict(heads=3), dict(heads=0), dict(heads=34), dict(type_=12), dict(q=None),
                                 dict(out=None), dict(start=None), dict(kv_len=None), dict(work=None), dict(qs=255),
                                 dict(os=255), dict(n=-1), dict(e=0), dict(e=4097), dict(q=4097), dict(type_=1, out=4097),
                                 dict(work=4100), dict(n=1 << 30), dict(out=4096)])
def test_attention_arguments_are_checked(bad):
    assert attention(view(), **bad) == lib.ERR_INVALID


def test_attention_refuses_more_units_of_work_than_it_counts():
    wide = view(page_size=256, max_pages=1 << 22)
    assert attention(wide) == lib.ERR_INVALID and attention(wide, e=4096) == lib.ERR_INVALID
    assert "too large" in lib.load().ijb_last_error(None).decode()


def test_attention_without_tokens_is_no_launch():
    L = lib.load()
    before = L.ijb_kernel_launches()
    assert attention(view(), n=0, q=None, out=None) == lib.OK
    assert L.ijb_kernel_launches() == before


def test_attention_workspace_of_a_bad_view_is_nothing():
    assert lib.load().ijb_paged_attention_workspace(ctypes.byref(view(head_dim=80))) == 0
    assert lib.load().ijb_paged_attention_workspace(None) == 0
