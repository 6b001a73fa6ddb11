"""ijb_kv_copy_pages on a B200: every byte of the pages named, and no other."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
CACHES = pytest.mark.parametrize("cache", ["f16", "e4m3", "e2m1"])


def make(cuda, cache, pages, kvh, page, hd, seed, status=None):
    import torch
    from ijb200 import ops
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    byte = lambda *s: torch.randint(0, 256, s, generator=g, device=cuda, dtype=torch.uint8)  # noqa: E731
    if cache == "f16":
        data, scale = byte(pages, 2, kvh, page, 2 * hd).view(torch.float16), None
    elif cache == "e4m3":
        data, scale = byte(pages, 2, kvh, page, hd).view(torch.float8_e4m3fn), byte(pages, 2, kvh, page)
    else:
        data, scale = byte(pages, 2, kvh, page, hd // 2).view(torch.float4_e2m1fn_x2), byte(pages, 2, kvh, page, hd // 32)
    return ops.PagedKV(data, torch.zeros((1, 1), dtype=torch.int32, device=cuda), scale, status)


def raw(kv):
    import torch
    return [t.view(torch.uint8).clone() for t in (kv.data, kv.scale) if t is not None]


@CACHES
@pytest.mark.parametrize("kvh,page,hd,n", [(1, 8, 64, 1), (1, 8, 64, 37), (3, 16, 128, 20), (8, 16, 64, 300), (8, 256, 128, 9),
                                           (5, 32, 64, 64)])
def test_pages_within_a_pool(cuda, cache, kvh, page, hd, n):
    import torch
    kv = make(cuda, cache, 2 * n + 3, kvh, page, hd, n)
    ids = np.random.default_rng(n).permutation(2 * n + 3)
    src, dst = ids[:n].copy(), ids[n:2 * n]
    src[n // 2:] = src[0]  # one page for many
    want = raw(kv)
    for w in want:
        w[dst] = w[src]
    i32 = lambda a: torch.from_numpy(a.astype(np.int32)).to(cuda)  # noqa: E731
    kv.copy_pages(i32(src), i32(dst))
    for w, g in zip(want, raw(kv)):
        assert torch.equal(w, g)


@CACHES
def test_pages_of_another_pool(cuda, cache):
    import torch
    a, b = make(cuda, cache, 9, 2, 16, 64, 1), make(cuda, cache, 30, 2, 16, 64, 2)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    want, before = raw(b), raw(a)
    for w, s in zip(want, before):
        w[[29, 0, 8]] = s[[0, 8, 0]]
    a.copy_pages(i32([0, 8, 0]), i32([29, 0, 8]), to=b)
    for w, g in zip(want + before, raw(b) + raw(a)):
        assert torch.equal(w, g)


@CACHES
def test_padding_and_pages_that_there_are_not(cuda, cache):
    import torch
    status = torch.zeros((1,), dtype=torch.int32, device=cuda)
    kv, other = make(cuda, cache, 6, 1, 8, 64, 3, status), make(cuda, cache, 4, 1, 8, 64, 4)
    before = raw(kv) + raw(other)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    for src, dst, to, bad in (([0], [-1], None, 0), ([-5], [-1], None, 0), ([-1], [1], None, 1), ([6], [1], None, 1),
                              ([1], [6], None, 1), ([1], [4], other, 1), ([1 << 30], [2], None, 1)):
        status.zero_()
        kv.copy_pages(i32(src), i32(dst), to)
        assert bool(int(status)) == bool(bad), (src, dst)
    kv.copy_pages(i32([]), i32([]))
    for w, g in zip(before, raw(kv) + raw(other)):
        assert torch.equal(w, g)


def test_scales_that_start_anywhere(cuda):
    """An e4m3 or e2m1 cache's scale bytes need no alignment for a copy."""
    import torch
    from ijb200 import ops
    for cache in ("e4m3", "e2m1"):
        kv = make(cuda, cache, 7, 3, 8, 64, 5)
        room = torch.zeros((kv.scale.numel() + 1,), dtype=torch.uint8, device=cuda)
        room[1:] = kv.scale.view(-1)
        odd = ops.PagedKV(kv.data, kv.page_table, room[1:].view(kv.scale.shape))
        want = raw(odd)
        for w in want:
            w[[5, 6]] = w[[0, 3]]
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
        odd.copy_pages(i32([0, 3]), i32([5, 6]))
        for w, g in zip(want, raw(odd)):
            assert torch.equal(w, g)
        assert int(room[0]) == 0


def test_a_captured_copy_reads_its_pages_when_it_runs(cuda):
    import torch
    kv = make(cuda, "e2m1", 50, 2, 16, 128, 6)
    src, dst = (torch.tensor(a, dtype=torch.int32, device=cuda) for a in ([0, 1], [2, 3]))
    kv.copy_pages(src, dst)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.copy_pages(src, dst)
    for a, b in (([4, 5], [6, 7]), ([8, 8], [9, 49])):
        src.copy_(torch.tensor(a, dtype=torch.int32))
        dst.copy_(torch.tensor(b, dtype=torch.int32))
        want = raw(kv)
        for w in want:
            w[b] = w[a]
        graph.replay()
        torch.cuda.synchronize()
        for w, g in zip(want, raw(kv)):
            assert torch.equal(w, g)


def test_refusals(cuda):
    import torch
    kv, other = make(cuda, "e2m1", 5, 2, 16, 64, 7), make(cuda, "e2m1", 5, 2, 8, 64, 7)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    from ijb200.lib import IjbError
    with pytest.raises(IjbError):
        kv.copy_pages(i32([0]), i32([1]), to=other)
    for src, dst in ((i32([0, 1]), i32([2])), (i32([0]).long(), i32([1])), (i32([0]).cpu(), i32([1])),
                     (i32([0, 1, 2, 3])[::2], i32([1, 4]))):
        with pytest.raises(ValueError):
            kv.copy_pages(src, dst)
