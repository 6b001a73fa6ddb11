"""ijb_paged_attention on a B200 where a page table names pages that the pool does not have, against 64 bits; the
tolerances are those of test_gpu_paged_attention.py."""
import numpy as np
import pytest
from test_gpu_paged_attention import CACHES, TYPES, build
from test_gpu_paged_attention_range import attend64
from test_gpu_paged_attention_sums import i32

pytestmark = pytest.mark.gpu


@CACHES
@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kvh,group,entries", [
    (2, 4, [(1, 40), (1, 33), (1, 900)]), (8, 1, [(1, 5), (2, 70)]), (1, 16, [(1, 3000)]),
    (2, 4, [(1, 700 + 9 * i) for i in range(40)]), (2, 4, [(40, 40), (200, 1000)]), (1, 4, [(150, 6000)]),
    (2, 2, [(700, 900)] + [(1, 100)] * 9)])
def test_pages_that_name_nothing(cuda, hd, kvh, group, entries, cache, dtype):
    """The positions of a page id outside the pool are absent: no other page is read for them, and they are reported."""
    import torch
    dtype = getattr(torch, dtype)
    page = 16
    kv, dense = build(cuda, [t for _, t in entries], kvh, hd, page, cache, 9)
    rng = np.random.default_rng(len(entries))
    pages = kv.data.shape[0]
    gone = {}
    for e, (l, t) in enumerate(entries):
        if e % 3 == 1:
            continue  # as it is
        have = -(-t // page)
        at = {0, have - 1} if e % 2 == 0 else {int(rng.integers(0, have))}
        gone[e] = {a: b for a, b in zip(at, (-1, pages))}
        for a, b in gone[e].items():
            kv.page_table[e, a] = b
    start = np.cumsum([0] + [l for l, _ in entries]).tolist()
    g = torch.Generator(device=cuda)
    g.manual_seed(2)
    q = (torch.randn((start[-1], kvh * group, hd), generator=g, device=cuda) * 1.5).to(dtype)
    args = (q, i32(cuda, start), i32(cuda, [t for _, t in entries]))
    got = kv.attention(*args, max_q=max(l for l, _ in entries)).double()
    assert int(kv.status) != 0
    for e, (l, t) in enumerate(entries):
        seen = torch.ones((t,), dtype=torch.bool, device=cuda)
        for a in gone.get(e, ()):
            seen[a * page:(a + 1) * page] = False
        k, v = dense[e][:, :, :t].permute(0, 2, 1, 3)
        want = attend64(q[start[e]:start[e + 1]], k, v, l, hd ** -0.5, seen)[0]
        top = float(v.abs().max())
        tol = 2e-5 * top if dtype == torch.float32 else 2e-5 * top + 2.0 ** -11 * (top + want.abs())
        assert ((got[start[e]:start[e + 1]] - want).abs() <= tol).all(), e
    kv._status = None  # a caller without a status word
    again = kv.attention(*args, max_q=max(l for l, _ in entries)).double()
    assert torch.equal(again, got)


@CACHES
@pytest.mark.parametrize("l", [1, 60])
def test_a_page_that_names_nothing_beside_values_that_are_not_finite(cuda, l, cache):
    """Both at once: absent positions have no weight, and a NaN stays with the tokens that see it."""
    import torch
    kv, dense = build(cuda, [l + 60], 1, 64, 16, cache, 9)
    kv.page_table[0, 0] = -1
    at = l + 59  # the last token's own position
    kv.data[int(kv.page_table[0, at // 16]), 1, 0, at % 16, 2] = float("nan")
    q = torch.randn((l, 2, 64), device=cuda)
    got = kv.attention(q, i32(cuda, [0, l]), i32(cuda, [l + 60]), max_q=l).double()
    seen = torch.arange(l + 60, device=cuda) >= 16
    k, v = dense[0].permute(0, 2, 1, 3)
    want = attend64(q, k, v, l, 64 ** -0.5, seen)[0]
    assert got[-1, :, 2].isnan().all()
    got[-1, :, 2] = want[-1, :, 2]
    assert ((got - want).abs() <= 2e-5 * float(v.abs().max())).all()
