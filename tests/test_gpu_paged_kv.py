"""The paged cache's write and read-back on a B200 against their definition in 64 bits.

e4m3 rows must be bit-exact: scaling by a power of two is exact, so the only rounding is the
one to e4m3.  Read-back is exact in fp32 (a power of two times a 4-bit significand) and one
rounding in fp16."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def quantise(x):
    """(e4m3 codes, scale bytes) of float64 rows, from the definition: nearest of all finite e4m3
    values, ties to the even code."""
    import torch
    table = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()  # 0..448, rising
    a = np.where(np.isfinite(x), np.abs(x), 0).max(-1)
    e = np.full(a.shape, -126)
    for i in np.ndindex(a.shape):
        while a[i] > 448.0 * 2.0 ** e[i]:
            e[i] += 1
    y = np.minimum(np.abs(x) / 2.0 ** e[..., None], 448.0)
    hi = np.searchsorted(table, np.nan_to_num(y)).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    d = (table[hi] - y) - (y - table[lo])  # < 0: hi is nearer
    code = np.where((d < 0) | ((d == 0) & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    code = np.where(np.isnan(x), 127, code)
    return code | (np.signbit(x).astype(np.uint8) << 7), (e + 127).astype(np.uint8)


def make(cuda, kvh, hd, page, e4m3, pages=40, seqs=5, max_pages=7, seed=0):
    import torch
    from ijb200 import ops
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    shape = (pages, 2, kvh, page, hd)
    data = torch.randint(0, 120, shape, generator=g, device=cuda, dtype=torch.uint8)
    data = data.view(torch.float8_e4m3fn) if e4m3 else data.half()
    scale = torch.randint(100, 140, shape[:-1], generator=g, device=cuda, dtype=torch.uint8) if e4m3 else None
    table = torch.randperm(pages, generator=g, device=cuda)[:seqs * max_pages].view(seqs, max_pages).int().contiguous()
    status = torch.zeros((1,), dtype=torch.int32, device=cuda)
    return ops.PagedKV(data, table, scale, status)


def rows(cuda, n, kvh, hd, dtype, seed):
    import torch
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((2, n, kvh, hd)) * 2.0 ** rng.integers(-12, 10, (2, n, kvh, 1))
    x = np.clip(x, -60000, 60000)
    if n > 3:
        x[0, 0] = 0
        x[1, 1, 0, :2] = [448.0, -448.0]          # exactly at a scale's border
        x[0, 1, 0] = np.linspace(0, 1, hd)
        x[1, 2, 0, 0] = np.nextafter(np.float32(448.0 * 64), np.float32(1e9)) if dtype == torch.float32 else 28688.0
    return torch.from_numpy(x).to(cuda).to(dtype)


@pytest.mark.parametrize("kvh,hd,page,n", [(1, 64, 8, 1), (2, 64, 16, 37), (8, 64, 16, 64), (3, 128, 32, 33),
                                           (8, 128, 256, 29), (5, 128, 8, 50), (8, 128, 256, 1100), (5, 128, 256, 1700), (7, 64, 256, 2400)])
@pytest.mark.parametrize("src", ["float32", "float16"])
@pytest.mark.parametrize("e4m3", [True, False])
def test_append_and_gather(cuda, kvh, hd, page, n, src, e4m3):
    import torch
    dtype = getattr(torch, src)
    kv = make(cuda, kvh, hd, page, e4m3)
    x = rows(cuda, n, kvh, hd, dtype, n + hd)
    rng = np.random.default_rng(n)
    slots = rng.permutation(5 * 7 * page)[:n]  # distinct places over all sequences
    seq, pos = slots // (7 * page), slots % (7 * page)
    st, pt = (torch.from_numpy(a.astype(np.int32)).to(cuda) for a in (seq, pos))
    before, before_s = kv.data.clone(), kv.scale.clone() if e4m3 else None
    kv.append(x[0], x[1], st, pt)
    pg, off = kv.page_table.cpu().numpy()[seq, pos // page], pos % page
    want, got = before.view(torch.uint8).cpu().numpy(), kv.data.view(torch.uint8).cpu().numpy()
    x64 = np.moveaxis(x.double().cpu().numpy(), 0, 1)  # [n, K V, kvh, hd]
    if e4m3:
        code, s = quantise(x64)
        want_s = before_s.cpu().numpy()
        for i in range(n):
            want[pg[i], :, :, off[i]], want_s[pg[i], :, :, off[i]] = code[i], s[i]
        np.testing.assert_array_equal(kv.scale.cpu().numpy(), want_s)
    else:
        for i in range(n):
            want[pg[i], :, :, off[i]] = x64[i].astype(np.float16).view(np.uint8)
    np.testing.assert_array_equal(got, want)  # the rows, and every other byte as it was
    for out in (torch.float32, torch.float16):
        k, v = kv.gather(st, pt, out)
        for which, y in ((0, k), (1, v)):
            val = kv.data[pg, which, :, off].double()
            if e4m3:
                val = val * torch.pow(2.0, kv.scale[pg, which, :, off].double() - 127).unsqueeze(-1)
            assert torch.equal(y, val.to(out))
    assert int(kv.status) == 0


def test_rows_with_strides_and_odd_alignment(cuda):
    import torch
    kv, ref = make(cuda, 2, 64, 16, True), make(cuda, 2, 64, 16, True)
    seq = torch.zeros((9,), dtype=torch.int32, device=cuda)
    pos = torch.arange(9, dtype=torch.int32, device=cuda)
    for dtype in (torch.float32, torch.float16):
        wide = torch.randn((9, 3 * 128 + 5), device=cuda).to(dtype)
        k, v = wide[:, 1:129], wide[:, 130:258]  # neither 16-byte aligned nor evenly spaced
        kv.append(k, v, seq, pos)
        ref.append(k.contiguous(), v.contiguous(), seq, pos)
        assert torch.equal(kv.data.view(torch.uint8), ref.data.view(torch.uint8)) and torch.equal(kv.scale, ref.scale)


def test_infinity_nan_and_tiny_rows(cuda):
    import torch
    kv = make(cuda, 1, 64, 16, True)
    x = torch.zeros((2, 6, 1, 64), device=cuda)
    inf, nan = float("inf"), float("nan")
    x[0, 0, 0, :4] = torch.tensor([inf, -inf, nan, 1.0])
    x[0, 1, 0, :] = nan
    x[0, 2, 0, :] = -inf
    x[0, 3, 0, :2] = torch.tensor([1e-45, -1e-40])
    x[0, 4, 0, :2] = torch.tensor([3.4e38, -1e38])
    x[0, 5, 0, 0] = -0.0
    seq = torch.zeros((6,), dtype=torch.int32, device=cuda)
    pos = torch.arange(6, dtype=torch.int32, device=cuda)
    kv.append(x[0], x[1], seq, pos)
    page = int(kv.page_table[0, 0])
    code, s = quantise(x[0].double().cpu().numpy()[:, 0, :])
    got = kv.data.view(torch.uint8)[page, 0, 0, :6].cpu().numpy()
    np.testing.assert_array_equal(got & np.where(np.isnan(x[0, :, 0].cpu().numpy()), 0x7f, 0xff),
                                  code & np.where(np.isnan(x[0, :, 0].cpu().numpy()), 0x7f, 0xff))
    np.testing.assert_array_equal(kv.scale[page, 0, 0, :6].cpu().numpy(), s)


def test_padding_and_indexes_that_name_nothing(cuda):
    """Padding is skipped silently; a sequence, position or page outside the cache is skipped and reported."""
    import torch
    kv = make(cuda, 2, 64, 16, True)
    kv.page_table[4, 6] = 40   # one past the pool
    kv.page_table[4, 5] = -1
    before, before_s = kv.data.view(torch.uint8).clone(), kv.scale.clone()
    x = torch.randn((2, 1, 2, 64), device=cuda)
    for seq, pos, bad in [(0, -1, 0), (-7, -1, 0), (5, 0, 1), (-1, 0, 1), (0, 7 * 16, 1), (4, 6 * 16, 1), (4, 5 * 16, 1)]:
        kv.status.zero_()
        s, p = (torch.tensor([a], dtype=torch.int32, device=cuda) for a in (seq, pos))
        kv.append(x[0], x[1], s, p)
        assert bool(int(kv.status)) == bool(bad), (seq, pos)
        kv.status.zero_()
        kv.gather(s, p)
        assert bool(int(kv.status)) == bool(bad), (seq, pos)
    assert torch.equal(kv.data.view(torch.uint8), before) and torch.equal(kv.scale, before_s)
