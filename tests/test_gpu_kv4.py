"""A paged cache in 4 bits (e2m1 codes, a scale for 32 dims) on a B200 against its definition in 64 bits.

Write: codes and scale bytes are equal to the definition's, whose only roundings to fp32 are max|x| times 1 / 6, 1 / scale
and its product with x.  Read-back: code * scale has 6 significant bits and is exact in fp32 and fp16.

Attention: K and V enter the products as the fp16 numbers that they are, so the bounds are those of the other caches
(test_gpu_paged_attention.py): fp32 queries 2e-5 * max|v| (sum |q k| scale about 11 in these inputs), fp16 queries
2^-11 * (max|v| + |out|) more."""
import numpy as np
import pytest

from test_gpu_paged_attention import plain

pytestmark = pytest.mark.gpu
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def scale_table():
    b = np.arange(256)
    with np.errstate(over="ignore"):
        return (b << 7).astype(np.uint16).view(np.float16).astype(np.float64)


def nearest(table, v):
    hi = np.searchsorted(table, v).clip(0, len(table) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = table[hi] - v, v - table[lo]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def quantise(x):
    """(packed codes, scale bytes) of float32 rows, from the definition."""
    x = np.asarray(x, np.float32)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    a = np.where(np.isfinite(b), np.abs(b), 0).max(-1)
    byte = nearest(scale_table()[:227], (a * (np.float32(1) / np.float32(6))).astype(np.float64))
    s = scale_table()[byte].astype(np.float32)
    inv = np.where(s > 0, np.float32(1) / np.where(s > 0, s, 1), 0).astype(np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        y = np.where(s[..., None] > 0, b * inv[..., None], 0).astype(np.float32)
    code = nearest(LEVELS, np.nan_to_num(np.abs(y.astype(np.float64)), posinf=1e30)) | np.signbit(y).astype(np.int64) << 3
    code = code.reshape(x.shape)
    byte = np.where(np.isnan(b).any(-1), 255, byte)
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), byte.astype(np.uint8)


def decode(data, scale):
    """float64 values of packed rows (torch)."""
    import torch
    b = data.view(torch.uint8)
    code = torch.stack([b & 15, b >> 4], -1).flatten(-2).long()
    t = torch.from_numpy(np.concatenate([LEVELS, -LEVELS])).to(b.device)
    s = torch.from_numpy(scale_table()).to(b.device)[scale.long()]
    return t[code] * s.repeat_interleave(32, -1)


def pool(cuda, pages, kvh, hd, page, seed=0):
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    data = torch.randint(0, 256, (pages, 2, kvh, page, hd // 2), generator=g, device=cuda, dtype=torch.uint8)
    scale = torch.randint(90, 130, (pages, 2, kvh, page, hd // 32), generator=g, device=cuda, dtype=torch.uint8)
    return data.view(torch.float4_e2m1fn_x2), scale


def make(cuda, kvh, hd, page, pages=40, seqs=5, max_pages=7, seed=0):
    import torch
    from ijb200 import ops
    data, scale = pool(cuda, pages, kvh, hd, page, seed)
    table = torch.randperm(pages, device=cuda)[:seqs * max_pages].view(seqs, max_pages).int().contiguous()
    return ops.PagedKV(data, table, scale, torch.zeros((1,), dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("kvh,hd,page,n", [(1, 64, 8, 1), (2, 64, 16, 37), (8, 64, 16, 64), (3, 128, 32, 33), (8, 128, 256, 29),
                                           (5, 128, 8, 50), (8, 128, 256, 1100), (5, 128, 256, 1700), (7, 64, 256, 2400)])
@pytest.mark.parametrize("src", ["float32", "float16"])
def test_append_and_gather(cuda, kvh, hd, page, n, src):
    import torch
    dtype = getattr(torch, src)
    kv = make(cuda, kvh, hd, page)
    rng = np.random.default_rng(n + hd)
    x = np.clip(rng.standard_normal((2, n, kvh, hd)) * 2.0 ** rng.integers(-18, 14, (2, n, kvh, 1)), -65000, 65000)
    if n > 3:
        x[0, 0] = 0
        x[1, 1, 0, :3] = [6.0, -6.0, 0.25]     # the scale's border, a tie
        x[0, 1, 0] = np.linspace(0, 6, hd)     # all codes, and ties between them
        x[1, 2, 0, 0] = 65000.0                # past 6 * 10240: the largest value
        x[0, 2, 0] = 2.0 ** -20                # no scale is that small: zeros
        x[0, 3, 0] = -0.0
    x = torch.from_numpy(x).to(cuda).to(dtype)
    slots = rng.permutation(5 * 7 * page)[:n]
    seq, pos = slots // (7 * page), slots % (7 * page)
    st, pt = (torch.from_numpy(a.astype(np.int32)).to(cuda) for a in (seq, pos))
    want, want_s = kv.data.view(torch.uint8).cpu().numpy(), kv.scale.cpu().numpy()
    kv.append(x[0], x[1], st, pt)
    pg, off = kv.page_table.cpu().numpy()[seq, pos // page], pos % page
    code, s = quantise(x.float().cpu().numpy())
    for i in range(n):
        want[pg[i], :, :, off[i]], want_s[pg[i], :, :, off[i]] = code[:, i], s[:, i]
    np.testing.assert_array_equal(kv.scale.cpu().numpy(), want_s)
    np.testing.assert_array_equal(kv.data.view(torch.uint8).cpu().numpy(), want)  # and every other byte as it was
    for out in (torch.float32, torch.float16):
        k, v = kv.gather(st, pt, out)
        for which, y in ((0, k), (1, v)):
            val = decode(kv.data.view(torch.uint8)[pg, which, :, off], kv.scale[pg, which, :, off])
            assert torch.equal(y.double(), val)
    assert int(kv.status) == 0


def test_every_scale_and_code_reads_back(cuda):
    """All 256 scale bytes, the infinite ones and NaN among them, with all 16 codes."""
    import torch
    kv = make(cuda, 4, 64, 32, pages=2, seqs=1, max_pages=2)
    kv.page_table[0] = torch.tensor([0, 1], dtype=torch.int32)
    kv.data.view(torch.uint8)[:] = torch.arange(256, device=cuda, dtype=torch.int32).to(torch.uint8).view(8, 32)[:4].repeat(2, 2, 1, 1).unsqueeze(3)
    kv.scale.view(-1)[:1024] = torch.arange(1024, device=cuda, dtype=torch.int32).to(torch.uint8)
    pos = torch.arange(64, dtype=torch.int32, device=cuda)
    want = decode(kv.data, kv.scale).permute(1, 0, 3, 2, 4).reshape(2, 64, 4, 64)
    for dtype in (torch.float32, torch.float16):
        for which, y in enumerate(kv.gather(torch.zeros_like(pos), pos, dtype)):
            w = want[which].to(dtype)
            assert torch.equal(torch.nan_to_num(y, nan=7.0), torch.nan_to_num(w, nan=7.0))


def test_rows_with_strides_and_odd_alignment(cuda):
    import torch
    kv, ref = make(cuda, 2, 64, 16), make(cuda, 2, 64, 16)
    ref.page_table.copy_(kv.page_table)
    seq = torch.zeros((9,), dtype=torch.int32, device=cuda)
    pos = torch.arange(9, dtype=torch.int32, device=cuda)
    for dtype in (torch.float32, torch.float16):
        wide = torch.randn((9, 3 * 128 + 5), device=cuda).to(dtype)
        k, v = wide[:, 1:129], wide[:, 130:258]
        kv.append(k, v, seq, pos)
        ref.append(k.contiguous(), v.contiguous(), seq, pos)
        assert torch.equal(kv.data.view(torch.uint8), ref.data.view(torch.uint8)) and torch.equal(kv.scale, ref.scale)


def test_infinity_nan_and_tiny_rows(cuda):
    import torch
    kv = make(cuda, 1, 64, 16)
    x = torch.zeros((2, 7, 1, 64), device=cuda)
    inf, nan = float("inf"), float("nan")
    x[0, 0, 0, :4] = torch.tensor([inf, -inf, 1.0, -0.25])   # infinities: the block's largest value
    x[0, 1, 0, 40] = nan                                     # the second block is NaN, the first is not
    x[0, 1, 0, :8] = 3.0
    x[0, 2, 0, :] = -inf
    x[0, 3, 0, :2] = torch.tensor([1e-45, -1e-40])
    x[0, 4, 0, :2] = torch.tensor([3.4e38, -1e38])
    x[0, 5, 0, 0] = -0.0
    x[0, 6, 0, :] = nan
    x[1] = torch.randn((7, 1, 64), device=cuda)
    seq = torch.zeros((7,), dtype=torch.int32, device=cuda)
    pos = torch.arange(7, dtype=torch.int32, device=cuda)
    kv.append(x[0], x[1], seq, pos)
    page = int(kv.page_table[0, 0])
    code, s = quantise(x.cpu().numpy())
    np.testing.assert_array_equal(kv.scale[page, :, 0, :7].cpu().numpy(), s[:, :, 0])
    ok = ~np.isnan(x.cpu().numpy())[:, :, 0].reshape(2, 7, 2, 32).any(-1).repeat(16, -1)  # a NaN block's codes mean nothing
    got = kv.data.view(torch.uint8)[page, :, 0, :7].cpu().numpy()
    np.testing.assert_array_equal(np.where(ok, got, 0), np.where(ok, code[:, :, 0], 0))
    k, _ = kv.gather(seq, pos)
    assert torch.isfinite(k[[0, 2, 3, 4, 5]]).all() and torch.isfinite(k[1, 0, :32]).all()
    assert k[1, 0, 32:].isnan().all() and k[6].isnan().all()
    assert k[4, 0, 0] == 61440.0 and k[0, 0, 0] == -k[0, 0, 1] == 6 * scale_table()[s[0, 0, 0, 0]]


def test_padding_and_indexes_that_name_nothing(cuda):
    import torch
    kv = make(cuda, 2, 64, 16)
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


# -------------------------------------------------------------- attention --

def build(cuda, lens, kvh, hd, page, seed=0):
    """A cache whose sequences hold lens[i] positions, pages in no order, unused page ids bad, unused rows NaN."""
    import torch
    from ijb200 import ops
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    need = [-(-max(n, 1) // page) for n in lens]
    width, total = max(need) + 1, sum(need) + 2
    table = torch.full((len(lens), width), -5, dtype=torch.int32)
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).int()
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    data = torch.randint(0, 256, (total, 2, kvh, page, hd // 2), generator=g, device=cuda, dtype=torch.uint8)
    scale = torch.full((total, 2, kvh, page, hd // 32), 255, device=cuda, dtype=torch.uint8)
    kv = ops.PagedKV(data.view(torch.float4_e2m1fn_x2), table.to(cuda), scale, torch.zeros((1,), dtype=torch.int32, device=cuda))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    for i, n in enumerate(lens):
        if n == 0:
            continue
        x = torch.randn((2, n, kvh, hd), generator=g, device=cuda)
        kv.append(x[0], x[1], i32([i] * n), i32(list(range(n))))
    dense = []
    for i, n in enumerate(lens):
        pos = torch.arange(n, device=cuda)
        pg = table[i].to(cuda)[pos // page].long()
        dense.append(decode(data[pg, :, :, pos % page], scale[pg, :, :, pos % page]).permute(1, 2, 0, 3))
    return kv, dense


def check(cuda, entries, kvh, group, hd, page, dtype, seed=0, seqs=None, max_q=None, stride=0, gaps=0):
    """entries: (new tokens, cached positions in all)."""
    import torch
    dtype = getattr(torch, dtype)
    seqs = list(range(len(entries))) if seqs is None else seqs
    lens = [max([t for (l, t), s in zip(entries, seqs) if s == i], default=1) for i in range(max(seqs) + 1)]
    kv, dense = build(cuda, lens, kvh, hd, page, seed)
    start = np.cumsum([0] + [l for l, _ in entries]).tolist()
    n = start[-1] + gaps
    g = torch.Generator(device=cuda)
    g.manual_seed(seed + 1)
    heads = kvh * group
    q = (torch.randn((n, heads * hd + stride), generator=g, device=cuda) * 1.5).to(dtype)[:, stride:].unflatten(1, (heads, hd))
    out = torch.full((n, heads, hd), 7.0, dtype=dtype, device=cuda)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    kv_len = [t for _, t in entries]
    mq = max(l for l, _ in entries) if max_q is None else max_q
    got = kv.attention(q, i32(start), i32(kv_len), seq=i32(seqs), max_q=mq, out=out)
    assert int(kv.status) == 0
    want = plain(q, start, seqs, kv_len, dense, group, hd ** -0.5)
    top = max(float(d[1].abs().max()) if d.numel() else 0.0 for d in dense)
    tol = torch.full_like(want, 2e-5 * top)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -11 * (top + want.abs())
    err = (got.double() - want).abs()
    bad = ~(err[:start[-1]] <= tol[:start[-1]])
    assert not bad.any(), (int(bad.sum()), float(err[:start[-1]].max()), bad.nonzero()[:4].tolist())
    assert torch.all(got[start[-1]:] == 7.0)
    return kv, q, got


TYPES = pytest.mark.parametrize("dtype", ["float32", "float16"])


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kvh,group,page,entries", [
    (1, 1, 8, [(1, 1)]), (2, 4, 16, [(1, 31), (1, 32), (1, 33)]), (8, 4, 16, [(1, 1957)]),
    (8, 3, 32, [(1, 5), (0, 9), (1, 700), (1, 64)]), (4, 8, 64, [(1, 1000), (2, 129)]), (3, 5, 8, [(3, 40), (1, 1), (2, 2)]),
    (1, 16, 16, [(1, 300)]), (2, 2, 128, [(8, 1000), (5, 5), (1, 20000)]), (8, 1, 256, [(16, 16), (16, 4000)]),
    (2, 3, 8, [(5, 5), (3, 9), (1, 777)]), (2, 8, 16, [(1, 65), (1, 4097)])])
def test_short_entries(cuda, hd, kvh, group, page, entries, dtype):
    check(cuda, entries, kvh, group, hd, page, dtype, seed=hd + page)


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
def test_ragged_batch(cuda, hd, dtype):
    rng = np.random.default_rng(5)
    check(cuda, [(1, int(t)) for t in rng.integers(1, 1300, 64)], 8, 4, hd, 16, dtype)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens", [1, 3, 100])
def test_long_sums_of_fp32_queries(cuda, hd, tokens):
    """Over many blocks the sums keep fp32's precision: rel-L2 within 2^-19."""
    import torch
    kv, dense = build(cuda, [20000], 2, hd, 16, 3)
    g = torch.Generator(device=cuda)
    g.manual_seed(4)
    q = torch.randn((tokens, 8, hd), generator=g, device=cuda)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    got = kv.attention(q, i32([0, tokens]), i32([20000]), max_q=tokens).double()
    want = plain(q, [0, tokens], [0], [20000], dense, 4, hd ** -0.5)
    assert float((got - want).norm() / want.norm()) < 2.0 ** -19


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_that_see_nothing(cuda, hd, dtype):
    """kv_len shorter than the entry, and 0: zeros, and the others as they are."""
    check(cuda, [(4, 2), (1, 0), (3, 0), (2, 70), (4, 4)], 2, 2, hd, 16, dtype, seed=3)
    check(cuda, [(40, 2), (50, 0), (30, 10)], 2, 2, hd, 16, dtype, seed=3)


@TYPES
def test_sequences_by_name_strides_and_rows_behind(cuda, dtype):
    check(cuda, [(1, 50), (2, 33), (1, 90), (1, 50)], 2, 4, 64, 16, dtype, seqs=[2, 0, 1, 2], stride=8, gaps=3)
    check(cuda, [(1, 50), (2, 33)], 2, 4, 128, 16, dtype, stride=3)
    check(cuda, [(60, 60), (70, 90)], 2, 4, 128, 16, dtype, stride=3, gaps=2)


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kvh,group,page,entries", [
    (2, 4, 16, [(33, 33)]), (1, 1, 8, [(130, 130), (17, 17)]), (2, 4, 16, [(64, 64), (65, 65), (31, 200)]),
    (2, 3, 32, [(257, 300)]), (1, 8, 16, [(100, 2000)]), (4, 4, 64, [(300, 300), (1, 900), (2, 129), (0, 5), (77, 1000)]),
    (1, 5, 16, [(513, 513)]), (2, 4, 16, [(40, 20), (200, 130)]), (8, 4, 16, [(128, 3001)]), (1, 16, 128, [(129, 129)]),
    (2, 2, 16, [(1000, 1000), (900, 1100)])])
def test_long_entries(cuda, hd, kvh, group, page, entries, dtype):
    check(cuda, entries, kvh, group, hd, page, dtype, seed=hd + page + 1)


@pytest.mark.parametrize("max_q", [0, 300])
def test_unknown_lengths(cuda, max_q):
    for entries in ([(1, 40), (1, 900)], [(200, 300)], [(1, 70), (150, 150), (3, 3), (1, 2000)],
                    [(1, 5)] * 12 + [(99, 99)] + [(2, 400)] * 6):
        check(cuda, entries, 2, 4, 64, 16, "float32", max_q=max_q)
        check(cuda, entries, 2, 4, 128, 16, "float16", max_q=max_q)


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("byte", [255, 248])
def test_blocks_behind_a_token_do_not_reach_it(cuda, hd, dtype, byte):
    """A block of K or V that is NaN (its scale's byte 255) or infinite (248) at a later token's position changes no
    earlier token's output; tokens that see it get no finite value where it stands."""
    import torch
    for entries, at in (([(1, 40), (6, 50), (3, 3)], 47), ([(300, 700), (40, 40)], 560), ([(600, 600)], 1), ([(900, 5000)], 4999)):
        e = 1 if len(entries) == 3 else 0
        kv, q, clean = check(cuda, entries, 2, 2, hd, 16, dtype, seed=11)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
        start, kv_len = np.cumsum([0] + [l for l, _ in entries]).tolist(), [t for _, t in entries]
        page, off = int(kv.page_table[e, at // 16]), at % 16
        first = start[e] + at - (kv_len[e] - entries[e][0])  # the token at that position
        for which, head, block in ((1, 0, 0), (1, 1, hd // 32 - 1), (0, 1, 1)):
            kept = kv.scale[page, which, head, off, block].clone()
            kv.scale[page, which, head, off, block] = byte
            got = kv.attention(q, i32(start), i32(kv_len), max_q=max(l for l, _ in entries))
            kv.scale[page, which, head, off, block] = kept
            heads = slice(head * 2, head * 2 + 2)
            sees = torch.zeros(got.shape[0], dtype=torch.bool, device=cuda)
            sees[first:start[e + 1]] = True
            assert torch.isfinite(got[~sees]).all()
            tol = 4e-5 * 6 if dtype == "float32" else 2.0 ** -9 * 6  # both sums' own errors (see above)
            assert float((got[~sees].double() - clean[~sees].double()).abs().max()) <= tol
            if which == 1:
                bad = got[sees][:, heads, 32 * block:32 * block + 32]
                assert not torch.isfinite(bad).any()
            elif byte == 255:
                assert not torch.isfinite(got[sees][:, heads]).any()
            other = torch.ones(got.shape[1], dtype=torch.bool)
            other[heads] = False
            assert torch.equal(got[sees][:, other.to(cuda)], clean[sees][:, other.to(cuda)])
        assert int(kv.status) == 0


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens", [1, 4, 90])
def test_pages_that_name_nothing_are_absent(cuda, hd, dtype, tokens):
    """Positions whose page id names no page have no weight, as if the sequence did not have them."""
    import torch
    kv, dense = build(cuda, [400], 2, hd, 16, 5)
    g = torch.Generator(device=cuda)
    g.manual_seed(6)
    q = torch.randn((tokens, 4, hd), generator=g, device=cuda).to(getattr(torch, dtype))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    for pages, ids in (([3], [-1]), ([0, 24], [1 << 30, -9]), (list(range(25)), [-1] * 25)):
        kept = kv.page_table[0].clone()
        for p, i in zip(pages, ids):
            kv.page_table[0, p] = i
        got = kv.attention(q, i32([0, tokens]), i32([400]), max_q=tokens)
        assert int(kv.status) != 0
        kv.status.zero_()
        kv.page_table[0].copy_(kept)
        there = torch.ones(400, dtype=torch.bool, device=cuda)
        for p in pages:
            there[16 * p:16 * p + 16] = False
        s = torch.einsum("lhgd,htd->hglt", q.double().view(tokens, 2, 2, hd), dense[0][0]) * hd ** -0.5
        seen = (torch.arange(400, device=cuda) <= (400 - tokens + torch.arange(tokens, device=cuda)).unsqueeze(1)) & there
        p = torch.exp(s - torch.where(seen, s, -torch.inf).amax(-1, keepdim=True).clamp(min=-1e300)) * seen
        p = torch.where(seen, p, 0.0)
        o = torch.einsum("hglt,htd->lhgd", p, dense[0][1]) / p.sum(-1).clamp(min=1e-300).permute(2, 0, 1).unsqueeze(-1)
        top = float(dense[0][1].abs().max())
        tol = 2e-5 * top + (2.0 ** -11 * 2 * top if dtype == "float16" else 0)
        assert float((got.double() - o.reshape(got.shape)).abs().max()) <= tol


@TYPES
def test_the_largest_values(cuda, dtype):
    """Scales up to 10240 and down to 2^-17: values up to 61440 enter the products as they are."""
    import torch
    kv, dense = build(cuda, [70], 1, 64, 16, 8)
    page = kv.page_table[0, :5].long()
    q = torch.zeros((1, 2, 64), device=cuda, dtype=getattr(torch, dtype))
    q[:, :, 0] = 1e-5
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    for byte in (226, 1):
        kv.scale[page] = byte
        val = decode(kv.data, kv.scale)
        rows = torch.cat([val[p] for p in page.tolist()], 2)[:, 0, :70]  # [K V, 70, 64]
        got = kv.attention(q, i32([0, 1]), i32([70]), max_q=1).double()
        s = (q[0].double() @ rows[0].T) * 0.125
        want = torch.softmax(s, -1) @ rows[1]
        top = float(rows[1].abs().max())
        # q: 1e-5 is below fp16's normal range: 2^-25 absolute (fp16 queries are that number); sum |q k| < 1
        tol = top * 2.0 ** -19 + top * 61440 * 2.0 ** -25 / 8 * 2 if dtype == "float32" and byte == 226 else top * 2.0 ** -19
        if dtype == "float16":
            # at byte 1 the outputs are below 2^-14, where fp16's steps are 2^-24: their rounding is off by up to 2^-25,
            # whatever their size
            tol = tol + 2.0 ** -11 * (top + want.abs()) + 2.0 ** -25
        assert bool(((got[0] - want).abs() <= tol).all())


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens", [1, 3])
def test_bad_blocks_and_absent_pages_among_many_entries(cuda, hd, dtype, tokens):
    """40 sequences (more than get a cluster of CTAs each): a NaN block of V behind a token's position, and pages that
    name nothing, reach no other entry and no earlier token."""
    import torch
    lens = [5 + 37 * i for i in range(40)]
    kv, q, clean = check(cuda, [(min(tokens, n), n) for n in lens], 2, 2, hd, 16, dtype, seed=13)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    start = list(range(0, 40 * tokens + 1, tokens))
    tol = 4e-5 * 6 if dtype == "float32" else 2.0 ** -9 * 6
    for e in (3, 30, 39):
        at = lens[e] - 1
        page = int(kv.page_table[e, at // 16])
        kept = kv.scale[page, 1, 0, at % 16].clone()
        kv.scale[page, 1, 0, at % 16] = 255
        got = kv.attention(q, i32(start), i32(lens), max_q=tokens)
        kv.scale[page, 1, 0, at % 16] = kept
        hit = torch.zeros(got.shape[:2], dtype=torch.bool, device=cuda)
        hit[start[e + 1] - 1, :2] = True  # the last token, the first KV head
        assert got[hit].isnan().all()
        assert float((got[~hit].double() - clean[~hit].double()).abs().max()) <= tol
        kept = int(kv.page_table[e, 0])
        kv.page_table[e, 0] = -1
        got = kv.attention(q, i32(start), i32(lens), max_q=tokens)
        assert int(kv.status) != 0
        kv.status.zero_()
        kv.page_table[e, 0] = kept
        other = torch.ones(got.shape[0], dtype=torch.bool, device=cuda)
        other[start[e]:start[e + 1]] = False
        assert float((got[other].double() - clean[other].double()).abs().max()) <= tol
        k, v = kv.gather(i32([e] * (lens[e] - 16)), i32(list(range(16, lens[e]))), torch.float32)
        for t in range(tokens):
            n = lens[e] - tokens + t + 1 - 16
            s = torch.einsum("hgd,thd->hgt", q[start[e] + t].double().view(2, 2, hd), k[:n].double()) * hd ** -0.5
            want = torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), v[:n].double()).reshape(4, hd)
            assert float((got[start[e] + t].double() - want).abs().max()) <= tol


@TYPES
@pytest.mark.parametrize("entries,kvh", [([(1, 2000)], 8), ([(1, 70)] * 3 + [(1, 3000)], 8), ([(4, 500), (1, 1)], 2),
                                         ([(1, 33000)], 1), ([(1, 31000), (2, 5)], 4), ([(0, 7)], 8), ([(3, 0), (1, 9)], 3)])
def test_calls_of_few_tiles(cuda, entries, kvh, dtype):
    """One launch (a cluster of CTAs a tile) up to its limits, two behind them."""
    from ijb200 import lib
    check(cuda, entries, kvh, 4, 64, 16, dtype, seed=2)
    check(cuda, entries, kvh, 4, 128, 16, dtype, seed=2)
    kv, _ = build(cuda, [max(t, 1) for _, t in entries], kvh, 64, 16)
    import torch
    n = sum(l for l, _ in entries)
    q = torch.zeros((max(n, 1), 4 * kvh, 64), device=cuda, dtype=getattr(torch, dtype))
    start = np.cumsum([0] + [l for l, _ in entries]).astype(np.int32)
    args = (q, torch.from_numpy(start).to(cuda), torch.tensor([t for _, t in entries], dtype=torch.int32, device=cuda))
    before = lib.load().ijb_kernel_launches()
    kv.attention(*args, max_q=max(l for l, _ in entries) or 1)
    tiles, positions = len(entries) * kvh, kv.page_table.shape[1] * 16
    few = positions <= 32768 if tiles <= 8 else tiles <= 32 and positions <= 512 * tiles
    assert lib.load().ijb_kernel_launches() - before == (1 if few else 2)
