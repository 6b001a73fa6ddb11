"""ijb_paged_attention on a B200 against softmax attention in 64 bits over the same cache.

Tolerances (before the first run).  fp32 queries: q and p enter as two fp16 parts (relative
2^-22), products are summed in fp32 over head_dim <= 128 terms, so a score of sum|q k| scale
<= 40 is off by about 40 * (2^-22 + 8 * 2^-24) < 3e-5 and the softmax weights by as much
relative; for the inputs here sum|q k| scale is about 11, which gives 1e-5, and twice that in
an output (weights and their sum): 2e-5 * max|v|.  fp16 queries add a rounding of each weight and of the
output, 2^-11 each: 2^-11 * (max|v| + |out|) more.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def build(cuda, lens, kvh, hd, page, cache, seed=0, extra_seqs=0):
    """A cache whose sequences hold lens[i] positions, pages in no order, unused page ids bad, unused rows NaN."""
    import torch
    from ijb200 import ops
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    need = [-(-max(n, 1) // page) for n in lens]
    width, total = max(need) + 1, sum(need) + 2
    table = torch.full((len(lens) + extra_seqs, width), -5, dtype=torch.int32)
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).int()
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    x = torch.full((total, 2, kvh, page, hd), float("nan"), device=cuda)
    dense = []
    for i, n in enumerate(lens):
        rows = torch.randn((2, n, kvh, hd), generator=g, device=cuda)
        pos = torch.arange(n, device=cuda)
        pg = table[i].to(cuda)[pos // page].long()
        x[pg, :, :, pos % page] = rows.permute(1, 0, 2, 3)
    scale = None
    if cache == "f16":
        data = x.half()
        val = data.double()
    else:
        a = torch.nan_to_num(x).abs().amax(-1)
        e = torch.ceil(torch.log2(a.clamp(min=1e-30) / 448)).clamp(min=-126)
        data = (x * torch.exp2(-e).unsqueeze(-1)).to(torch.float8_e4m3fn)
        scale = torch.where(a > 0, e + 127, torch.full_like(e, 254)).to(torch.uint8)  # unused rows: a huge scale
        val = data.double() * torch.pow(2.0, scale.double() - 127).unsqueeze(-1)
    for i, n in enumerate(lens):
        pos = torch.arange(n, device=cuda)
        pg = table[i].to(cuda)[pos // page].long()
        dense.append(val[pg, :, :, pos % page].permute(1, 2, 0, 3))  # [K V, kvh, n, hd]
    status = torch.zeros((1,), dtype=torch.int32, device=cuda)
    return ops.PagedKV(data, table.to(cuda), scale, status), dense


def plain(q, start, seqs, kv_len, dense, group, scale):
    import torch
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for e in range(len(kv_len)):
        l, t = start[e + 1] - start[e], kv_len[e]
        if l == 0 or t == 0:
            continue
        k, v = dense[seqs[e]][:, :, :t]
        x = q[start[e]:start[e + 1]].double().view(l, -1, group, q.shape[2])
        s = torch.einsum("lhgd,htd->hglt", x, k) * scale
        seen = torch.arange(t, device=q.device) <= (t - l + torch.arange(l, device=q.device)).unsqueeze(1)
        p = torch.where(seen, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
        p = torch.where(seen, torch.exp(s - torch.where(seen, s, -torch.inf).amax(-1, keepdim=True)), 0.0)
        o = torch.einsum("hglt,htd->lhgd", p, v) / p.sum(-1).permute(2, 0, 1).unsqueeze(-1)
        o[~seen.any(-1)] = 0
        out[start[e]:start[e + 1]] = o.reshape(l, -1, q.shape[2])
    return out


def check(cuda, entries, kvh, group, hd, page, cache, dtype, seed=0, seqs=None, max_q=None, stride=0, gaps=0):
    """entries: (new tokens, cached positions in all)."""
    import torch
    dtype = getattr(torch, dtype)
    seqs = list(range(len(entries))) if seqs is None else seqs
    lens = [max([t for (l, t), s in zip(entries, seqs) if s == i], default=1) for i in range(max(seqs) + 1)]
    kv, dense = build(cuda, lens, kvh, hd, page, cache, seed)
    start = np.cumsum([0] + [l for l, _ in entries]).tolist()
    n = start[-1] + gaps
    g = torch.Generator(device=cuda)
    g.manual_seed(seed + 1)
    heads = kvh * group
    q = (torch.randn((n, heads * hd + stride), generator=g, device=cuda) * 1.5).to(dtype)[:, stride:].view(n, heads, hd) \
        if stride else (torch.randn((n, heads, hd), generator=g, device=cuda) * 1.5).to(dtype)
    out = torch.full((n, heads, hd), 7.0, dtype=dtype, device=cuda)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    kv_len = [t for _, t in entries]
    mq = max(l for l, _ in entries) if max_q is None else max_q
    got = kv.attention(q, i32(start), i32(kv_len), seq=i32(seqs), max_q=mq, out=out)
    assert int(kv.status) == 0
    want = plain(q, start, seqs, kv_len, dense, group, hd ** -0.5)
    top = max(float(d[1].abs().max()) if d.numel() else 0.0 for d in dense)
    tol = 2e-5 * top
    if dtype == torch.float16:
        tol = tol + 2.0 ** -11 * (top + want.abs())
    err = (got.double() - want).abs()
    bad = ~(err[:start[-1]] <= (tol[:start[-1]] if dtype == torch.float16 else tol))
    assert not bad.any(), (int(bad.sum()), float(err[:start[-1]].max()), bad.nonzero()[:4].tolist())
    assert torch.all(got[start[-1]:] == 7.0)
    return kv, q, got


CACHES = pytest.mark.parametrize("cache", ["f16", "e4m3"])
TYPES = pytest.mark.parametrize("dtype", ["float32", "float16"])


@CACHES
@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kvh,group,page,entries", [
    (1, 1, 8, [(1, 1)]), (2, 4, 16, [(1, 31), (1, 32), (1, 33)]), (8, 4, 16, [(1, 1957)]),
    (8, 3, 32, [(1, 5), (0, 9), (1, 700), (1, 64)]), (4, 8, 64, [(1, 1000), (2, 129)]), (3, 5, 8, [(3, 40), (1, 1), (2, 2)]),
    (1, 16, 16, [(1, 300)]), (2, 2, 128, [(8, 1000), (5, 5), (1, 20000)]), (8, 1, 256, [(16, 16), (16, 4000)])])
def test_short_entries(cuda, hd, kvh, group, page, entries, cache, dtype):
    check(cuda, entries, kvh, group, hd, page, cache, dtype, seed=hd + page)


@CACHES
@TYPES
def test_ragged_batch(cuda, cache, dtype):
    rng = np.random.default_rng(5)
    check(cuda, [(1, int(t)) for t in rng.integers(1, 1300, 64)], 8, 4, 64, 16, cache, dtype)


@CACHES
@pytest.mark.parametrize("hd", [64, 128])
def test_long_sums_of_fp32_queries(cuda, cache, hd):
    """Over many blocks the sums keep fp32's precision: rel-L2 within 2^-19 (1.9e-6; the 32-bit plain form has 3e-6 here)."""
    import torch
    kv, dense = build(cuda, [20000], 2, hd, 16, cache, 3)
    g = torch.Generator(device=cuda)
    g.manual_seed(4)
    q = torch.randn((100, 8, hd), generator=g, device=cuda)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    got = kv.attention(q, i32([0, 100]), i32([20000]), max_q=100).double()
    want = plain(q, [0, 100], [0], [20000], dense, 4, hd ** -0.5)
    assert float((got - want).norm() / want.norm()) < 2.0 ** -19


@CACHES
@TYPES
def test_rows_that_see_nothing(cuda, cache, dtype):
    """kv_len shorter than the entry, and 0: zeros, and the others as they are."""
    check(cuda, [(4, 2), (1, 0), (3, 0), (2, 70), (4, 4)], 2, 2, 64, 16, cache, dtype, seed=3)


@TYPES
def test_sequences_by_name_strides_and_rows_behind(cuda, dtype):
    """Entries that name sequences in another order, one of them twice; a row stride; rows behind the last entry."""
    check(cuda, [(1, 50), (2, 33), (1, 90), (1, 50)], 2, 4, 64, 16, "f16", dtype, seqs=[2, 0, 1, 2], stride=8, gaps=3)
    check(cuda, [(1, 50), (2, 33)], 2, 4, 128, 16, "e4m3", dtype, stride=3)


@CACHES
@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kvh,group,page,entries", [
    (2, 4, 16, [(33, 33)]), (1, 1, 8, [(130, 130), (17, 17)]), (2, 4, 16, [(64, 64), (65, 65), (31, 200)]),
    (2, 3, 32, [(257, 300)]), (1, 8, 16, [(100, 2000)]), (4, 4, 64, [(300, 300), (1, 900), (2, 129), (0, 5), (77, 1000)]),
    (1, 5, 16, [(513, 513)]), (2, 4, 16, [(40, 20), (200, 130)]), (8, 4, 16, [(128, 3001)]), (1, 16, 128, [(129, 129)]),
    (2, 2, 16, [(1000, 1000), (900, 1100)])])
def test_long_entries(cuda, hd, kvh, group, page, entries, cache, dtype):
    check(cuda, entries, kvh, group, hd, page, cache, dtype, seed=hd + page + 1)


@pytest.mark.parametrize("max_q", [0, 300])
def test_unknown_lengths(cuda, max_q):
    """max_q 0 (unknown) or larger than any entry, on short, long and mixed batches."""
    for entries in ([(1, 40), (1, 900)], [(200, 300)], [(1, 70), (150, 150), (3, 3), (1, 2000)],
                    [(1, 5)] * 12 + [(99, 99)] + [(2, 400)] * 6):
        check(cuda, entries, 2, 4, 64, 16, "f16", "float32", max_q=max_q)
        check(cuda, entries, 2, 4, 128, 16, "e4m3", "float16", max_q=max_q)


@CACHES
@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_values_behind_a_token_do_not_reach_it(cuda, hd, cache, dtype, value):
    """A K or V that is not finite at a later token's position changes no earlier token's output (an e4m3
    cache holds no infinity); tokens that see it get no finite value where it stands."""
    import torch
    if cache == "e4m3" and value == float("inf"):
        pytest.skip("e4m3 has no infinity")
    for entries, at in (([(1, 40), (6, 50), (3, 3)], 47), ([(300, 700), (40, 40)], 560), ([(600, 600)], 1), ([(900, 5000)], 4999)):
        e = 1 if len(entries) == 3 else 0
        kv, q, clean = check(cuda, entries, 2, 2, hd, 16, cache, dtype, seed=11)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
        start, kv_len = np.cumsum([0] + [l for l, _ in entries]).tolist(), [t for _, t in entries]
        page, off = int(kv.page_table[e, at // 16]), at % 16
        first = start[e] + at - (kv_len[e] - entries[e][0])  # the token at that position
        for which, head, dim in ((1, 0, 5), (0, 1, hd - 1)):
            kept = kv.data[page, which, head, off].clone()
            kv.data[page, which, head, off, dim] = value
            got = kv.attention(q, i32(start), i32(kv_len), max_q=max(l for l, _ in entries))
            kv.data[page, which, head, off] = kept
            heads = slice(head * 2, head * 2 + 2)
            sees = torch.zeros(got.shape[0], dtype=torch.bool, device=cuda)
            sees[first:start[e + 1]] = True
            assert torch.isfinite(got[~sees]).all()
            tol = 4e-5 * 5 if dtype == "float32" else 2.0 ** -9 * 5  # both sums' own errors (see above)
            assert float((got[~sees].double() - clean[~sees].double()).abs().max()) <= tol
            if which == 1 or value != value:
                bad = got[sees][:, heads, dim] if which == 1 else got[sees][:, heads]
                assert not torch.isfinite(bad).any()
            other = torch.ones(got.shape[1], dtype=torch.bool)
            other[heads] = False
            assert torch.equal(got[sees][:, other.to(cuda)], clean[sees][:, other.to(cuda)])
        assert int(kv.status) == 0


@CACHES
@TYPES
@pytest.mark.parametrize("entry", [(5, 3), (300, 40)])
def test_values_that_are_not_finite_and_rows_that_see_nothing(cuda, entry, cache, dtype):
    """Tokens before position 0 get zeros whatever V holds at the positions there are."""
    import torch
    kv, q, clean = check(cuda, [entry], 2, 2, 64, 16, cache, dtype, seed=4)
    kv.data[int(kv.page_table[0, 0]), 1, :, 0, 3] = float("nan")
    got = kv.attention(q, torch.tensor([0, entry[0]], dtype=torch.int32, device=cuda),
                       torch.tensor([entry[1]], dtype=torch.int32, device=cuda))
    none = entry[0] - entry[1]
    assert torch.all(got[:none] == 0) and torch.all(got[none:, :, 3].isnan())


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_scores_that_are_not_finite(cuda, hd, dtype, value):
    """A score of NaN or +infinity at any position, in the first block of an entry or a later one, leaves no finite
    value in the rows that see it."""
    import torch
    kv, q, clean = check(cuda, [(200, 500)], 1, 2, hd, 16, "f16", dtype, seed=5)
    for at in [*range(16), 301, 318, 319, 400, 415]:
        page, off = int(kv.page_table[0, at // 16]), at % 16
        kept = kv.data[page, 0, 0, off, 0].clone()
        kv.data[page, 0, 0, off, 0] = value
        got = kv.attention(q, torch.tensor([0, 200], dtype=torch.int32, device=cuda),
                           torch.tensor([500], dtype=torch.int32, device=cuda))
        kv.data[page, 0, 0, off, 0] = kept
        hit = torch.arange(300, 500, device=cuda).unsqueeze(1) >= at
        hit = hit & (q[:, :, 0] > 0) if value > 0 else hit.expand(200, 2)
        assert not torch.isfinite(got[hit]).any(), at
        rest = torch.arange(300, 500, device=cuda) < at
        tol = 4e-5 * 5 if dtype == "float32" else 2.0 ** -9 * 5
        assert rest.sum() == 0 or float((got[rest].double() - clean[rest].double()).abs().max()) <= tol


def test_entries_that_do_not_fit_are_left_and_reported(cuda):
    """Bad starts, sequences and lengths, and an entry longer than max_q: unwritten and reported, the others computed."""
    import torch
    kv, q, clean = check(cuda, [(1, 30), (1, 31), (1, 32), (1, 33)], 2, 2, 64, 16, "f16", "float32")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    good = dict(start=[0, 1, 2, 3, 4], len=[30, 31, 32, 33], seq=[0, 1, 2, 3], max_q=1)
    for name, row, value in (("len", 1, -1), ("len", 1, 16 * kv.page_table.shape[1] + 1), ("seq", 1, 4), ("seq", 1, -1)):
        case = {k: list(v) if isinstance(v, list) else v for k, v in good.items()}
        case[name][row] = value
        out = torch.full_like(q, 9.0)
        kv.status.zero_()
        kv.attention(q, i32(case["start"]), i32(case["len"]), seq=i32(case["seq"]), max_q=1, out=out)
        assert int(kv.status) != 0
        # the work is cut elsewhere without the bad entry: each result is within 2e-5 max|v| of the exact one
        assert torch.all(out[1] == 9.0) and float((out[[0, 2, 3]] - clean[[0, 2, 3]]).abs().max()) <= 4e-5 * 5
    for start, left in (([0, 1, 2, 3, 5], 3), ([0, 1, 2, 3, 2], 3), ([-1, 1, 2, 3, 4], 0)):
        out = torch.full_like(q, 9.0)
        kv.status.zero_()
        kv.attention(q, i32(start), i32(good["len"]), max_q=1, out=out)
        assert int(kv.status) != 0
        assert torch.all(out[left] == 9.0) and torch.all(out[1:3] != 9.0)
    # starts that fall again and again: more tiles than tokens, none computed
    kv, q, clean = check(cuda, [(520, 530)] + [(1, 9)] * 9, 2, 4, 64, 16, "f16", "float32")
    out = torch.full_like(q, 9.0)
    kv.status.zero_()
    kv.attention(q, i32([0, 520] * 2048 + [0]), i32([530] * 4096), seq=i32([0] * 4096), out=out)
    assert int(kv.status) != 0 and torch.all(out == 9.0)
    kv, q, clean = check(cuda, [(1, 30), (9, 31)], 1, 2, 64, 16, "f16", "float32")
    out = torch.full_like(q, 9.0)
    kv.status.zero_()
    kv.attention(q, i32([0, 1, 10]), i32([30, 31]), max_q=2, out=out)
    assert int(kv.status) != 0 and torch.all(out[1:] == 9.0) and float((out[:1] - clean[:1]).abs().max()) <= 4e-5 * 5
