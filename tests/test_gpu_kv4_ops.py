"""The operators around a 4-bit cache together, as a program without an engine uses them: prompts written and attended
to, sequences forked by copying the page they end in, steps of write -> attention -> sample captured into a graph and
replayed, against the same in 64 bits over the values that the cache holds; calls on several streams; a pool past
2^32 bytes."""
import numpy as np
import pytest

from test_gpu_kv4 import decode

pytestmark = pytest.mark.gpu


def cache(cuda, pages, kvh, page, hd, table, fill=0):
    import torch
    from ijb200 import ops
    data = torch.full((pages, 2, kvh, page, hd // 2), fill, dtype=torch.uint8, device=cuda).view(torch.float4_e2m1fn_x2)
    scale = torch.full((pages, 2, kvh, page, hd // 32), 200, dtype=torch.uint8, device=cuda)
    return ops.PagedKV(data, table, scale, torch.zeros((1,), dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_forks_and_captured_steps(cuda, hd):
    import torch
    from ijb200 import ops
    g = torch.Generator(device=cuda)
    g.manual_seed(7)
    kvh, heads, page, width, vocab = 2, 8, 16, 8, 1000
    lens = [1, 5, 16, 17, 31, 48, 64, 77, 90]
    seqs = 2 * len(lens)  # every prompt, and a fork of it
    rand = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.randperm(seqs * width, generator=g, device=cuda).view(seqs, width).int().contiguous()
    kv = cache(cuda, seqs * width, kvh, page, hd, table)
    head = rand(heads * hd, vocab) * 0.1
    start = np.cumsum([0] + lens)
    seq = i32([s for s, n in enumerate(lens) for _ in range(n)])
    pos = i32([p for n in lens for p in range(n)])
    k, v, q = rand(int(start[-1]), kvh, hd), rand(int(start[-1]), kvh, hd), rand(int(start[-1]), heads, hd)
    kv.append(k, v, seq, pos)
    prompt = kv.attention(q, i32(start.tolist()), i32(lens), max_q=max(lens))
    # forks: full pages by name, the last one copied
    own = table.clone()
    src, dst = [], []
    for i, n in enumerate(lens):
        full = n // page
        table[len(lens) + i, :full] = own[i, :full]
        if n % page:
            src.append(int(own[i, full]))
            dst.append(int(own[len(lens) + i, full]))
    kv.copy_pages(i32(src), i32(dst))
    again = kv.attention(q, i32(start.tolist()), i32(lens), seq=i32(list(range(len(lens), seqs))), max_q=max(lens))
    assert torch.equal(prompt, again)  # the same rows, cut the same way

    def attend64(e, n, x):  # one token over n positions, from what the cache holds
        kk, vv = kv.gather(i32([e] * n), i32(list(range(n))))
        s = torch.einsum("hgd,thd->hgt", x.double().view(kvh, -1, hd), kk.double()) * hd ** -0.5
        return torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), vv.double()).reshape(-1)

    both = lens + lens
    st = dict(k=rand(seqs, kvh, hd), v=rand(seqs, kvh, hd), q=rand(seqs, heads, hd), pos=i32(both),
              len=i32([n + 1 for n in both]), u=torch.rand((seqs,), generator=g, device=cuda))
    every, ones = i32(list(range(seqs))), i32(list(range(seqs + 1)))
    t, p = torch.full((seqs,), 0.8, device=cuda), torch.full((seqs,), 0.9, device=cuda)

    def step():
        kv.append(st["k"], st["v"], every, st["pos"])
        o = kv.attention(st["q"], ones, st["len"], max_q=1)
        logits = o.view(seqs, -1) @ head
        return o, logits, ops.sample(logits, st["u"], t, None, p)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, logits, (token, prob) = step()
    for n in range(4):
        for name in "kvq":
            st[name].copy_(rand(*st[name].shape))
        st["u"].copy_(torch.rand((seqs,), generator=g, device=cuda))
        st["pos"].copy_(i32([x + n for x in both]))
        st["len"].copy_(i32([x + n + 1 for x in both]))
        graph.replay()
        torch.cuda.synchronize()
        for e in range(seqs):
            want = attend64(e, both[e] + n + 1, st["q"][e])
            # fp32 queries: 2e-5 of the largest value (test_gpu_kv4.py); |v| < 6 here
            assert float((o[e].reshape(-1).double() - want).abs().max()) <= 2e-5 * 6.0
        one, one_p = ops.sample(logits, st["u"], t, None, p)
        assert torch.equal(token, one) and torch.equal(prob, one_p)
    assert int(kv.status) == 0


def test_calls_on_several_streams_at_once(cuda):
    """Single tokens of few rows and of many, a prompt, a write and read-back elsewhere, and copies elsewhere, each on its
    own stream, give what each gives alone, bit for bit."""
    import torch
    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    kvh, heads, hd, page, seqs, width = 2, 8, 128, 16, 8, 64
    rand = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    table = torch.randperm(seqs * width, generator=g, device=cuda).view(seqs, width).int()
    kv, other, third = (cache(cuda, seqs * width, kvh, page, hd, table) for _ in range(3))
    for e in range(seqs):
        x = rand(2, 1024, kvh, hd)
        kv.append(x[0], x[1], i32([e] * 1024), i32(list(range(1024))))
    lens = i32([1, 1000, 17, 512, 1024, 3, 700, 900])
    one, ones = rand(seqs, heads, hd), i32(list(range(seqs + 1)))
    four, fours = rand(4 * seqs, heads, hd), i32(list(range(0, 4 * seqs + 1, 4)))
    prompt, p_start, p_len = rand(800, heads, hd).half(), i32([0, 500, 800]), i32([900, 300])
    rows, r_pos, r_seq = rand(1024, kvh, hd), i32(list(range(1024))), i32([2] * 1024)
    src, dst = i32(list(range(200))), i32(list(range(200, 400)))

    def write():
        other.append(rows, rows, r_seq, r_pos)
        return other.gather(r_seq, r_pos)[0]

    def copy():
        kv.copy_pages(src, dst, to=third)
        return torch.cat([third.data.view(torch.uint8)[200:400].flatten(), third.scale[200:400].flatten()])

    calls = [lambda: kv.attention(one, ones, lens, max_q=1), lambda: kv.attention(four, fours, lens, max_q=4),
             lambda: kv.attention(one.half(), ones, lens, max_q=1), lambda: kv.attention(prompt, p_start, p_len), write, copy]
    alone = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(10):
        for f, s, out in zip(calls, streams, got):
            with torch.cuda.stream(s):
                out.append(f())
    torch.cuda.synchronize()
    for want, outs in zip(alone, got):
        for x in outs:
            assert torch.equal(x, want)


@pytest.mark.parametrize("hd", [64, 128])
def test_a_pool_past_4_gigabytes(cuda, hd):
    """Pages at both ends of a pool of more than 2^32 bytes: written, read, copied and attended to alike."""
    import torch
    kvh, page, tokens = 8, 32, 100
    pages = (1 << 32) // (2 * kvh * page * hd // 2) + 1000
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    table = i32([[0, 1, 2, 3], [pages - 4, pages - 3, pages - 2, pages - 1], [pages - 10, 17, pages - 12, 19]])
    kv = cache(cuda, pages, kvh, page, hd, table)
    assert kv.data.view(torch.uint8).numel() > 1 << 32
    x = torch.randn((2, tokens, kvh, hd), device=cuda)
    for e in (0, 1):
        kv.append(x[0], x[1], i32([e] * tokens), i32(list(range(tokens))))
    kv.copy_pages(table[1].clone(), table[2].clone())
    read = [kv.gather(i32([e] * tokens), i32(list(range(tokens)))) for e in range(3)]
    for k, v in read[1:]:
        assert torch.equal(k, read[0][0]) and torch.equal(v, read[0][1])
    last = table[1].long()
    assert torch.equal(decode(kv.data.view(torch.uint8)[last, 0], kv.scale[last, 0]).permute(0, 2, 1, 3).reshape(-1, kvh, hd)[:tokens],
                       read[0][0].double())
    for n, dtype in ((1, torch.float32), (1, torch.float16), (70, torch.float16)):
        q = torch.randn((n, 4 * kvh, hd), device=cuda).to(dtype)
        out = [kv.attention(q, i32([0, n]), i32([tokens]), seq=i32([e]), max_q=n) for e in range(3)]
        assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])
    assert int(kv.status) == 0


def test_refusals_of_tensors(cuda):
    import torch
    from ijb200 import ops
    table = torch.zeros((1, 2), dtype=torch.int32, device=cuda)
    data = torch.zeros((2, 2, 1, 16, 32), dtype=torch.uint8, device=cuda)
    scale = torch.zeros((2, 2, 1, 16, 2), dtype=torch.uint8, device=cuda)
    packed = data.view(torch.float4_e2m1fn_x2)
    ops.PagedKV(packed, table, scale)
    for bad in ((data, table, scale), (packed, table, None), (packed, table, scale[..., :1]), (packed, table, scale[..., 0]),
                (packed, table, scale.int()), (packed, table, scale.cpu()), (packed[:, :, :, ::2], table, scale[:, :, :, ::2])):
        with pytest.raises(ValueError):
            ops.PagedKV(*bad)
    from ijb200.lib import IjbError
    odd = torch.zeros((129,), dtype=torch.uint8, device=cuda)[1:].view(scale.shape)
    kv = ops.PagedKV(packed, table, odd)
    k = torch.zeros((1, 1, 64), device=cuda)
    z = torch.zeros((1,), dtype=torch.int32, device=cuda)
    kv.append(k, k, z, z)  # any alignment will do for rows
    kv.gather(z, z)
    with pytest.raises(IjbError, match="16-byte"):
        kv.attention(torch.zeros((1, 1, 64), device=cuda), torch.tensor([0, 1], dtype=torch.int32, device=cuda), z + 1, max_q=1)
    with pytest.raises(ValueError):
        kv.append(k.double(), k.double(), z, z)
