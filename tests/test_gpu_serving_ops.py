"""The serving operators together, as a program without an engine uses them: several
steps of write -> attention -> projection -> sample over one e4m3 cache, captured into a
graph and replayed, against the same steps in 64 bits over the values the cache holds."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
def test_steps_of_write_attend_sample(cuda, hd):
    import torch
    from ijb200 import ops
    g = torch.Generator(device=cuda)
    g.manual_seed(7)
    kvh, heads, page, seqs, width, vocab = 2, 8, 16, 9, 6, 1000
    rand = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    data = torch.zeros((seqs * width, 2, kvh, page, hd), dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    scale = torch.full((seqs * width, 2, kvh, page), 200, dtype=torch.uint8, device=cuda)
    table = torch.randperm(seqs * width, generator=g, device=cuda).view(seqs, width).int()
    status = torch.zeros((1,), dtype=torch.int32, device=cuda)
    kv = ops.PagedKV(data, table, scale, status)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    head = rand(heads * hd, vocab) * 0.1
    # a prompt for every sequence, of 1..90 tokens, in one ragged call
    lens = [1, 5, 16, 17, 31, 48, 64, 77, 90]
    start = np.cumsum([0] + lens)
    seq = i32([s for s, n in enumerate(lens) for _ in range(n)])
    pos = i32([p for n in lens for p in range(n)])
    k, v, q = rand(int(start[-1]), kvh, hd), rand(int(start[-1]), kvh, hd), rand(int(start[-1]), heads, hd)
    kv.append(k, v, seq, pos)
    kv.attention(q, i32(start.tolist()), i32(lens), max_q=max(lens))

    def attend64(e, n, x):  # one token over n positions, from what the cache holds
        kk, vv = kv.gather(i32([e] * n), i32(list(range(n))))
        s = torch.einsum("hgd,thd->hgt", x.double().view(kvh, -1, hd), kk.double()) * hd ** -0.5
        return torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), vv.double()).reshape(-1)

    st = dict(k=rand(seqs, kvh, hd), v=rand(seqs, kvh, hd), q=rand(seqs, heads, hd), pos=i32(lens),
              len=i32([n + 1 for n in lens]), u=torch.rand((seqs,), generator=g, device=cuda))
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
        st["pos"].copy_(i32([x + n for x in lens]))
        st["len"].copy_(i32([x + n + 1 for x in lens]))
        graph.replay()
        torch.cuda.synchronize()
        for e in range(seqs):
            want = attend64(e, lens[e] + n + 1, st["q"][e])
            # fp32 queries: 2e-5 of the largest value (see test_gpu_paged_attention.py)
            assert float((o[e].reshape(-1).double() - want).abs().max()) <= 2e-5 * 5.0
        again, again_p = ops.sample(logits, st["u"], t, None, p)
        assert torch.equal(token, again) and torch.equal(prob, again_p)
    assert int(status) == 0


def test_calls_on_several_streams_at_once(cuda):
    """A ragged call of single tokens, a prompt's attention, a write elsewhere and sampling, each on its own stream,
    give what each gives alone, bit for bit."""
    import torch
    from ijb200 import ops
    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    kvh, heads, hd, page, seqs, width = 2, 8, 128, 16, 8, 64
    rand = lambda *s: torch.randn(s, generator=g, device=cuda)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    data = rand(seqs * width, 2, kvh, page, hd).half()
    table = torch.randperm(seqs * width, generator=g, device=cuda).view(seqs, width).int()
    kv = ops.PagedKV(data, table)
    other = ops.PagedKV(torch.zeros_like(data), table)
    one, lens = rand(seqs, heads, hd), i32([1, 1000, 17, 512, 1024, 3, 700, 900])
    ones = i32(list(range(seqs + 1)))
    prompt, p_start, p_len = rand(800, heads, hd).half(), i32([0, 500, 800]), i32([900, 300])
    rows, r_pos, r_seq = rand(1024, kvh, hd), i32(list(range(1024))), i32([2] * 1024)
    logits, u = rand(40, 50000) * 3, torch.rand((40,), generator=g, device=cuda)
    k40, p90 = torch.full((40,), 40, dtype=torch.int32, device=cuda), torch.full((40,), 0.9, device=cuda)

    def write():
        other.append(rows, rows, r_seq, r_pos)
        return other.gather(r_seq, r_pos)[0]

    calls = [lambda: kv.attention(one, ones, lens, max_q=1), lambda: kv.attention(prompt, p_start, p_len), write,
             lambda: ops.sample(logits, u, None, k40, p90)[0]]
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
