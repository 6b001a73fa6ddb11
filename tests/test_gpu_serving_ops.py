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
