"""ijb_sample on a B200 against its definition in 64 bits.

The plain implementation below takes the operator's own fp32 weights exp((x - max) / T)
(torch's fp32 exp, which is CUDA's), turns them into whole multiples of 2^-44 and does
everything else in 64-bit integers, so tokens must be equal and the probability is one
rounding of a quotient: off by at most 2^-23 relative (the fp64 quotient, then fp32)."""
import numpy as np
import pytest

from ijb200 import lib

pytestmark = pytest.mark.gpu
FIXED = 1 << 44


def plain(logits, u, temperature, top_k, top_p, min_p):
    import torch
    tokens, probs = [], []
    n, vocab = logits.shape
    for i in range(n):
        x = torch.where(logits[i].isnan(), -float("inf"), logits[i])
        top = x.max()
        if top == -float("inf"):
            tokens.append(-1)
            probs.append(0.0)
            continue
        if not temperature[i] > 0:
            best = torch.nonzero(x == top).flatten().tolist()
            # equal maxima: the framework's argmax order (block, then place, bit-reversed)
            tokens.append(min(best, key=lambda j: (int(f"{j >> 8:09b}"[::-1], 2), int(f"{j & 255:08b}"[::-1], 2))))
            probs.append(1.0)
            continue
        t = torch.tensor(float(temperature[i]), dtype=torch.float32, device=x.device)
        w = torch.exp(torch.where(x == top, torch.zeros_like(x), (x - top) / t))
        fixed = torch.where(w > 0, torch.round(w.double() * FIXED), 0.0).long().cpu().numpy().astype(object)
        xs, ws = x.cpu().numpy(), w.cpu().numpy()
        order = np.lexsort((np.arange(vocab), -xs.astype(np.float64)))
        mass = np.cumsum(fixed[order])
        kept = int(mass[-1])
        k = int(top_k[i])
        if 0 < k < vocab:
            kept = int(mass[k - 1])
        p = float(np.float32(top_p[i]))
        if p < 1:
            want = max(1, min(kept, int(np.ceil(p * float(kept)))))
            kept = int(next(m for m in mass if m >= want))
        keep = (ws >= np.float32(min_p[i])) | (xs == xs.max())
        kept = min(kept, int(fixed[keep].sum()))
        target = max(0, min(kept - 1, int(np.floor(float(np.float32(u[i])) * float(kept)))))
        at = int(next(j for j in range(vocab) if mass[j] > target))
        tokens.append(int(order[at]))
        probs.append(float(fixed[order[at]]) / float(kept))
    return np.array(tokens), np.array(probs)


def run(logits, u, temperature, top_k, top_p, min_p):
    import torch
    from ijb200 import ops
    dev = logits.device
    f = lambda v, t: torch.tensor(v, dtype=t, device=dev)  # noqa: E731
    token, prob = ops.sample(logits, f(u, torch.float32), f(temperature, torch.float32), f(top_k, torch.int32),
                             f(top_p, torch.float32), f(min_p, torch.float32))
    return token.cpu().numpy(), prob.cpu().numpy()


def check(logits, u, temperature, top_k, top_p, min_p):
    want_t, want_p = plain(logits, u, temperature, top_k, top_p, min_p)
    got_t, got_p = run(logits, u, temperature, top_k, top_p, min_p)
    np.testing.assert_array_equal(got_t, want_t)
    np.testing.assert_allclose(got_p, want_p, rtol=2.0 ** -23, atol=0)


def settings(rng, n):
    return ([float(v) for v in rng.random(n)], [float(v) for v in rng.choice([0.0, 0.3, 0.7, 1.0, 2.0], n)],
            [int(v) for v in rng.choice([0, -3, 1, 2, 40, 700, 1500, 10 ** 6], n)],
            [float(v) for v in rng.choice([0.0, 0.1, 0.5, 0.9, 0.999, 1.0, 1.5], n)],
            [float(v) for v in rng.choice([0.0, 0.0, 0.02, 0.3, 1.0], n)])


@pytest.mark.parametrize("vocab,n,spread", [(1, 3, 1.0), (2, 8, 1.0), (31, 9, 2.0), (1000, 12, 3.0), (2049, 8, 0.2),
                                            (4999, 8, 1.0), (16385, 6, 6.0), (50257, 5, 2.5), (128256, 8, 2.5),
                                            (131072, 3, 0.5), (128255, 3, 30.0)])
def test_sample_matches_definition(cuda, vocab, n, spread):
    import torch
    rng = np.random.default_rng(vocab + n)
    g = torch.Generator(device=cuda)
    g.manual_seed(vocab)
    check(torch.randn((n, vocab), generator=g, device=cuda) * spread, *settings(rng, n))


def test_sample_equal_logits(cuda):
    """Long runs of equal values: more than the sorted list holds, all in one bin, all one value."""
    import torch
    rng = np.random.default_rng(1)
    n = 10
    for vocab, levels in ((128256, 1), (128256, 3), (9000, 40), (6000, 2)):
        x = torch.from_numpy(rng.integers(0, levels, (n, vocab)).astype(np.float32) * 1e-3).to(cuda)
        check(x, *settings(rng, n))
    # close but not equal: one bin, split by the low bits of the logits
    x = torch.from_numpy((8.0 + rng.integers(0, 5000, (n, 60000)) * 2.0 ** -20).astype(np.float32)).to(cuda)
    check(x, *settings(rng, n))


def test_sample_infinities_and_nan(cuda):
    import torch
    inf, nan = float("inf"), float("nan")
    x = torch.randn((8, 3000), device=cuda)
    x[0, ::2] = -inf
    x[1, :] = -inf
    x[2, :] = nan
    x[3, 5:2900] = nan
    x[4, 77] = inf
    x[5, [9, 2000]] = inf
    x[6, 1:] = -inf
    x[7, :] = torch.finfo(torch.float32).min
    n = 8
    for t in (0.0, 0.8):
        check(x, [0.9] * n, [t] * n, [0] * n, [1.0] * n, [0.0] * n)
        check(x, [0.4] * n, [t] * n, [50] * n, [0.9] * n, [0.1] * n)


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0, 5.0, -1.0, float("nan")])
def test_sample_ends_of_the_uniform_range(cuda, u):
    """u = 0 takes the largest; u just below 1 (and beyond, and below 0) stays inside the kept tokens."""
    import torch
    x = torch.randn((3, 777), device=cuda)
    got, _ = run(x, [u] * 3, [1.0] * 3, [5] * 3, [1.0] * 3, [0.0] * 3)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1].cpu().numpy()
    for i in range(3):
        if u >= 1.0 - 2.0 ** -24:
            assert got[i] == order[i, 4]
        else:
            assert got[i] == order[i, 0]


def test_sample_strides_defaults_and_greedy(cuda):
    """A row stride, NULL settings, and temperature 0 against ijb_argmax."""
    import torch
    from ijb200 import ops
    big = torch.randn((6, 5003), device=cuda)
    view = big[:, 1:4098]
    u = torch.rand((6,), device=cuda)
    a, pa = ops.sample(view, u)
    b, pb = ops.sample(view.contiguous(), u)
    assert torch.equal(a, b) and torch.equal(pa, pb)
    zero = torch.zeros((6,), device=cuda)
    view[2, [300, 512, 7]] = 50.0
    token, prob = ops.sample(view, u, temperature=zero)
    L = lib.load()
    for i in range(6):
        idx = torch.zeros(1, dtype=torch.int32, device=cuda)
        row = view[i].contiguous()
        lib.check(L.ijb_argmax(row.data_ptr(), row.numel(), idx.data_ptr(), None))
        torch.cuda.synchronize()
        assert int(token[i]) == int(idx)
    assert torch.all(prob == 1)


def test_sample_same_row_in_any_batch_stream_and_graph(cuda):
    import torch
    from ijb200 import ops
    n, vocab = 70, 32003
    x = torch.randn((n, vocab), device=cuda) * 3
    u = torch.rand((n,), device=cuda)
    t = torch.full((n,), 0.8, device=cuda)
    p = torch.full((n,), 0.9, device=cuda)
    all_t, all_p = ops.sample(x, u, t, None, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one_t, one_p = ops.sample(x[33:34], u[33:34], t[33:34], None, p[33:34])
    torch.cuda.synchronize()
    assert int(one_t) == int(all_t[33]) and float(one_p) == float(all_p[33])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g_t, g_p = ops.sample(x, u, t, None, p)
    x.copy_(torch.randn((n, vocab), device=cuda) * 3)
    graph.replay()
    torch.cuda.synchronize()
    want_t, want_p = ops.sample(x, u, t, None, p)
    assert torch.equal(g_t, want_t) and torch.equal(g_p, want_p)


def test_quotient_is_rounded_to_nearest(cuda):
    """The operator forms (x - m) / T from 1 / T and one residual correction; a division gives the same.  For
    quotients t in [-15, -8] a wrong last bit is 2^-20 and moves exp(t) by 2^-20 of itself; expf is good to two
    units in the last place, 2^-22, and min_p's own rounding is 2^-24.  So with min_p at exp(t) (1 -+ 2^-21) the
    token of weight exp(t) is kept and dropped."""
    import torch
    from ijb200 import ops
    n = 1 << 16
    rng = np.random.default_rng(5)
    T = np.exp(rng.uniform(np.log(1e-3), np.log(1e3), n)).astype(np.float32)
    d = (rng.uniform(8.01, 15.0, n) * T).astype(np.float32)
    dT, dd = torch.from_numpy(T).to(cuda), torch.from_numpy(-d).to(cuda)
    t = (dd / dT).double()  # CUDA's division, in fp32
    x = torch.zeros((n, 2), dtype=torch.float32, device=cuda)
    x[:, 1] = dd
    u = torch.full((n,), 1 - 2.0 ** -24, dtype=torch.float32, device=cuda)  # the last token kept
    for sign in (-1, 1):
        token, _ = ops.sample(x, u, dT, None, None, (torch.exp(t) * (1 + sign * 2.0 ** -21)).float())
        assert int((token != (0 if sign > 0 else 1)).sum()) == 0


def test_sample_cuts_one_after_another(cuda):
    """A short top-k list serves the cuts behind it as it stands in shared memory: each has to be read by all threads
    before the next one is written, which only a barrier there gives (repeated runs show its absence rarely).  The
    same batch many times beside other work, each run against the definition."""
    import torch
    from ijb200 import ops
    n, vocab = 48, 9001
    g = torch.Generator(device=cuda)
    g.manual_seed(12)
    x = torch.randn((n, vocab), generator=g, device=cuda) * 2.5
    u = torch.rand((n,), generator=g, device=cuda)
    t, p, m = torch.full((n,), 0.7, device=cuda), torch.full((n,), 0.95, device=cuda), torch.zeros((n,), device=cuda)
    k = torch.tensor([40, 1, 2, 64, 100, 120], dtype=torch.int32, device=cuda).repeat(8)
    p[1::2] = torch.linspace(0.05, 0.999, n // 2, device=cuda)
    m[::3] = 0.02
    want_t, want_p = plain(x, u.tolist(), t.tolist(), k.tolist(), p.tolist(), m.tolist())
    a = torch.randn((2048, 2048), device=cuda)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(60):
            a = torch.tanh(a @ a)
    tokens, probs = zip(*[ops.sample(x, u, t, k, p, m) for _ in range(400)])
    torch.cuda.synchronize()
    for token, prob in zip(tokens, probs):
        np.testing.assert_array_equal(token.cpu().numpy(), want_t)
        np.testing.assert_allclose(prob.cpu().numpy(), want_p, rtol=2.0 ** -23, atol=0)
