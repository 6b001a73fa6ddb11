"""Each layer of an engine with a 4-bit pool against the layer in 64 bits, with K and V as the pool's definition holds them
(test_gpu_kv4.py).  A layer starts from the engine's own residuals behind the one before, so roundings do not build up.

What a layer adds to the residuals is held to 2e-2 (rel-L2 over all tokens).  The engine's fp32 projections and attention
are 1e-5 and less of it.  What is more are K/V values that fp32 puts on the other side of a border between two codes:
one in 10^5 or so, about one of a layer's 40,000.  That moves a stored value by a third of the largest of its 32 (about 2 to
3) at most, in the 4 heads that read it: four of them, each seen with a weight of 1, come to 4 * 1.2 of a norm of
sqrt(150 * 512) = 277 of attention outputs near 1, 1.7e-2.  K or V with another layer's, head's or block's scales are off by
a third and more."""
import numpy as np
import pytest

import oracle as O
from ijb200 import synth
from test_gpu_kv4 import LEVELS, quantise, scale_table

CFG128 = synth.ModelConfig("hd128", dim=512, layers=3, heads=4, kv_heads=1, hidden=1024, vocab=2048)
CFG64 = synth.ModelConfig("hd64", dim=512, layers=3, heads=8, kv_heads=2, hidden=768, vocab=2048)
N = 150


def held(x):
    """The values that a 4-bit pool holds for rows x."""
    codes, byte = quantise(x)
    c = np.stack([codes & 15, codes >> 4], -1).reshape(x.shape)
    return np.concatenate([LEVELS, -LEVELS])[c] * np.repeat(scale_table()[byte], 32, -1)


def layer(cfg, w, l, x, cache):
    """The residuals behind layer l of one sequence's x [n][dim], in 64 bits; K and V rows enter as cache(rows)."""
    n, hd, g = len(x), cfg.head_dim, cfg.heads // cfg.kv_heads

    def mat(name, y):
        full = f"blk.{l}.{name}.weight"
        t = next(t for m, t, _, _ in cfg.matrices() if m == full)
        return y @ O.dequant(t, w[full]).astype(np.float64).reshape(len(w[full]), -1).T

    def norm(name, y):
        return y / np.sqrt((y * y).mean(-1, keepdims=True) + cfg.eps) * w[f"blk.{l}.{name}.weight"]
    cos, sin = (t.astype(np.float64)[:n, None] for t in O.rope_tables(n, hd, cfg.rope_base))

    def rope(y):
        a, b = y[..., 0::2], y[..., 1::2]
        return np.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(y.shape)
    h = norm("attn_norm", x)
    q = rope(mat("attn_q", h).reshape(n, cfg.heads, hd))
    k = cache(rope(mat("attn_k", h).reshape(n, cfg.kv_heads, hd)))
    v = cache(mat("attn_v", h).reshape(n, cfg.kv_heads, hd))
    s = np.einsum("qhd,khd->hqk", q, np.repeat(k, g, 1)) / np.sqrt(hd)
    s = np.where(np.tril(np.ones((n, n), bool)), s, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    x = x + mat("attn_output", np.einsum("hqk,khd->qhd", p, np.repeat(v, g, 1)).reshape(n, -1))
    h = norm("ffn_norm", x)
    gate = mat("ffn_gate", h)
    return x + mat("ffn_down", gate / (1 + np.exp(-gate)) * mat("ffn_up", h))


def embedding(cfg, w, tokens):
    return O.dequant(synth.Q6_K, w["token_embd.weight"][tokens]).astype(np.float64).reshape(len(tokens), -1)


def off(cfg, w, tokens, trace, cache):
    """rel-L2 of what each layer adds, trace [n][layers][dim] being the residuals behind them."""
    x, out = embedding(cfg, w, tokens), []
    for l in range(cfg.layers):
        add = layer(cfg, w, l, x, cache) - x
        out.append(float(np.linalg.norm(trace[:, l] - x - add) / np.linalg.norm(add)))
        x = trace[:, l].astype(np.float64)
    return out


@pytest.mark.parametrize("cfg", [CFG64, CFG128], ids=["hd64", "hd128"])
def test_the_layers_of_this_file_are_the_oracle_s(cfg):
    w = synth.make_model(cfg, seed=5)
    tokens = synth.prompt_tokens(20, seed=2, vocab_limit=cfg.vocab)
    state = O.OracleModel(cfg, w, 64, use_dp4a=False, use_q6_dp4a=False).new_state()
    trace = np.array([state.forward(int(t), i, False, trace=True)[1] for i, t in enumerate(tokens)])
    assert max(off(cfg, w, tokens, trace, lambda x: x)) < 1e-5
    assert min(off(cfg, w, tokens, trace, held)) > 2e-2  # and that the bound tells a 4-bit cache from others


@pytest.mark.gpu
@pytest.mark.parametrize("max_batch", [1, 4, 8])
@pytest.mark.parametrize("cfg", [CFG64, CFG128], ids=["hd64", "hd128"])
def test_layers_over_a_4_bit_pool(cuda, cfg, max_batch):
    """Single tokens, runs of 4 (16 rows) and of 8 (the tile kernel), projections on the CUDA cores."""
    from ijb200.engine import Engine
    w = synth.make_model(cfg, seed=5)
    tokens = synth.prompt_tokens(N, seed=2, vocab_limit=cfg.vocab)
    e = Engine(cfg, w, kv_type="e2m1", context=N + 8, max_batch=max_batch, max_seqs=2, use_dp4a=False, use_q6_dp4a=False)
    trace = e.prefill_traced(tokens)[1]
    assert max(off(cfg, w, tokens, trace, held)) < 2e-2
    e.close()
