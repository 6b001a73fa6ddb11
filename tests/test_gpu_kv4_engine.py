"""Engines whose pool is held in 4 bits, against engines of ijb_create on the same weights.

A 4-bit pool rounds a value by about a sixth of the largest of its 32 at most (half the step between 4 and 6, where 6 is
the largest, give or take a scale's rounding by a sixteenth); logits are held to two sixths, as an e4m3 pool's are to
twice its own largest rounding (test_gpu_paged_engine.py)."""
import numpy as np
import pytest

from ijb200 import synth
from ijb200.engine import Engine

pytestmark = pytest.mark.gpu
CFG128 = synth.ModelConfig("hd128", dim=512, layers=2, heads=4, kv_heads=2, hidden=1024, vocab=4096)
BAR = 2 / 6


def rel_l2(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.mark.parametrize("cfg", [synth.TINY, CFG128], ids=["tiny", "hd128"])
@pytest.mark.parametrize("max_batch", [1, 64])
def test_prefill_decode_and_mixed_steps(cuda, cfg, max_batch):
    weights = synth.make_model(cfg, seed=23)
    kw = dict(context=300, max_batch=max_batch, max_seqs=6, use_dp4a=False, use_q6_dp4a=False)
    a, b = Engine(cfg, weights, kv_type="e2m1", **kw), Engine(cfg, weights, **kw)
    prompt = synth.prompt_tokens(150, seed=2, vocab_limit=cfg.vocab)
    sa, sb = a.seq_open(), b.seq_open()
    a.seq_prefill(sa, prompt)
    nxt = b.seq_prefill(sb, prompt)
    row = (len(prompt) - 1) % max_batch if max_batch > 1 else 0
    assert rel_l2(a.logits(row + 1)[row], b.logits(row + 1)[row]) < BAR
    for _ in range(8):
        a.decode_step([sa], [nxt])
        nxt = int(b.decode_step([sb], [nxt])[0])
        assert rel_l2(a.logits(1), b.logits(1)) < BAR
    if max_batch > 1:
        ta, tb = a.seq_open(), b.seq_open()
        for plan in ([0, 1], [0] * 30 + [1] * 5, [0, 1, 0, 1, 1], [1] * 64):
            tok = np.random.default_rng(len(plan)).integers(0, cfg.vocab, len(plan))
            a.decode_step([(sa, ta)[i] for i in plan], tok)
            b.decode_step([(sb, tb)[i] for i in plan], tok)
            assert rel_l2(a.logits(len(plan)), b.logits(len(plan))) < BAR, plan
    a.close()
    b.close()


def test_generate_matches_steps_and_sampled_steps_run(cuda):
    cfg = synth.TINY
    weights = synth.make_model(cfg, seed=9)
    prompt = synth.prompt_tokens(30, seed=5, vocab_limit=cfg.vocab)
    a, b = (Engine(cfg, weights, context=128, max_batch=16, max_seqs=2, kv_type="e2m1") for _ in range(2))
    sa, sb = a.seq_open(), b.seq_open()
    na, nb = a.seq_prefill(sa, prompt), b.seq_prefill(sb, prompt)
    got, want = a.generate(sa, na, 40), [nb]
    for _ in range(39):
        nb = int(b.decode_step([sb], [nb])[0])
        want.append(nb)
    assert got == want
    tok, prob = b.decode_sample([sb], [nb], [0.3], [0.8])
    assert 0 <= tok[0] < cfg.vocab and 0 < prob[0] <= 1
    a.close()
    b.close()


def test_a_step_reads_what_the_pool_holds(cuda):
    """Bytes that a layer's attention reads: 17 of 32 values' (16 of codes, one of scale)."""
    cfg = synth.TINY
    e = Engine(cfg, synth.make_model(cfg, seed=9), context=128, max_batch=16, max_seqs=2, kv_type="e2m1")
    s = e.seq_open()
    e.seq_prefill(s, synth.prompt_tokens(30, seed=5, vocab_limit=cfg.vocab))
    assert e.time_layer_attention([s], reps=2)[1] == 30 * cfg.kv_heads * 2 * (cfg.head_dim // 2 + cfg.head_dim // 32)
    e.close()
