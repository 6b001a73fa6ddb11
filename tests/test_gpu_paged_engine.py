"""Engines made by ijb_create_kv (paged attention operators, fp16 or e4m3 pool) and
ijb_decode_sample, against engines of ijb_create on the same weights.

With an fp16 pool both engines cache the same rows and attend over them to fp32 accuracy,
so on the FP32 activation path logits agree to the project's bar for two summation orders
(rel-L2 1e-2; about 1e-3 is seen between paths).  An e4m3 pool rounds every cached value by up to 2^-4 of
itself (1.8 % rms): logits are held to 2 * 2^-4."""
import ctypes

import numpy as np
import pytest

from ijb200 import lib, synth
from ijb200.engine import Engine

pytestmark = pytest.mark.gpu
CFG128 = synth.ModelConfig("hd128", dim=512, layers=2, heads=4, kv_heads=2, hidden=1024, vocab=4096)


def rel_l2(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


@pytest.fixture(scope="module", params=["tiny", "hd128"])
def model(request):
    cfg = synth.TINY if request.param == "tiny" else CFG128
    return cfg, synth.make_model(cfg, seed=23)


BAR = {"f16": 1e-2, "e4m3": 2 * 2.0 ** -4}


@pytest.mark.parametrize("kv_type", ["f16", "e4m3"])
@pytest.mark.parametrize("max_batch", [1, 64])
def test_prefill_and_decode(cuda, model, kv_type, max_batch):
    cfg, weights = model
    kw = dict(context=300, max_batch=max_batch, max_seqs=4, use_dp4a=False, use_q6_dp4a=False)
    a, b = Engine(cfg, weights, kv_type=kv_type, **kw), Engine(cfg, weights, **kw)
    prompt = synth.prompt_tokens(150, seed=2, vocab_limit=cfg.vocab)
    sa, sb = a.seq_open(), b.seq_open()
    a.seq_prefill(sa, prompt)
    nxt = b.seq_prefill(sb, prompt)
    row = (len(prompt) - 1) % max_batch if max_batch > 1 else 0
    assert rel_l2(a.logits(row + 1)[row], b.logits(row + 1)[row]) < BAR[kv_type]
    for _ in range(8):
        a.decode_step([sa], [nxt])
        nxt = int(b.decode_step([sb], [nxt])[0])
        assert rel_l2(a.logits(1), b.logits(1)) < BAR[kv_type]
    # sequence 0, the single-sequence runner
    a.prefill(prompt[:40])
    b.prefill(prompt[:40])
    a.forward(int(prompt[40]), 40)
    b.forward(int(prompt[40]), 40)
    assert rel_l2(a.logits(1), b.logits(1)) < BAR[kv_type]
    na, la, qa = a.forward_traced(int(prompt[41]), 41)
    nb, lb, qb = b.forward_traced(int(prompt[41]), 41)
    assert rel_l2(la, lb) < BAR[kv_type]
    a.close()
    b.close()


@pytest.mark.parametrize("kv_type", ["f16", "e4m3"])
def test_ragged_and_mixed_steps(cuda, model, kv_type):
    """Single tokens of many sequences, several tokens of some of them, a sequence named twice."""
    cfg, weights = model
    kw = dict(context=200, max_batch=64, max_seqs=21, use_dp4a=False, use_q6_dp4a=False)
    a, b = Engine(cfg, weights, kv_type=kv_type, **kw), Engine(cfg, weights, **kw)
    rng = np.random.default_rng(4)
    seqs = [(a.seq_open(), b.seq_open()) for _ in range(20)]
    for i, (sa, sb) in enumerate(seqs):
        p = synth.prompt_tokens(int(rng.integers(1, 100)), seed=i, vocab_limit=cfg.vocab)
        a.seq_prefill(sa, p)
        b.seq_prefill(sb, p)
    for plan in (list(range(20)), list(range(20)) + [3, 3], [0] * 30 + [1, 2] + [5] * 7, [7, 8, 7, 8, 8], [2] * 64, [4, 4, 4]):
        tok = rng.integers(0, cfg.vocab, len(plan))
        a.decode_step([seqs[i][0] for i in plan], tok)
        b.decode_step([seqs[i][1] for i in plan], tok)
        assert rel_l2(a.logits(len(plan)), b.logits(len(plan))) < BAR[kv_type], plan
    a.close()
    b.close()


@pytest.mark.parametrize("kv_type", ["f16", "e4m3"])
def test_generate_matches_steps(cuda, kv_type):
    """The device-side loop and single steps run the same launches: equal bits."""
    cfg = synth.TINY
    weights = synth.make_model(cfg, seed=9)
    prompt = synth.prompt_tokens(30, seed=5, vocab_limit=cfg.vocab)
    a, b = (Engine(cfg, weights, context=128, max_batch=16, max_seqs=2, kv_type=kv_type) for _ in range(2))
    sa, sb = a.seq_open(), b.seq_open()
    first = a.seq_prefill(sa, prompt)
    assert first == b.seq_prefill(sb, prompt)
    got = a.generate(sa, first, 40)
    want = [first]
    for _ in range(39):
        want.append(int(b.decode_step([sb], [want[-1]])[0]))
    assert got == want
    a.decode_step([sa], [got[-1]])
    b.decode_step([sb], [want[-1]])
    np.testing.assert_array_equal(a.logits(1).view(np.uint32), b.logits(1).view(np.uint32))
    a.close()
    b.close()


@pytest.mark.parametrize("kv_type", [None, "e4m3"])
def test_decode_sample(cuda, kv_type):
    """Greedy rows are decode_step's tokens; the others are ops.sample's on the step's logits."""
    import torch
    from ijb200 import ops
    cfg = synth.TINY
    weights = synth.make_model(cfg, seed=10)
    kw = dict(context=96, max_batch=16, max_seqs=8, kv_type=kv_type)
    a, b = Engine(cfg, weights, **kw), Engine(cfg, weights, **kw)
    rng = np.random.default_rng(1)
    sa, sb = [a.seq_open() for _ in range(6)], [b.seq_open() for _ in range(6)]
    for i in range(6):
        p = synth.prompt_tokens(5 + 7 * i, seed=i, vocab_limit=cfg.vocab)
        a.seq_prefill(sa[i], p)
        b.seq_prefill(sb[i], p)
    tok = rng.integers(0, cfg.vocab, 6)
    got, prob = a.decode_sample(sa, tok, np.zeros(6), temperature=np.zeros(6))
    np.testing.assert_array_equal(got, b.decode_step(sb, tok))
    assert np.all(prob == 1)
    u = rng.random(6).astype(np.float32)
    t, k = np.array([0, .7, 1, 1, 2, .5], np.float32), np.array([0, 40, 0, 3, 0, 1], np.int32)
    p, mp = np.array([1, .9, 1, 1, .5, 1], np.float32), np.array([0, 0, .1, 0, 0, 0], np.float32)
    got, prob = a.decode_sample(sa, tok, u, t, k, p, mp)
    d = lambda v: torch.from_numpy(v).to(cuda)  # noqa: E731
    want, want_p = ops.sample(d(a.logits(6)), d(u), d(t), d(k), d(p), d(mp))
    np.testing.assert_array_equal(got, want.cpu().numpy())
    np.testing.assert_array_equal(prob, want_p.cpu().numpy())
    assert [a.seq_length(s) for s in sa] == [5 + 7 * i + 2 for i in range(6)]
    got, prob = a.decode_sample(sa[:2], tok[:2], u[:2])
    want, _ = ops.sample(d(a.logits(2)), d(u[:2]))
    np.testing.assert_array_equal(got, want.cpu().numpy())
    with pytest.raises(lib.IjbError):
        a.decode_sample([77], [0], [0.5])
    a.close()
    b.close()


def test_timing_helpers_on_a_paged_engine(cuda):
    cfg = synth.TINY
    e = Engine(cfg, synth.make_model(cfg, seed=3), context=96, max_batch=16, max_seqs=4, kv_type="e4m3")
    seqs = [e.seq_open() for _ in range(3)]
    for i, s in enumerate(seqs):
        e.seq_prefill(s, synth.prompt_tokens(10 + i, seed=i, vocab_limit=cfg.vocab))
    ms, kv_bytes = e.time_layer_attention(seqs, reps=3)
    assert ms > 0 and kv_bytes == 33 * cfg.kv_heads * 2 * (cfg.head_dim + 1)
    out = ctypes.c_float()
    assert e.lib.ijb_time_layer_projections(e.h, 8, 3, ctypes.byref(out)) == lib.OK and out.value > 0
    want = e.decode_step(seqs, [1, 2, 3])
    f = Engine(cfg, synth.make_model(cfg, seed=3), context=96, max_batch=16, max_seqs=4, kv_type="e4m3")
    again = [f.seq_open() for _ in range(3)]
    for i, s in enumerate(again):
        f.seq_prefill(s, synth.prompt_tokens(10 + i, seed=i, vocab_limit=cfg.vocab))
    np.testing.assert_array_equal(f.decode_step(again, [1, 2, 3]), want)  # the timing left no trace
    e.close()
    f.close()


def test_create_kv_refuses_other_types(cuda):
    L = lib.load()
    h = ctypes.c_void_p()
    d = lib.ModelDesc()
    views = (lib.TensorView * 1)()
    for t in (-1, 1, 3):
        assert L.ijb_create_kv(ctypes.byref(d), views, 0, t, ctypes.byref(h)) == lib.ERR_INVALID
        assert "cache type" in L.ijb_last_error(None).decode()


@pytest.mark.parametrize("kw,what", [(dict(page_size=12), "page_size"), (dict(max_batch=4097), "4096"),
                                     (dict(max_batch=64, kv_heads=1), "heads")])
def test_create_kv_refuses_what_its_attention_would(cuda, kw, what):
    cfg = synth.TINY
    if "kv_heads" in kw:
        kw.pop("kv_heads")
        cfg = synth.ModelConfig("mqa", dim=32 * 64, layers=1, heads=32, kv_heads=1, hidden=256, vocab=512)
    with pytest.raises(lib.IjbError, match=what):
        Engine(cfg, synth.make_model(cfg, seed=3), kv_type="f16", **dict(dict(context=96, max_batch=4, max_seqs=4), **kw))
