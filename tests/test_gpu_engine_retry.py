"""Engines on a B200 that ran out of pages in the middle of a call, and go on: against engines that had enough, step by
step the same (logits equal bit for bit)."""
import numpy as np
import pytest

from ijb200 import lib, synth
from ijb200.engine import Engine

pytestmark = pytest.mark.gpu
KW = dict(context=160, max_batch=8, max_seqs=5, use_dp4a=False, use_q6_dp4a=False)  # pages of 16
TYPES = pytest.mark.parametrize("kv_type", [None, "f16", "e4m3", "e2m1"])


@pytest.fixture(scope="module")
def weights():
    return synth.make_model(synth.TINY, seed=37)


def out_of_pages(call):
    with pytest.raises(lib.IjbError) as err:
        call()
    assert err.value.code == lib.ERR_CAPACITY


def step(e, seq, tokens):
    out = []
    for t in tokens:
        e.decode_step([seq], [int(t)])
        out.append(e.logits(1)[0])
    return np.array(out)


@TYPES
def test_steps_after_a_generate_that_ran_out_of_pages(cuda, weights, kv_type):
    """It takes what pages there are before it fails; they are the next steps'."""
    rng = np.random.default_rng(1)
    other, prompt, tail = (rng.integers(0, synth.TINY.vocab, n) for n in (40, 30, 50))
    a, b = Engine(synth.TINY, weights, kv_type=kv_type, num_pages=8, **KW), Engine(synth.TINY, weights, kv_type=kv_type, **KW)
    logits = []
    for e in (a, b):
        o, s = e.seq_open(), e.seq_open()
        e.seq_prefill(o, other)
        e.seq_prefill(s, prompt)      # 3 + 2 of the 8 pages
        if e is a:
            out_of_pages(lambda: e.generate(s, int(tail[0]), 120))
        logits.append(step(e, s, tail))
        logits[-1] = np.concatenate([logits[-1], step(e, o, tail[:8])])
        e.close()
    assert np.array_equal(*logits)


@TYPES
@pytest.mark.parametrize("pos", [20, 32])
def test_a_shared_page_without_a_page_to_replace_it(cuda, weights, kv_type, pos):
    """Sequence 0 writes to a page that a fork shares when none is left, goes on behind it, and writes there again later."""
    rng = np.random.default_rng(2)
    prompt, filler, tail = (rng.integers(0, synth.TINY.vocab, n) for n in (48, 32, 12))
    a, b = Engine(synth.TINY, weights, kv_type=kv_type, num_pages=5, **KW), Engine(synth.TINY, weights, kv_type=kv_type, **KW)
    logits = []
    for e in (a, b):
        e.prefill(prompt)
        f = e.seq_fork(0, 48)         # 3 pages, shared
        o = e.seq_open()
        e.seq_prefill(o, filler)      # the other 2
        if e is a:
            out_of_pages(lambda: e.forward(int(tail[0]), pos))
            assert e.seq_length(0) == 48 and e.seq_length(f) == 48
        e.seq_close(o)
        out = [step(e, f, tail[:2])]
        for i, t in enumerate(tail[:6]):
            e.forward(int(t), pos + i)
            out.append(e.logits(1))
        out.append(step(e, f, tail[6:]))
        logits.append(np.concatenate(out))
        e.close()
    assert np.array_equal(*logits)
