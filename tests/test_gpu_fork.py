"""Forked sequences of an engine on a B200 (ijb_seq_fork) against sequences that were prefilled by themselves.

On an engine of ijb_create whose projections all run on the CUDA cores (max_batch below 16) a token's result does not
depend on the step it runs in, so a fork's logits are equal bit for bit to those of a sequence with the same tokens.
With tensor-core projections (steps of 3 tokens and more) or a cache type they are as long as the same steps ran: a
fork of a whole sequence goes on in the same steps as one that was prefilled alike."""
import numpy as np
import pytest

from ijb200 import lib, synth
from ijb200.engine import Engine

pytestmark = pytest.mark.gpu
KW = dict(context=160, max_batch=64, max_seqs=8, use_dp4a=False, use_q6_dp4a=False)
TYPES = pytest.mark.parametrize("kv_type", [None, "f32", "f16", "e4m3", "e2m1"])


@pytest.fixture(scope="module")
def weights():
    return synth.make_model(synth.TINY, seed=31)


def engine(weights, kv_type, **kw):
    kw = dict(KW, **kw)
    if kv_type == "f32":
        return Engine(synth.TINY, weights, kv_f32=True, **kw)
    return Engine(synth.TINY, weights, kv_type=kv_type, **kw)


def step(e, seq, tokens):
    """The logits of each of tokens, fed one at a time."""
    out = []
    for t in tokens:
        e.decode_step([seq], [int(t)])
        out.append(e.logits(1)[0])
    return np.array(out)


@TYPES
@pytest.mark.parametrize("length", [1, 15, 16, 17, 33, 48, 50])
def test_fork_and_its_parent_go_on_by_themselves(cuda, weights, kv_type, length):
    cfg = synth.TINY
    rng = np.random.default_rng(length)
    prompt, mine, theirs = (rng.integers(0, cfg.vocab, n) for n in (50, 40, 40))
    cut = prompt[:length] if kv_type in (None, "f32") else prompt  # what the sequences hold (see above)
    wide = 8 if kv_type in (None, "f32") else 64
    a, b = engine(weights, kv_type, max_batch=wide), engine(weights, kv_type, max_batch=wide)
    s, t = a.seq_open(), b.seq_open()
    a.seq_prefill(s, prompt)
    f = a.seq_fork(s, len(cut))
    b.seq_prefill(t, cut)
    u = b.seq_open()
    b.seq_prefill(u, prompt)
    for k in range(0, 40, 8):  # in turn, past the end of their pages
        got, want = step(a, f, mine[k:k + 8]), step(b, t, mine[k:k + 8])
        assert np.array_equal(got, want)
        got, want = step(a, s, theirs[k:k + 8]), step(b, u, theirs[k:k + 8])
        assert np.array_equal(got, want)
    a.seq_close(s)
    assert np.array_equal(step(a, f, theirs[:20]), step(b, t, theirs[:20]))
    a.close()
    b.close()


@TYPES
def test_forks_of_forks_in_one_step(cuda, weights, kv_type):
    """A prompt, several answers: all in one packed step, against sequences of their own."""
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, synth.TINY.vocab, 37)
    a, b = engine(weights, kv_type), engine(weights, kv_type)
    sa = [a.seq_open()]
    a.seq_prefill(sa[0], prompt)
    sb = []
    for _ in range(6):
        sb.append(b.seq_open())
        b.seq_prefill(sb[-1], prompt)
    while len(sa) < 6:
        sa.append(a.seq_fork(sa[len(sa) // 2]))
    for k in range(30):
        tok = rng.integers(0, synth.TINY.vocab, 6)
        assert np.array_equal(a.decode_step(sa, tok), b.decode_step(sb, tok))
        assert np.array_equal(a.logits(6), b.logits(6))
    a.close()
    b.close()


@TYPES
def test_sequence_0_set_back_leaves_its_forks_alone(cuda, weights, kv_type):
    rng = np.random.default_rng(5)
    p, q, tail = (rng.integers(0, synth.TINY.vocab, n) for n in (45, 70, 20))
    a, b = engine(weights, kv_type), engine(weights, kv_type)
    a.prefill(p)
    f = a.seq_fork(0)
    t = b.seq_open()
    b.seq_prefill(t, p)
    a.forward(int(q[0]), 20)  # in the middle of a shared page
    b.prefill(p)
    b.forward(int(q[0]), 20)
    assert np.array_equal(a.logits(1), b.logits(1))
    assert np.array_equal(step(a, f, tail[:5]), step(b, t, tail[:5]))
    a.prefill(q)              # over the others
    b.prefill(q)
    assert np.array_equal(a.logits(1), b.logits(1))
    assert np.array_equal(step(a, f, tail[5:]), step(b, t, tail[5:]))
    a.close()
    b.close()


def test_generate_on_a_fork(cuda, weights):
    p = synth.prompt_tokens(30, seed=5, vocab_limit=synth.TINY.vocab)
    for kv_type in (None, "e2m1"):
        e = engine(weights, kv_type)
        s = e.seq_open()
        nxt = e.seq_prefill(s, p)
        f, g = e.seq_fork(s), e.seq_fork(s)
        want = e.generate(s, nxt, 50)
        assert e.generate(f, nxt, 50) == want and e.generate(g, nxt, 50) == want
        assert e.seq_length(f) == e.seq_length(s)
        e.close()


def test_a_pool_of_shared_pages(cuda, weights):
    """Twelve pages hold five sequences of 5 pages each, which share 4; then there is none left."""
    e = engine(weights, "e2m1", num_pages=12, max_seqs=12)
    s = e.seq_open()
    e.seq_prefill(s, synth.prompt_tokens(64, seed=2, vocab_limit=synth.TINY.vocab))
    forks = [s] + [e.seq_fork(s) for _ in range(7)]
    e.decode_step(forks, [1] * 8)
    with pytest.raises(lib.IjbError) as err:
        e.seq_fork(forks[1])  # 65 positions: a page of its own
    assert err.value.code == lib.ERR_CAPACITY
    for f in forks[1:]:
        e.seq_close(f)
    t = e.seq_fork(s)
    assert np.array_equal(step(e, t, [7, 8, 9])[0], step(e, s, [7])[0])
    e.close()
