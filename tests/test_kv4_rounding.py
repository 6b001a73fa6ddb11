"""How 4-bit cache rows are rounded, at the ends of their scales: the definition that the kernel is held to
(test_gpu_kv4.py) against the bounds that the header states, and the kernel against the definition there."""
import numpy as np
import pytest

from test_gpu_kv4 import LEVELS, nearest, quantise, scale_table


def blocks(largest):
    """Blocks of 32 dims, a row of 64 each two, whose largest magnitudes are `largest`: their other values all over the
    range up to it."""
    largest = np.asarray(largest, np.float32)
    rng = np.random.default_rng(7)
    x = (largest[:, None] * rng.uniform(-1, 1, (len(largest), 32))).astype(np.float32)
    x[:, 1:9] = largest[:, None] * np.array([0.25, 0.4, 0.5, 0.6, 0.75, 0.8, 0.83, 0.84], np.float32)
    x[:, 17] = largest * rng.choice([-1, 1], len(largest))
    return x


def values(x):
    """What is read back of blocks x, in 64 bits."""
    codes, byte = quantise(x)
    c = np.stack([codes & 15, codes >> 4], -1).reshape(x.shape)
    return np.concatenate([LEVELS, -LEVELS])[c] * scale_table()[byte]


def spread(lo, hi, n=40000):
    return np.exp(np.random.default_rng(3).uniform(np.log(lo), np.log(hi), n))


def test_error_of_scales_that_are_normal_numbers():
    """The scale is off by 1 / 17 of itself at most, and values by half the step between 4 and 6 (up to half of the largest:
    between 2 and 3) times it: 18 / 17 / 6 = 0.1765 of the largest, 0.0883."""
    lo, hi = 6 * 2.0 ** -14, 61440.0
    x = blocks(np.concatenate([[lo, hi, np.nextafter(np.float32(7.125), np.float32(0))], spread(lo, hi)]))
    a, err = np.abs(x).max(-1, keepdims=True).astype(np.float64), np.abs(values(x) - x)
    assert (err <= 0.18 * a).all()
    assert (err <= np.where(np.abs(x) <= a / 2, 0.09, 0.18) * a).all()
    assert (err > 0.17 * a).any() and (err > np.where(np.abs(x) <= a / 2, 0.08, 1) * a).any()  # the bounds are near


def test_error_of_smaller_blocks():
    """Scales in steps of 2^-17: off by 2^-18 at most.  Codes up to 6 are off by a scale at most, larger values by six times
    what the scale is off."""
    x = blocks(np.concatenate([[8.9 * 2.0 ** -17, 5.9 * 2.0 ** -18, 6.1 * 2.0 ** -18], spread(2.0 ** -24, 6 * 2.0 ** -14)]))
    a, err = np.abs(x).max(-1, keepdims=True).astype(np.float64), np.abs(values(x) - x)
    assert (err <= np.maximum(a / 6 + 2.0 ** -18, 6 * 2.0 ** -18) * (1 + 2.0 ** -20)).all()  # (fp32's products in it)
    assert (err > 0.3 * a).any()
    assert (values(blocks([5.9 * 2.0 ** -18])) == 0).all()


def test_larger_values_and_infinities_become_the_largest():
    x = blocks([61440.0 * 1.01, 1e6, 3.4e38])
    v = values(x)
    assert (np.abs(v).max(-1) == 61440).all() and (np.abs(v) <= 61440).all()
    x = blocks([3.0, 2.0 ** -20])
    x[:, 5] = np.inf
    assert (values(x)[:, 5] == [3.0, 0.0]).all()
    assert (values(np.full((1, 32), -np.inf, np.float32)) == 0).all()


def borders():
    """Largest magnitudes where max|x| times fp32's 1 / 6 is halfway between two scales, or beside that.  Below 7.125
    (0x1.c7fffep+2) the product is a tie, and rounds up, where the quotient lies a unit of the last place below it."""
    m = np.array([1.0625, 1.1875, 1.3125, 1.4375, 1.5625, 1.6875, 1.8125, 1.9375], np.float32) * np.float32(6)
    near = np.stack([np.nextafter(m, np.float32(0)), m, np.nextafter(m, np.float32(99))])
    return (near[..., None] * np.float32(2) ** np.arange(-16, 14, dtype=np.float32)).ravel()


def test_the_borders_tell_the_product_from_the_quotient():
    a = borders()
    scales = scale_table()[:227]
    by = [nearest(scales, r.astype(np.float64)) for r in (a * (np.float32(1) / np.float32(6)), a / np.float32(6))]
    assert (by[0] != by[1]).any()
    low = np.nextafter(np.float32(7.125), np.float32(0))
    assert quantise(blocks([low]))[1].item() == 122 and scales[121] < low / np.float32(6) < scales[[121, 122]].mean()


@pytest.mark.gpu
@pytest.mark.parametrize("kvh,hd", [(1, 64), (2, 64), (8, 64), (1, 128), (8, 128)])
def test_kernel_at_the_borders(cuda, kvh, hd):
    """Codes and scale bytes at the borders and all over the range, rows of few heads a thread each and of many."""
    import torch
    from test_gpu_kv4 import make
    a = np.concatenate([borders(), spread(2.0 ** -24, 1e5, 20000 // hd * hd), [0.0] * 16]).astype(np.float32)
    x = blocks(a)
    n = len(x) * 32 // (2 * kvh * hd)
    x = x[:n * 2 * kvh * hd // 32].reshape(2, n, kvh, hd)
    kv = make(cuda, kvh, hd, 16, pages=-(-n // 16), seqs=1, max_pages=-(-n // 16))
    seq = torch.zeros((n,), dtype=torch.int32, device=cuda)
    pos = torch.arange(n, dtype=torch.int32, device=cuda)
    t = torch.from_numpy(x).to(cuda)
    kv.append(t[0], t[1], seq, pos)
    code, s = quantise(x)
    page = kv.page_table[0, (pos // 16).long()].cpu().numpy()
    off = pos.cpu().numpy() % 16
    got, got_s = kv.data.view(torch.uint8).cpu().numpy(), kv.scale.cpu().numpy()
    for which in range(2):
        np.testing.assert_array_equal(got_s[page, which, :, off], s[which])
        np.testing.assert_array_equal(got[page, which, :, off], code[which])
