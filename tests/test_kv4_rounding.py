"""How 4-bit cache rows are rounded, at the ends of their scales: the definition that the kernel is held to
(test_gpu_kv4.py) against the bounds that the header states, and the kernel against the definition there."""
import numpy as np
import pytest

from test_gpu_kv4 import LEVELS, quantise, scale_table


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
