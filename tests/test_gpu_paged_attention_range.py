"""ijb_paged_attention on a B200 over e4m3 rows of very small and very large values, against 64 bits.

Tolerances (before the first run), on top of those in test_gpu_paged_attention.py (2e-5 of the largest
value; fp16 queries 2^-11 of a value and of the output more): a value of an e4m3 row enters as the nearest
fp16 number, which is the value itself where that is normal in fp16 (it has four bits), else off by 2^-25 at
most.  The weights sum to 1, so V's rounding moves an output by 2^-25 at most.  K's moves a score by D at most,
which the test computes from both values in 64 bits; the weights, quotients of exponentials, then move by
e^(2 D) - 1 of themselves at most, and so does an output relative to the largest value.
"""
import numpy as np
import pytest
from test_gpu_paged_attention import TYPES
from test_gpu_paged_attention_sums import i32

pytestmark = pytest.mark.gpu


def stored(cuda, n, kvh, hd, which, mag, seed):
    """An e4m3 cache of one sequence, written by append: rows of up to `mag` in K (0) or V (1), of up to 1 in the other."""
    import torch
    from ijb200 import ops
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    page, pages = 16, -(-n // 16)
    data = torch.zeros((pages, 2, kvh, page, hd), dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)
    scale = torch.zeros((pages, 2, kvh, page), dtype=torch.uint8, device=cuda)
    status = torch.zeros((1,), dtype=torch.int32, device=cuda)
    kv = ops.PagedKV(data, torch.randperm(pages, generator=g, device=cuda).view(1, -1).int(), scale, status)
    x = torch.rand((2, n, kvh, hd), generator=g, device=cuda) * 2 - 1
    x[which] *= mag
    seq, pos = i32(cuda, [0] * n), i32(cuda, list(range(n)))
    kv.append(x[0], x[1], seq, pos)
    return kv, x, seq, pos


def attend64(q, k, v, l, scale, seen=None):
    """(output, scores) in 64 bits; q [l, heads, hd] the last of the positions of k, v [t, kv heads, hd]."""
    import torch
    t, group = k.shape[0], q.shape[1] // k.shape[1]
    s = torch.einsum("lhd,thd->hlt", q.double(), k.double().repeat_interleave(group, 1)) * scale
    mask = torch.arange(t, device=q.device) <= (t - l + torch.arange(l, device=q.device)).unsqueeze(1)
    if seen is not None:
        mask = mask & seen
    s = torch.where(mask, s, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    return torch.einsum("hlt,thd->lhd", p, v.double().repeat_interleave(group, 1)), torch.where(mask, s, 0.0)


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("l", [1, 3, 40, 150])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("mag", [2.0 ** -40, 1e-6, 1e-5, 2e-5, 1e-3, 2.0 ** -7, 300.0, 2.0 ** 15, 6e4])
def test_e4m3_rows_of_any_size(cuda, hd, l, which, mag, dtype):
    import torch
    dtype = getattr(torch, dtype)
    n = l + 37
    kv, x, seq, pos = stored(cuda, n, 2, hd, which, mag, hd + l)
    k, v = (y.double() for y in kv.gather(seq, pos))
    g = torch.Generator(device=cuda)
    g.manual_seed(l)
    q = (torch.randn((l, 8, hd), generator=g, device=cuda) * 1.5).to(dtype)
    scale = hd ** -0.5 * (2.0 / mag if which == 0 and mag > 2.0 ** -30 else 2.0)
    got = kv.attention(q, i32(cuda, [0, l]), i32(cuda, [n]), max_q=l, scale=scale).double()
    assert int(kv.status) == 0
    want, s = attend64(q, k, v, l, scale)
    off = float((attend64(q, k.half(), v, l, scale)[1] - s).abs().max())
    top = float(v.abs().max())
    tol = (2e-5 + float(np.expm1(2 * off))) * top + 2.0 ** -25
    if dtype == torch.float16:
        tol = tol + 2.0 ** -11 * (top + want.abs()) + 2.0 ** -25  # the output may be subnormal in fp16
    assert ((got - want).abs() <= tol).all(), (float((got - want).abs().max()), float(want.abs().max()), off)


@TYPES
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("l", [1, 40])
def test_e4m3_values_beyond_fp16(cuda, hd, l, dtype):
    """A value that rounds past 65504 is an infinity to the tokens that see it; the others of its row are what they are."""
    import torch
    dtype = getattr(torch, dtype)
    n = l + 20
    kv, x, seq, pos = stored(cuda, n, 1, hd, 1, 1.0, 5)
    x[1, 7] = 1000.0
    x[1, 7, 0, 3] = 1e8
    kv.append(x[0], x[1], seq, pos)
    k, v = (y.double() for y in kv.gather(seq, pos))
    q = torch.randn((l, 2, hd), device=cuda).to(dtype)
    got = kv.attention(q, i32(cuda, [0, l]), i32(cuda, [n]), max_q=l).double()
    assert not torch.isfinite(got[:, :, 3]).any()
    rest = [d for d in range(hd) if d != 3]
    want = attend64(q, k, v, l, hd ** -0.5)[0][:, :, rest]
    top = float(v[:, :, rest].abs().max())
    tol = 2e-5 * top if dtype == torch.float32 else 2e-5 * top + 2.0 ** -11 * (top + want.abs())
    assert ((got[:, :, rest] - want).abs() <= tol).all()
