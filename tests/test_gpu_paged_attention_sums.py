"""ijb_paged_attention on a B200: fp32 queries' sums over long runs of one warp, against 64 bits.

Tolerance (before the first run): a product of 16 positions is rounded once, and added to fp32 sums
that are rounded to nearest, two additions for 32 positions.  2^-25 rms an addition over the 1250 of 20000
positions gives 2^-25 * sqrt(1250) = 1.1e-6 if every sum on the way is as large as the last one; they are walks,
so about half.  Scores (8 products, truncated, 2^-24 of up to 16 each, times scale) and weights (22 bits) give
3e-7 more: 2^-19 (1.9e-6) rel-L2 holds, as for the chunks.
"""
import pytest
from test_gpu_paged_attention import CACHES, build

pytestmark = pytest.mark.gpu


def i32(cuda, v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device=cuda)


@CACHES
@pytest.mark.parametrize("group", [4, 12])
@pytest.mark.parametrize("hd", [64, 128])
def test_long_runs_of_single_tokens(cuda, cache, hd, group):
    """One token behind 20000, alone and as 300 entries of one sequence: runs of some thousand positions a warp."""
    import torch
    kv, dense = build(cuda, [20000], 2, hd, 16, cache, 3)
    g = torch.Generator(device=cuda)
    g.manual_seed(4)
    n = 300
    q = torch.randn((n, 2 * group, hd), generator=g, device=cuda)
    got = kv.attention(q, i32(cuda, list(range(n + 1))), i32(cuda, [20000] * n), seq=i32(cuda, [0] * n), max_q=1).double()
    k, v = dense[0]
    want = torch.empty((n, 2 * group, hd), dtype=torch.float64, device=cuda)
    for h in range(2 * group):
        want[:, h] = torch.softmax(q[:, h].double() @ k[h // group].T * hd ** -0.5, -1) @ v[h // group]
    assert float((got - want).norm() / want.norm()) < 2.0 ** -19
    one = kv.attention(q[:1], i32(cuda, [0, 1]), i32(cuda, [20000]), max_q=1).double()
    assert float((one - want[:1]).norm() / want[:1].norm()) < 2.0 ** -19
