"""The sampler at its edges: random numbers outside their range, one row for all, settings beyond their type."""
import numpy as np
import pytest
import torch

import tattletale_b200 as ttq
from paged_util import sample64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("u", [1.0, 2.0, float("inf"), -1.0, float("nan")])
@pytest.mark.parametrize("v", [7, 1000, 100000])
def test_random_numbers_outside_their_range(ctx, v, u):
    """They count as the nearest in [0, 1): every row gets a token that was kept, flat rows of a great total weight too."""
    logits = torch.zeros(5, v, device="cuda")
    logits[2, v // 2] = -float("inf")
    logits[3, v - 1] = -float("inf")
    clamped = np.float32(0 if u != u else min(max(u, 0.0), 1.0 - 2.0 ** -24))
    for s in (dict(), dict(top_k=max(1, v // 3)), dict(top_p=0.37), dict(temperature=9.0)):
        for dtype in (torch.float32, torch.bfloat16):
            out = torch.full((5,), -7, dtype=torch.int64, device="cuda")
            ttq.sample(ctx, logits.to(dtype), torch.full((5,), u, device="cuda"), out=out, **s)
            want = [sample64(logits[r].cpu().numpy(), clamped, np.float32(s.get("temperature", 1.0)), s.get("top_k", 0), np.float32(s.get("top_p", 1.0)), 0.0)
                    for r in range(5)]
            assert out.tolist() == want


@pytest.mark.parametrize("v", [1, 5000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_draws_from_one_row(ctx, v, dtype):
    """Rows of pitch 0: an expanded row is as good as copies of it."""
    g = torch.Generator().manual_seed(v)
    x, u = torch.randn(v, generator=g).to(dtype).cuda(), torch.rand(300, generator=g).cuda()
    for s in (dict(), dict(top_k=40, top_p=0.9), dict(temperature=0.0)):
        assert torch.equal(ttq.sample(ctx, x.expand(300, -1), u, **s), ttq.sample(ctx, x.repeat(300, 1), u, **s))


def test_overlapping_rows_are_refused(ctx):
    with pytest.raises(ttq.TtqError) as ei:
        ttq.sample(ctx, torch.zeros(150, device="cuda").as_strided((2, 100), (50, 1)), torch.zeros(2, device="cuda"))
    assert ei.value.status == 2


def test_top_k_beyond_32_bits(ctx):
    """More than the vocabulary, or 0 and less: no cut."""
    g = torch.Generator().manual_seed(1)
    x, u = torch.randn(64, 5000, generator=g).cuda(), torch.rand(64, generator=g).cuda()
    want = ttq.sample(ctx, x, u)
    for k in (5000, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, 2 ** 40, -1, -2 ** 32 + 5):
        assert torch.equal(ttq.sample(ctx, x, u, top_k=k), want), k


@pytest.mark.parametrize("min_p", [1.0, 1.5, float("inf")])
def test_min_p_of_one_keeps_the_largest_logit_alone(ctx, min_p):
    """A weight of 1 - 10^-14 is less than 1, though not as 2^-44 fixed point; equal logits are all the largest."""
    x = torch.zeros(4, 600, device="cuda")
    x[:, ::2] = -1e-10
    x[1:, 11:] = -1e-10
    x[2:, 3] = -1e-10
    for u in (0.0, 0.3, 0.7, 0.9999):
        got = ttq.sample(ctx, x, torch.full((4,), u, device="cuda"), temperature=1e4, min_p=min_p)
        u = float(np.float32(u))
        want = [1 + 2 * int(u * 300), 1 + 2 * int(u * 5), [1, 5, 7, 9][int(u * 4)], [1, 5, 7, 9][int(u * 4)]]
        assert got.tolist() == want
