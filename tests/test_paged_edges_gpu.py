"""Paged attention and append at their edges: odd numbers of units, faint weights, empty sequences, extreme lengths and windows."""
import pytest
import torch

import tattletale_b200 as ttq
from paged_util import Batch, check_attention

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def run(ctx, bt, max_q=None, **kw):
    plan = bt.plan(ctx)
    out = plan.forward(bt.q, bt.k, bt.v, bt.batch(max_q), **kw)
    ctx.check_device_status()
    plan.close()
    return out


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("units", [1, 2, 3, 5, 7])
def test_items_of_odd_length_follow_each_other(ctx, units, d):
    """Items of one stream (128 rows or fewer) whose number of 128-key units is odd: the streams' places in the ring of tiles change with
    every item.  More such items than multiprocessors, then items of two streams among them; the same bits every time."""
    short, rows = [(40, 128 * units - 40 - i % 50) for i in range(90)], [(100, 128 * units + i) for i in range(9)]
    bt = Batch(short + rows + short[:20], 16, 8, d, 16, BF16, seed=units)
    first = run(ctx, bt)
    check_attention(first, bt)
    for _ in range(20):
        assert torch.equal(run(ctx, bt), first)
