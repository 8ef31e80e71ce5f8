"""Paged attention and append at their edges: odd numbers of units, faint weights, empty sequences, extreme lengths and windows."""
import math

import pytest
import torch

import tattletale_b200 as ttq
from paged_util import Batch, attention64, check_attention

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


@pytest.mark.parametrize("new", [1, 12, 40])
def test_faint_weights_behind_a_dominant_key(ctx, new):
    """f16: a first key of value zero that outweighs each of 30000 others by 2^25.  The result is theirs: weights that the 16-bit type
    cannot hold relative to the row's largest still have to count.  320 sequences that share their pages, so that a CTA sees whole
    rows.  The bound: as in attention64, and weights off by 2^-34 of the largest (half a step of 2^-24 at a largest weight of 2^9),
    and half a step of 2^-24 of the result."""
    past, d, hq, seqs, page = 30000, 64, 2, 320, 64
    bt = Batch([(new, past)], hq, 1, d, page, F16, seed=1)
    total = past + new
    pos = torch.arange(total)
    pages, slots = bt.table_host[0][pos // page].long().cuda(), (pos % page).cuda()
    g = torch.Generator(device="cuda").manual_seed(2)
    k = torch.zeros(total, d, device="cuda")
    k[:, 0] = 0.3 * torch.rand(total, generator=g, device="cuda")
    k[0, 0] = 17.7
    v = 1.0 + torch.rand(total, d, generator=g, device="cuda")
    v[0] = 0.0
    bt.k[pages, 0, slots], bt.v[pages, 0, slots] = k.to(F16), v.to(F16)
    bt.q.zero_()
    bt.q[..., 0] = 8.0
    k64, v64 = bt.keys(0)
    q = bt.q.double().transpose(0, 1)
    seen = torch.arange(total, device="cuda")[None] <= torch.arange(past, total, device="cuda")[:, None]
    w = torch.softmax(torch.where(seen, q @ k64.transpose(1, 2) / 8.0, -math.inf), -1)
    want = (w @ v64).transpose(0, 1)
    u, err_s = 2.0 ** -11, d * 2.0 ** -23 * 17.7
    bound = want * (2 * u + 2 * err_s + 2.0 ** -18) + 2.0 ** -34 * v64.abs().sum(1)[0] + 2.0 ** -25
    ints = torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
    batch = ttq.PagedBatch(ints * new, torch.full((seqs,), total, dtype=torch.int32, device="cuda"), bt.table.expand(seqs, -1).contiguous(), max_q=new)
    plan = ttq.PagedAttention(ctx, hq, 1, d, page, max_seqs=seqs, max_tokens=seqs * new, dtype=F16)
    got = plan.forward(bt.q.repeat(seqs, 1, 1), bt.k, bt.v, batch).double().view(seqs, new, hq, d)
    ctx.check_device_status()
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()


@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("slope", [-0.5, 0.03, 0.5])
def test_f16_scores_of_great_range(ctx, new, slope):
    """Scores that grow or fall by up to hundreds along the keys: weights stay finite in f16 and the reference follows."""
    bt = Batch([(new, 900)], 4, 2, 64, 16, F16, seed=7)
    pos = torch.arange(900 + new)
    pages, slots = bt.table_host[0][pos // 16].long().cuda(), (pos % 16).cuda()
    bt.k[pages, :, slots, 0] = (slope * pos.float()).to(F16).cuda()[:, None]
    bt.q[..., 0] = 4.0
    check_attention(run(ctx, bt), bt)


@pytest.mark.parametrize("new", [1, 150])
def test_f16_flat_scores(ctx, new):
    """Equal scores everywhere: the largest sums of weights that a tile can have."""
    bt = Batch([(new, 900)], 4, 2, 64, 16, F16, seed=7)
    bt.q.fill_(0.0)
    check_attention(run(ctx, bt), bt)
    bt.k[:], bt.q[:] = 0.5, 0.5
    check_attention(run(ctx, bt), bt)


@pytest.mark.parametrize("sinks", [0, 5])
@pytest.mark.parametrize("new", [1, 40])
def test_padding_sequences_of_a_batch_with_a_prefix(ctx, new, sinks):
    """A sequence of length 0 that brings a token (a batch padded for a graph) sees nothing, so it makes nothing visible either: what the
    prefix holds before everybody's window stays unread, and its pages may have been given away."""
    window, prefix = 64, 777
    bt = Batch([(new, 20), (1, 0), (new, 30)], 8, 2, 128, 16, BF16, prefix=prefix, seed=3)
    bt.kv_len[1] = 0
    plan = bt.plan(ctx)
    want = plan.forward(bt.q, bt.k, bt.v, bt.batch(), window=window, sinks=sinks)
    ctx.check_device_status()
    rows = torch.arange(bt.rows, device="cuda") != new
    w64, bound = attention64(bt, window, sinks)
    assert ((want.double() - w64).abs() <= bound)[rows].all() and (want[new] == 0).all()
    hidden = slice(1 if sinks else 0, (prefix + 20 - window + 1) // 16)
    for page in bt.prefix_host[hidden].tolist():
        bt.k[page], bt.v[page] = float("nan"), float("nan")
    given_away = bt.prefix_host.clone()
    given_away[hidden] = -1
    for table in (bt.prefix_host, given_away):
        batch = ttq.PagedBatch(bt.q_start, bt.kv_len, bt.table, max_q=new, prefix_len=prefix, prefix_table=table.cuda())
        assert torch.equal(plan.forward(bt.q, bt.k, bt.v, batch, window=window, sinks=sinks), want)
        ctx.check_device_status()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 62])
@pytest.mark.parametrize("new,kv", [(10, 4), (300, 200), (2, 900)])
@pytest.mark.parametrize("prefix", [0, 40])
def test_windows_beyond_every_position(ctx, new, kv, window, prefix):
    """As no window at all, with tokens before position 0 too."""
    bt = Batch([(new, 1000)], 8, 2, 128, 16, BF16, prefix=prefix, seed=4)
    bt.kv_len[0] = kv
    want = run(ctx, bt)
    assert torch.equal(run(ctx, bt, window=window), want)
    assert torch.isfinite(want).all() and (want[:max(0, new - kv)] == 0).all()


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("window", [0, 50])
def test_lengths_at_the_ends_of_their_type(ctx, new, window):
    """Negative lengths are no length; a length beyond the table is reported.  The other sequence is as it was."""
    bt = Batch([(new, 90), (new, 70)], 8, 2, 128, 16, BF16, prefix=33, seed=5)
    want, bound = attention64(bt, window)
    plan = bt.plan(ctx)
    for length in (0, -1, -5000, -2 ** 31, -2 ** 31 + 40):
        bt.kv_len[0] = length
        out = plan.forward(bt.q, bt.k, bt.v, bt.batch(), window=window)
        ctx.check_device_status()
        assert (out[:new] == 0).all()
        assert ((out.double() - want).abs() <= bound)[new:].all()
    bt.kv_len[0] = 2 ** 31 - 1
    plan.forward(bt.q, bt.k, bt.v, bt.batch(), window=window)
    with pytest.raises(ttq.TtqError) as ei:
        ctx.check_device_status()
    assert ei.value.status == 2


def test_append_at_negative_lengths_of_a_wide_table(ctx):
    """A position below zero is outside whatever the table's width: nothing is read or written for its token.  (With 2^27 - 1 pages and a
    prefix, its distance from the prefix passes 32 bits and would be a place in the table.)"""
    bt = Batch([(1, 20)], 4, 2, 64, 16, BF16, prefix=100, seed=1)
    wide = torch.zeros(1, (2 ** 31 - 1) // 16, dtype=torch.int32, device="cuda")
    plan = bt.plan(ctx)
    k0 = bt.k.clone()
    for length in (0, 100, -2 ** 31, -2 ** 31 + 50):
        bt.kv_len[0] = length
        batch = ttq.PagedBatch(bt.q_start, bt.kv_len, wide, max_q=1, prefix_len=100, prefix_table=bt.prefix_host.cuda())
        out = torch.full((1, 4, 64), 3.0, dtype=BF16, device="cuda")
        plan.append(torch.ones(1, 8 * 64, dtype=BF16, device="cuda"), bt.k, bt.v, batch, torch.ones(200, 64, device="cuda"), torch.ones(200, 64, device="cuda"), q_out=out)
        with pytest.raises(ttq.TtqError) as ei:
            ctx.check_device_status()
        assert ei.value.status == 2 and (out == 3).all() and torch.equal(k0.view(torch.int16), bt.k.view(torch.int16))


def test_a_plan_outlives_its_context():
    """Contexts are closed and collected in any order: a plan that goes later asks nothing of its context."""
    ctx = ttq.Context(0)
    plans = [ttq.PagedAttention(ctx, 8, 2, 64, 16, max_seqs=4, max_tokens=4) for _ in range(2)]
    ctx.close()
    held = torch.cuda.mem_get_info()[0]
    for plan in plans:
        plan.close()
    assert torch.cuda.mem_get_info()[0] >= held and torch.cuda.current_device() == 0
    with pytest.raises(ttq.TtqError):
        ttq.PagedAttention(ctx, 8, 2, 64, 16, max_seqs=4, max_tokens=4)


def test_a_batch_shared_by_plans(ctx):
    """Two threads with contexts of their own may use one batch: a call's arguments stay as they were handed over."""
    bt = Batch([(1, 20), (2, 20)], 8, 2, 128, 16, BF16)
    plan, batch = bt.plan(ctx), bt.batch()
    first = batch._for(plan, 3)
    second = batch._for(plan, 2)
    assert (first.n_tokens, second.n_tokens) == (3, 2) and second.kv_len_dev == first.kv_len_dev == bt.kv_len.data_ptr()
    check_attention(plan.forward(bt.q, bt.k, bt.v, batch), bt)


@pytest.mark.parametrize("d,new,prefix", [(128, 40, 0), (64, 100, 0), (128, 25, 59000)])
def test_one_item_cut_into_as_many_parts_as_there_are_ctas(ctx, d, new, prefix):
    """One row tile against 60000 keys: every multiprocessor has a part of it."""
    bt = Batch([(new, 60000 - prefix)], 4, 1, d, 64, BF16, prefix=prefix, seed=d)
    first = run(ctx, bt)
    check_attention(first, bt)
    assert torch.equal(run(ctx, bt), first)
