"""Paged append and paged attention (windows, sinks, shared prefixes) against their definitions in 64 bits."""
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


# ---- attention ------------------------------------------------------------------------------------------------------

STEPS = [
    ([(1, 0)], 4, 4, 128, 16),                                   # one token, one key
    ([(1, 14), (1, 15), (1, 16), (1, 63), (1, 64)], 8, 2, 64, 16),   # around a page and a unit
    ([(1, 1530)], 32, 8, 128, 16),
    ([(1, 700), (1, 3), (1, 5000), (1, 0), (1, 129)], 28, 4, 128, 32),   # 7 query heads a kv head
    ([(3, 200), (1, 77), (2, 0)], 5, 5, 64, 64),                 # short drafts, no sharing of kv heads
    ([(1, 333)] * 40, 16, 1, 128, 128),
    ([(1, 90)], 64, 2, 64, 1024),                                # more query heads than a tile has rows
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("lens,hq,hkv,d,page", STEPS)
def test_steps(ctx, lens, hq, hkv, d, page, dtype):
    bt = Batch(lens, hq, hkv, d, page, dtype, seed=len(lens) + hq)
    check_attention(run(ctx, bt), bt)


PROMPTS = [
    ([(2, 0)], 4, 2, 128, 16),
    ([(17, 0), (1, 40), (130, 3)], 8, 2, 128, 16),               # prompts and a step in one batch
    ([(257, 0), (0, 9), (64, 511), (5, 0)], 12, 4, 64, 32),      # a sequence without new tokens
    ([(129, 1000)], 7, 1, 128, 64),
    ([(700, 0), (33, 2100)], 8, 8, 128, 128),
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("lens,hq,hkv,d,page", PROMPTS)
def test_prompts(ctx, lens, hq, hkv, d, page, dtype):
    bt = Batch(lens, hq, hkv, d, page, dtype, seed=len(lens) + hq)
    check_attention(run(ctx, bt), bt)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("lens,hq,hkv,d,page,window", [([(1500, 0), (777, 300)], 32, 8, 128, 64, 0), ([(1111, 40)], 40, 8, 64, 16, 300),
                                                       ([(900, 2000), (1, 5), (400, 0)], 28, 4, 128, 32, 0), ([(40, 3)] * 60, 16, 8, 64, 128, 0)])
def test_many_items_per_cta(ctx, lens, hq, hkv, d, page, window, dtype):
    """More row tiles and heads than the card has multiprocessors: every CTA serves items of several lengths, of one sequence and of
    several, whole ones and ends of ones begun elsewhere."""
    bt = Batch(lens, hq, hkv, d, page, dtype, seed=hq)
    check_attention(run(ctx, bt, window=window, sinks=5), bt, window, 5)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 0), (50, 4), (64, 64), (200, 130), (100000, 5)])
@pytest.mark.parametrize("lens,hq,hkv,d,page", [STEPS[3], PROMPTS[1], PROMPTS[2], PROMPTS[4]])
def test_windows(ctx, lens, hq, hkv, d, page, window, sinks):
    bt = Batch(lens, hq, hkv, d, page, BF16, seed=window)
    check_attention(run(ctx, bt, window=window, sinks=sinks), bt, window, sinks)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("prefix", [1, 16, 100, 777, 4097])
@pytest.mark.parametrize("lens,hq,hkv,d,page", [([(1, 0)], 8, 2, 128, 16), ([(1, 5), (1, 300), (1, 0)] * 7, 8, 2, 64, 32),
                                                ([(19, 0), (40, 7), (1, 64), (0, 3)], 28, 4, 128, 16), ([(150, 90), (3, 3)], 4, 4, 128, 64)])
def test_shared_prefix(ctx, lens, hq, hkv, d, page, prefix, dtype):
    bt = Batch(lens, hq, hkv, d, page, dtype, prefix=prefix, seed=prefix)
    check_attention(run(ctx, bt), bt)


@pytest.mark.parametrize("window,sinks", [(1, 2), (40, 0), (90, 17), (333, 64), (5000, 4)])
@pytest.mark.parametrize("lens", [[(1, 5), (1, 300), (1, 0)], [(19, 0), (40, 7), (1, 64)]])
def test_window_over_a_shared_prefix(ctx, lens, window, sinks):
    bt = Batch(lens, 8, 2, 128, 16, BF16, prefix=777, seed=window)
    check_attention(run(ctx, bt, window=window, sinks=sinks), bt, window, sinks)


@pytest.mark.parametrize("lens,hq,hkv,d,page,prefix", [
    ([(1, 30), (1, 700)], 160, 1, 64, 16, 0),        # more query heads on a kv head than a stream of the tensor-memory kernel has rows
    ([(3, 10), (40, 0)], 160, 1, 64, 32, 90),
    ([(3, 10), (70, 200)], 128, 1, 128, 256, 40),    # as many; pages longer than a unit
    ([(3, 10), (70, 200)], 65, 1, 64, 512, 0),       # half a stream idle
    ([(300, 1000)], 96, 2, 128, 1024, 0),
])
def test_many_query_heads_and_long_pages(ctx, lens, hq, hkv, d, page, prefix):
    bt = Batch(lens, hq, hkv, d, page, BF16, prefix=prefix, seed=hq)
    check_attention(run(ctx, bt), bt)
    check_attention(run(ctx, bt, window=64, sinks=7), bt, 64, 7)


@pytest.mark.parametrize("lens", [[(1, i % 97) for i in range(1000)], [(i % 5, 3 * i % 211) for i in range(800)], [(150, 0)] + [(1, 40)] * 500 + [(33, 70)]])
@pytest.mark.parametrize("prefix", [0, 33])
def test_many_sequences(ctx, lens, prefix):
    """More sequences than a CTA has threads."""
    bt = Batch(lens, 4, 2, 64, 16, BF16, prefix=prefix, seed=5)
    check_attention(run(ctx, bt), bt)
    plan = bt.plan(ctx)
    qkv = torch.randn(bt.rows, 8 * 64, device="cuda").to(BF16)
    n_rope = int(bt.kv_len.max())
    q = plan.append(qkv, bt.k, bt.v, bt.batch(), torch.ones(n_rope, 64, device="cuda"), torch.zeros(n_rope, 64, device="cuda"))
    ctx.check_device_status()
    assert torch.equal(q, qkv.view(-1, 8, 64)[:, :4])
    row = 0
    for b, (n, p) in enumerate(lens):
        if n and b % 50 == 0:
            at = p + n - 1
            assert torch.equal(bt.k[int(bt.table_host[b, at // 16]), :, at % 16], qkv[row + n - 1].view(8, 64)[4:6])
        row += n


@pytest.mark.parametrize("prefix", [0, 33])
@pytest.mark.parametrize("max_q", [1, 500])
def test_a_batch_without_new_tokens(ctx, prefix, max_q):
    """Every sequence sits this call out: nothing is written."""
    bt = Batch([(1, 20), (2, 300)], 8, 2, 128, 16, BF16, prefix=prefix)
    bt.q_start.zero_()
    out = torch.full((3, 8, 128), 3.0, dtype=BF16, device="cuda")
    plan = bt.plan(ctx)
    plan.forward(bt.q, bt.k, bt.v, bt.batch(max_q), out=out)
    assert (out == 3).all()
    k0 = bt.k.clone()
    plan.append(torch.ones(3, 12 * 128, dtype=BF16, device="cuda"), bt.k, bt.v, bt.batch(max_q), torch.ones(400, 128, device="cuda"),
                torch.ones(400, 128, device="cuda"), q_out=out)
    ctx.check_device_status()
    assert (out == 3).all() and torch.equal(k0.view(torch.int16), bt.k.view(torch.int16))


@pytest.mark.parametrize("new", [1, 200])
def test_infinite_values_that_nobody_sees(ctx, new):
    """Infinities and the type's extremes behind a sequence's end, in pages of nobody and before its window."""
    window = 70
    bt = Batch([(new, 400), (new, 77)], 8, 2, 128, 16, F16, seed=6)
    want = run(ctx, bt, window=window)
    for x, v in ((bt.k, float("inf")), (bt.v, -65504.0)):
        x[torch.isnan(x)] = v
    first = 400 - window + 1  # of sequence 0: no token sees the pages before this position
    for page in bt.table_host[0, :first // 16].tolist():
        bt.k[page], bt.v[page] = float("nan"), float("inf")
    got = run(ctx, bt, window=window)
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [1, 150])
def test_scores_of_great_range(ctx, new):
    """Scores that grow by hundreds along the keys, and rows whose first keys dwarf the rest: the running reference has to follow."""
    for sign in (1, -1):
        bt = Batch([(new, 900)], 4, 2, 64, 16, BF16, seed=7)
        pos = torch.arange(900 + new, device="cuda")
        pages, slots = bt.table_host[0][pos.cpu() // 16].long().cuda(), pos % 16
        bt.k[pages, :, slots, 0] = (sign * pos.float() * 0.5).to(BF16)[:, None]
        bt.q[..., 0] = 4.0
        check_attention(run(ctx, bt), bt)


@pytest.mark.parametrize("layout", ["nhd", "joint"])
def test_page_layouts(ctx, layout):
    bt = Batch([(1, 200), (9, 31), (140, 0)], 8, 4, 128, 16, BF16, layout=layout, seed=3)
    assert layout == "joint" or not bt.k.is_contiguous()
    check_attention(run(ctx, bt), bt)


def test_row_strides_scale_and_out(ctx):
    """q and out as column slices of wider buffers, a scale of one's own; the columns beside them stay."""
    bt = Batch([(1, 200), (30, 31)], 8, 4, 64, 16, F16, seed=4)
    wide = torch.zeros(bt.rows, 8 * 64 + 64, dtype=F16, device="cuda")
    wide[:, 64:] = bt.q.view(bt.rows, -1)
    out = torch.full((bt.rows, 8 * 64 + 8), 7.0, dtype=F16, device="cuda")
    plan = bt.plan(ctx)
    plan.forward(wide[:, 64:], bt.k, bt.v, bt.batch(), scale=0.2, out=out[:, :512])
    check_attention(out[:, :512].reshape(bt.rows, 8, 64), bt, scale=0.2)
    assert (out[:, 512:] == 7).all()


@pytest.mark.parametrize("lens", [[(1, 9), (1, 70)], [(50, 0), (200, 100)]])
@pytest.mark.parametrize("prefix", [0, 40])
def test_padded_batch_leaves_the_rows_behind_alone(ctx, lens, prefix):
    bt = Batch(lens, 8, 2, 128, 16, BF16, prefix=prefix, pad_rows=5)
    out = torch.full((bt.rows + 5, 8, 128), 3.0, dtype=BF16, device="cuda")
    plan = bt.plan(ctx)
    plan.forward(bt.q, bt.k, bt.v, bt.batch(), out=out)
    check_attention(out, bt)
    assert (out[bt.rows:] == 3).all()


def test_rows_without_keys_are_zero(ctx):
    """kv_len smaller than the new tokens: the first tokens have no position and see nothing; kv_len 0: none does."""
    bt = Batch([(6, 0), (300, 0)], 8, 2, 128, 16, BF16)
    bt.kv_len = torch.tensor([0, 296], dtype=torch.int32, device="cuda")
    out = run(ctx, bt)
    assert (out[:10] == 0).all()
    cut = Batch([(296, 0)], 8, 2, 128, 16, BF16)
    cut.table_host, cut.k, cut.v, cut.q = bt.table_host[1:], bt.k, bt.v, bt.q[10:]
    check_attention(out[10:], cut)


def test_no_sequences_and_no_tokens(ctx):
    bt = Batch([(1, 3)], 4, 2, 64, 16, BF16)
    plan = bt.plan(ctx)
    empty = ttq.PagedBatch(bt.q_start[:1], bt.kv_len[:0], bt.table[:0])
    out = torch.full((1, 4, 64), 3.0, dtype=BF16, device="cuda")
    plan.forward(bt.q, bt.k, bt.v, empty, out=out)
    assert (out == 3).all()
    assert plan.forward(bt.q[:0], bt.k, bt.v, bt.batch()).shape == (0, 4, 64)


def test_pages_out_of_the_window_are_not_read(ctx):
    """Pages that slid out of the window may have been given away: their table entries are -1."""
    bt = Batch([(1, 900), (40, 700)], 8, 2, 128, 16, BF16, seed=8)
    window, sinks = 100, 4
    want = run(ctx, bt, window=window, sinks=sinks)
    for b, (n, p) in enumerate(bt.lens):
        bt.table[b, 1:(p - window + 1) // 16] = -1
    assert torch.equal(run(ctx, bt, window=window, sinks=sinks), want)
    check_attention(want, bt, window, sinks)


def test_bad_pages_are_reported(ctx):
    for bad in (-1, 10 ** 9):
        bt = Batch([(1, 100), (20, 5)], 8, 2, 128, 16, BF16, seed=8)
        good = run(ctx, bt)
        bt.table[0, 3] = bad
        plan = bt.plan(ctx)
        out = plan.forward(bt.q, bt.k, bt.v, bt.batch())
        with pytest.raises(ttq.TtqError) as ei:
            ctx.check_device_status()
        assert ei.value.status == 2
        ctx.check_device_status()  # reported once
        assert torch.equal(out[1:], good[1:])  # the other sequence is as it was
    # more tokens than the table has pages for
    bt = Batch([(1, 100)], 8, 2, 128, 16, BF16, seed=8)
    bt.kv_len += 4000
    plan = bt.plan(ctx)
    plan.forward(bt.q, bt.k, bt.v, bt.batch())
    with pytest.raises(ttq.TtqError) as ei:
        ctx.check_device_status()
    assert ei.value.status == 2


def test_same_bits_whatever_max_q_says_and_twice(ctx):
    """A batch repeats bit for bit; max_q is a hint: each kernel gives results within the bound for any batch."""
    bt = Batch([(1, 2000), (37, 5), (200, 900)], 8, 2, 128, 16, BF16, prefix=50, seed=9)
    for max_q in (None, 0, 1, 1000):
        a, b = run(ctx, bt, max_q), run(ctx, bt, max_q)
        assert torch.equal(a, b)
        check_attention(a, bt)


def test_a_page_in_two_tables(ctx):
    """Two sequences may share pages (a forked chat)."""
    bt = Batch([(1, 200), (1, 200)], 8, 2, 128, 16, BF16, seed=10)
    bt.table[1] = bt.table[0]
    bt.table_host[1] = bt.table_host[0]
    check_attention(run(ctx, bt), bt)


@pytest.mark.parametrize("new", [1, 200])
def test_captured_call_follows_the_lengths(ctx, new):
    """A captured graph reads lengths, tables and rows anew at every replay; two graphs of two plans replay side by side."""
    lens = [(new, 700), (new, 64), (new, 1500)]
    bt = Batch(lens, 8, 2, 128, 16, BF16, seed=11)
    plans, outs, graphs, streams = [], [], [], [torch.cuda.Stream() for _ in range(2)]
    batch = bt.batch()
    for s in streams:
        plan = bt.plan(ctx)
        out = torch.zeros_like(bt.q)
        plan.forward(bt.q, bt.k, bt.v, batch, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            plan.forward(bt.q, bt.k, bt.v, batch, out=out)
        plans.append(plan), outs.append(out), graphs.append(graph)
    shorter = Batch([(new, 300), (new, 1), (new, 1499)], 8, 2, 128, 16, BF16, seed=11)
    bt.kv_len.copy_(shorter.kv_len)
    shorter.k, shorter.v, shorter.table_host, shorter.q = bt.k, bt.v, bt.table_host, bt.q
    for _ in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            check_attention(out, shorter)
    assert torch.equal(outs[0], outs[1])
    ctx.check_device_status()
    del graphs


def test_far_offsets(ctx):
    """A cache of more than 2^32 bytes whose used pages lie at its end, through a table wider than it needs to be."""
    page, hkv, d = 64, 8, 128
    n_pages = (1 << 33) // (page * hkv * d * 2) + 40   # 8 GB of keys
    bt = Batch([(1, 500), (20, 100)], 16, hkv, d, page, BF16, seed=12)
    k, v = (torch.zeros(n_pages, hkv, page, d, dtype=BF16, device="cuda") for _ in range(2))
    k[-bt.n_pages:], v[-bt.n_pages:] = bt.k, bt.v
    first = n_pages - bt.n_pages
    batch = ttq.PagedBatch(bt.q_start, bt.kv_len, torch.where(bt.table >= 0, bt.table + first, -1), max_q=20)
    plan = bt.plan(ctx)
    check_attention(plan.forward(bt.q, k, v, batch), bt)
    qkv = torch.randn(bt.rows, (16 + 2 * hkv) * d, device="cuda").to(BF16)
    cos, sin = torch.ones(601, d, device="cuda"), torch.zeros(601, d, device="cuda")
    plan.append(qkv, k, v, batch, cos, sin)
    ctx.check_device_status()
    page_of = first + int(bt.table_host[0, 500 // page])
    assert torch.equal(v[page_of, :, 500 % page], qkv[0].view(-1, d)[16 + hkv:])
    assert torch.equal(k[page_of, :, 500 % page], qkv[0].view(-1, d)[16:16 + hkv])


# ---- append ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,rope", [(BF16, torch.float32), (BF16, BF16), (F16, torch.float32), (F16, F16)])
@pytest.mark.parametrize("lens,hq,hkv,d,page,prefix", [([(1, 0)], 4, 4, 64, 16, 0), ([(1, 100), (1, 15), (1, 16)], 32, 8, 128, 16, 0),
                                                       ([(33, 0), (0, 7), (150, 20), (1, 63)], 28, 4, 128, 64, 0),
                                                       ([(1500, 10)], 5, 1, 64, 32, 0), ([(3, 4), (20, 0)], 8, 2, 128, 16, 37)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(ctx, lens, hq, hkv, d, page, prefix, dtype, rope, norm):
    bt = Batch(lens, hq, hkv, d, page, dtype, prefix=prefix, seed=hq, pad_rows=2)
    g = torch.Generator(device="cuda").manual_seed(hq)
    n = bt.rows
    wide = torch.randn(n + 2, (hq + 2 * hkv) * d + 8, generator=g, device="cuda").to(dtype)
    qkv = wide[:, :-8]  # a row pitch of its own
    longest = int(bt.kv_len.max())
    ang = torch.arange(longest, device="cuda", dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    cos, sin = (torch.cat([f(ang), f(ang) * 0.9], 1).to(rope) for f in (torch.cos, torch.sin))  # halves need not repeat
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype) if norm else None for _ in range(2))
    k0, v0 = bt.k.clone(), bt.v.clone()
    q_out = torch.full((n + 2, hq, d), 5.0, dtype=dtype, device="cuda")
    plan = bt.plan(ctx)
    q = plan.append(qkv, bt.k, bt.v, bt.batch(), cos, sin, q_norm=wq, k_norm=wk, eps=1e-6, q_out=q_out)
    ctx.check_device_status()
    assert q is q_out and (q_out[n:] == 5).all()
    u = torch.finfo(dtype).eps / 2
    row = 0
    for b, (new, past) in enumerate(lens):
        pos = torch.arange(past, past + new)
        pages, slots = bt.table_host[b][pos // page].long().cuda(), (pos % page).cuda()
        x = qkv[row:row + new].double().view(new, hq + 2 * hkv, d)
        c, s = cos.double()[prefix + pos.cuda()][:, None], sin.double()[prefix + pos.cuda()][:, None]
        for heads, weight, got in ((x[:, :hq], wq, q[row:row + new]), (x[:, hq:hq + hkv], wk, bt.k[pages, :, slots])):
            if weight is not None:
                heads = heads / ((heads ** 2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
            turned = torch.cat([-heads[..., d // 2:], heads[..., :d // 2]], -1)
            want = heads * c + turned * s
            # one rounding to the type; a dozen 32-bit roundings of the two terms (rsqrt, sums of squares: 2^-20 in all)
            bound = u * want.abs() + 2.0 ** -20 * ((heads * c).abs() + (turned * s).abs()) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
            assert ((got.double() - want).abs() <= bound).all()
        assert torch.equal(bt.v[pages, :, slots], qkv[row:row + new].reshape(new, hq + 2 * hkv, d)[:, hq + hkv:])
        k0[pages, :, slots], v0[pages, :, slots] = bt.k[pages, :, slots], bt.v[pages, :, slots]
        row += new
    assert torch.equal(k0.view(torch.int16), bt.k.view(torch.int16)) and torch.equal(v0.view(torch.int16), bt.v.view(torch.int16))  # nothing else was written


@pytest.mark.parametrize("layout", ["nhd", "joint"])
def test_append_into_other_layouts(ctx, layout):
    bt = Batch([(5, 30), (1, 2)], 4, 2, 64, 16, BF16, layout=layout, seed=1)
    qkv = torch.randn(bt.rows, 8 * 64, device="cuda").to(BF16)
    plan = bt.plan(ctx)
    plan.append(qkv, bt.k, bt.v, bt.batch(), torch.ones(40, 64, device="cuda"), torch.zeros(40, 64, device="cuda"))
    heads = qkv.view(bt.rows, 8, 64)
    for row, (b, pos) in enumerate([(0, 30), (0, 31), (0, 32), (0, 33), (0, 34), (1, 2)]):
        at = int(bt.table_host[b, pos // 16])
        assert torch.equal(bt.k[at, :, pos % 16], heads[row, 4:6]) and torch.equal(bt.v[at, :, pos % 16], heads[row, 6:])


def test_append_reports_bad_positions(ctx):
    """A page id or a position outside the tables: that token is skipped, the others are written, the status says so."""
    for what in ("page", "far page", "table", "rope", "negative"):
        bt = Batch([(2, 30), (1, 2)], 4, 2, 64, 16, BF16, seed=1)
        qkv = torch.randn(3, 8 * 64, device="cuda").to(BF16)
        n_rope = 40
        if what == "page":
            bt.table[0, 1] = -1
        elif what == "far page":
            bt.table[0, 1] = bt.n_pages
        elif what == "table":
            bt.kv_len[0] += 1000
            n_rope = 2000
        elif what == "rope":
            n_rope = 30
        else:
            bt.kv_len[0] = 0
        k0, v0 = bt.k.clone(), bt.v.clone()
        plan = bt.plan(ctx)
        q_out = torch.full((3, 4, 64), 5.0, dtype=BF16, device="cuda")
        plan.append(qkv, bt.k, bt.v, bt.batch(), torch.ones(n_rope, 64, device="cuda"), torch.zeros(n_rope, 64, device="cuda"), q_out=q_out)
        with pytest.raises(ttq.TtqError) as ei:
            ctx.check_device_status()
        assert ei.value.status == 2, what
        assert (q_out[:2] == 5).all() and torch.equal(q_out[2], qkv[2].view(8, 64)[:4])
        at = int(bt.table_host[1, 0])
        k0[at, :, 2], v0[at, :, 2] = qkv[2].view(8, 64)[4:6], qkv[2].view(8, 64)[6:]
        assert torch.equal(k0.view(torch.int16), bt.k.view(torch.int16)) and torch.equal(v0.view(torch.int16), bt.v.view(torch.int16))


# ---- refusals -------------------------------------------------------------------------------------------------------

def refused(status, fn, *a, **kw):
    with pytest.raises(ttq.TtqError) as ei:
        fn(*a, **kw)
    assert ei.value.status == status, ei.value


def test_plan_refusals(ctx):
    for status, args in ((2, (6, 4, 128, 16)), (2, (0, 0, 128, 16)), (3, (8, 2, 96, 16)), (3, (8, 2, 256, 16)), (3, (8, 2, 128, 8)), (3, (8, 2, 128, 48))):
        refused(status, ttq.PagedAttention, ctx, *args, max_seqs=4, max_tokens=4)
    refused(1, ttq.PagedAttention, ctx, 8, 2, 128, 16, max_seqs=4, max_tokens=4, dtype=torch.float32)
    refused(2, ttq.PagedAttention, ctx, 8, 2, 128, 16, max_seqs=0, max_tokens=4)
    refused(2, ttq.PagedAttention, ctx, 8, 2, 128, 16, max_seqs=1, max_tokens=1 << 40)
    refused(2, ttq.PagedAttention, ctx, 8, 2, 128, 16, max_seqs=1, max_tokens=4, max_prefix_tokens=5)


def test_call_refusals(ctx):
    bt = Batch([(1, 20), (2, 20)], 8, 2, 128, 16, BF16)
    plan = bt.plan(ctx)
    batch = bt.batch()
    refused(2, plan.forward, bt.q[:, :4], bt.k, bt.v, batch)                       # heads missing
    refused(1, plan.forward, bt.q.to(F16), bt.k, bt.v, batch)
    refused(1, plan.forward, bt.q.cpu(), bt.k, bt.v, batch)
    refused(2, plan.forward, bt.q, bt.k[:, :1], bt.v, batch)
    refused(2, plan.forward, bt.q, bt.k, bt.v.clone().transpose(0, 1).contiguous().transpose(0, 1), batch)   # strides differ
    refused(2, plan.forward, bt.q, bt.k, bt.v, batch, window=-1)
    refused(1, plan.forward, bt.q, bt.k, bt.v, batch, scale=0.0)
    refused(1, plan.forward, bt.q, bt.k, bt.v, batch, scale=float("nan"))
    refused(7, plan.forward, torch.cat([bt.q, bt.q]), bt.k, bt.v, batch)           # more rows than the plan holds
    off = torch.zeros(bt.q.numel() + 8, dtype=BF16, device="cuda")[4:-4].view_as(bt.q)
    refused(1, plan.forward, off, bt.k, bt.v, batch)                               # rows at 8-byte offsets
    big = torch.zeros(bt.k.numel() + 8, dtype=BF16, device="cuda")[4:-4].view_as(bt.k)
    refused(1, plan.forward, bt.q, big, big, batch)
    odd = torch.zeros(bt.n_pages, 2, 16, 132, dtype=BF16, device="cuda")[..., :128]
    refused(2, plan.forward, bt.q, odd, odd, batch)                                # slots 264 bytes apart
    few = ttq.PagedAttention(ctx, 8, 2, 128, 16, max_seqs=1, max_tokens=3)
    refused(7, few.forward, bt.q, bt.k, bt.v, batch)                               # more sequences
    pre = Batch([(1, 20), (2, 20)], 8, 2, 128, 16, BF16, prefix=20)
    none = pre.plan(ctx, max_prefix_tokens=2)
    refused(7, none.forward, pre.q, pre.k, pre.v, pre.batch())
    refused(2, plan.forward, bt.q, bt.k, bt.v, ttq.PagedBatch(bt.q_start, bt.kv_len, bt.table, prefix_len=17, prefix_table=bt.table[0, :1]))
    refused(2, plan.forward, bt.q, bt.k, bt.v, ttq.PagedBatch(bt.q_start, bt.kv_len, bt.table, prefix_len=-1))
    cos = torch.ones(30, 128, device="cuda")
    qkv = torch.zeros(3, 12 * 128, dtype=BF16, device="cuda")
    refused(2, plan.append, qkv[:, :-128], bt.k, bt.v, batch, cos, cos)
    refused(1, plan.append, qkv, bt.k, bt.v, batch, cos.half(), cos.half())        # neither f32 nor the plan's type
    refused(2, plan.append, qkv, bt.k, bt.v, batch, cos[:, :64], cos[:, :64])
    refused(2, plan.append, qkv, bt.k, bt.v, batch, cos, cos, q_norm=torch.ones(64, dtype=BF16, device="cuda"))
    refused(2, plan.append, qkv, bt.k, bt.v, batch, cos, cos, q_out=torch.empty(3, 8, 64, dtype=BF16, device="cuda"))
    refused(1, plan.append, qkv, bt.k, bt.v, batch, cos[:0], cos[:0])            # no rows: no pointer
    ctx.check_device_status()
