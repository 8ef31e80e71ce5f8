"""The sampler against its definition in 64 bits: tokens have to be equal."""
import numpy as np
import pytest
import torch

import tattletale_b200 as ttq
from paged_util import sample64

pytestmark = pytest.mark.gpu
SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.95, 0.0), (0.8, 50, 0.9, 0.0), (1.3, 1000, 1.0, 0.02), (0.0, 0, 1.0, 0.0), (1.1, 0, 0.99, 0.001),
            (0.5, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (2.0, 3, 0.5, 0.0), (1.0, 0, 1.0, 1.0), (0.01, 0, 0.5, 0.0), (50.0, 0, 0.3, 0.0), (float("nan"), 5, 0.5, 0.0)]


def expect(logits, u, settings):
    x, uu = logits.float().cpu().numpy(), u.cpu().numpy()
    f = [np.float32(s) for s in np.asarray([s[0] for s in settings])], [np.float32(s[2]) for s in settings], [np.float32(s[3]) for s in settings]
    return torch.tensor([sample64(x[r], uu[r], f[0][r], settings[r][1], f[1][r], f[2][r]) for r in range(len(x))])


def per_row(settings):
    t = torch.tensor(settings, dtype=torch.float64)
    return dict(temperature=t[:, 0].float().cuda(), top_k=t[:, 1].int().cuda(), top_p=t[:, 2].float().cuda(), min_p=t[:, 3].float().cuda())


def check(ctx, logits, u, settings):
    got = ttq.sample(ctx, logits, u, **per_row(settings)).cpu()
    want = expect(logits, u, settings)
    assert torch.equal(got, want), (got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [1, 2, 31, 1000, 4097, 32001, 128256, 262144])
def test_settings(ctx, v, dtype):
    """Every combination of settings, rows in a pitch of their own; 16-bit logits tie all over the row."""
    g = torch.Generator().manual_seed(v)
    m = len(SETTINGS) * (3 if v < 40000 else 1)
    wide = 3.0 * torch.randn(m, v + 3, generator=g)
    logits = wide.to(dtype).cuda()[:, 1:v + 1]
    u = torch.rand(m, generator=g).cuda()
    check(ctx, logits, u, [SETTINGS[r % len(SETTINGS)] for r in range(m)])


def test_random_settings_and_numbers(ctx):
    g = torch.Generator().manual_seed(1)
    rng = np.random.default_rng(1)
    m, v = 400, 5003
    logits = (torch.rand(m, 1, generator=g) * 6 * torch.randn(m, v, generator=g)).cuda()
    settings = [(float(rng.choice([0.3, 0.9, 1.0, 1.7])), int(rng.choice([0, 1, 2, 7, 40, 900, 9000])), float(rng.choice([1.0, 0.2, 0.8, 0.97])),
                 float(rng.choice([0.0, 0.01, 0.3]))) for _ in range(m)]
    check(ctx, logits, torch.rand(m, generator=g).cuda(), settings)


def test_ties_and_signed_zeros(ctx):
    """Equal logits are kept lowest index first; -0 and +0 are equal."""
    v = 1000
    flat = torch.zeros(v)
    flat[1::2] = -0.0
    few = torch.where(torch.arange(v) % 7 == 3, 2.0, -1.0)
    rows, us, settings = [], [], []
    for x in (flat, few):
        for s in ((1.0, 10, 1.0, 0.0), (1.0, 0, 0.25, 0.0), (1.0, 500, 0.5, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.9), (0.7, 143, 0.999, 0.0)):
            for u in (0.0, 0.3, 0.5, 0.99999994):
                rows.append(x), us.append(u), settings.append(s)
    check(ctx, torch.stack(rows).cuda(), torch.tensor(us).cuda(), settings)
    # uniform weights: the definition's cuts are exact
    got = ttq.sample(ctx, flat[None].cuda(), torch.tensor([0.99999994]).cuda(), top_p=0.5)
    assert int(got) == 499
    got = ttq.sample(ctx, flat[None].cuda(), torch.tensor([0.0]).cuda(), temperature=0.0)
    assert int(got) == 0


def test_many_equal_logits(ctx):
    """Ten thousands of tokens that tie at the cut, and a bulk far narrower than the row's range."""
    v = 60000
    g = torch.Generator().manual_seed(7)
    flat = torch.zeros(v)
    flat[100] = 3.0
    narrow = 5.0 + 1e-6 * torch.randn(v, generator=g)
    narrow[::1000] = -20.0
    coarse = torch.round(torch.randn(v, generator=g)).to(torch.float32)
    rows, us, settings = [], [], []
    for x in (flat, narrow, coarse):
        for s in ((1.0, 5000, 1.0, 0.0), (1.0, 0, 0.7, 0.0), (0.3, 30000, 0.9, 0.0), (1.0, 2500, 0.5, 0.1), (20.0, 0, 0.5, 0.0)):
            for u in (0.1, 0.77):
                rows.append(x), us.append(u), settings.append(s)
    check(ctx, torch.stack(rows).cuda(), torch.tensor(us).cuda(), settings)


def test_infinities_nan_and_rows_of_nothing(ctx):
    v = 777
    g = torch.Generator().manual_seed(2)
    base = torch.randn(v, generator=g)
    masked = base.clone()
    masked[torch.rand(v, generator=g) < 0.9] = -float("inf")
    holes = base.clone()
    holes[::3] = float("nan")
    lowest = torch.full((v,), torch.finfo(torch.float32).min)
    lowest[5], lowest[700] = 1.0, 0.5
    tops = base.clone()
    tops[[40, 600]] = float("inf")
    one = torch.full((v,), -float("inf"))
    one[321] = -1e30
    rows = [masked, holes, lowest, tops, one]
    settings = [(1.0, 0, 1.0, 0.0), (0.9, 20, 0.9, 0.0), (1.0, 0, 0.99, 0.01), (0.0, 0, 1.0, 0.0)]
    for s in settings:
        for u in (0.0, 0.4, 0.99):
            check(ctx, torch.stack(rows).cuda(), torch.full((len(rows),), u).cuda(), [s] * len(rows))
    nothing = torch.stack([torch.full((v,), -float("inf")), torch.full((v,), float("nan")), base]).cuda()
    for t in (0.0, 1.0):
        got = ttq.sample(ctx, nothing, torch.full((3,), 0.5).cuda(), temperature=t, top_k=5)
        assert got[:2].tolist() == [-1, -1] and int(got[2]) >= 0


def test_one_setting_for_all_and_out(ctx):
    g = torch.Generator().manual_seed(3)
    logits, u = torch.randn(9, 3001, generator=g).cuda(), torch.rand(9, generator=g).cuda()
    out = torch.full((9,), -7, dtype=torch.int64, device="cuda")
    got = ttq.sample(ctx, logits, u, temperature=0.8, top_k=40, top_p=0.9, min_p=0.01, out=out)
    assert got is out
    assert torch.equal(got.cpu(), expect(logits, u, [(0.8, 40, 0.9, 0.01)] * 9))
    assert ttq.sample(ctx, logits[:0], u[:0]).numel() == 0
    # the same numbers again, and through a captured graph with other contents
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ttq.sample(ctx, logits, u, temperature=0.8, top_k=40, top_p=0.9, min_p=0.01, out=out)
    logits.copy_(torch.randn(9, 3001, generator=g))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), expect(logits, u, [(0.8, 40, 0.9, 0.01)] * 9))


@pytest.mark.parametrize("v", [3000, 20000])
def test_a_row_per_multiprocessor(ctx, v):
    """Batches large enough for one CTA per row, held in shared memory and not."""
    g = torch.Generator().manual_seed(v)
    m = 2 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    logits = (2.0 * torch.randn(m, v, generator=g)).cuda()
    check(ctx, logits, torch.rand(m, generator=g).cuda(), [SETTINGS[r % len(SETTINGS)] for r in range(m)])


def test_distribution(ctx):
    """Evenly spaced random numbers: every token comes up in proportion to its weight, to one draw."""
    n = 20000
    x = torch.tensor([1.0, -2.0, 0.5, 3.0, -1.0, 2.0, 2.0])
    u = ((torch.arange(n) + 0.5) / n).cuda()
    got = ttq.sample(ctx, x.expand(n, -1).cuda(), u, temperature=1.5, top_k=5)
    p = torch.softmax(torch.where(x >= 0.5, x, -float("inf")).double() / 1.5, 0)
    count = torch.bincount(got.cpu(), minlength=7)
    assert ((count - n * p).abs() <= 1.01).all()


def test_refusals(ctx):
    x, u = torch.randn(3, 100, device="cuda"), torch.rand(3, device="cuda")
    for status, args, kw in ((1, (x.cpu(), u), {}), (2, (x[0], u), {}), (2, (x, u[:2]), {}), (2, (x, u.double()), {}), (1, (x.double(), u), {}),
                             (2, (x, u), dict(top_k=torch.ones(2, dtype=torch.int32, device="cuda"))), (2, (x, u), dict(top_p=u.half())),
                             (2, (x, u), dict(out=torch.empty(3, dtype=torch.int32, device="cuda"))), (2, (x[:, :0], u), {}),
                             (7, (torch.zeros(1, (1 << 18) + 1, device="cuda"), u[:1]), {})):
        with pytest.raises(ttq.TtqError) as ei:
            ttq.sample(ctx, *args, **kw)
        assert ei.value.status == status, (ei.value, kw)
