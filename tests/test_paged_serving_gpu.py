"""The paged operators together, as a server runs them: prompts enter a shared cache, steps follow, tokens are drawn."""
import math

import numpy as np
import pytest
import torch

import tattletale_b200 as ttq
from paged_util import sample64
from tattletale_b200.decoder import DecoderConfig, DecoderStack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks,prefix", [(0, 0, 0), (48, 4, 0), (0, 0, 100), (64, 8, 100)])
def test_prompts_steps_and_sampling(ctx, window, sinks, prefix):
    """One attention layer with a linear in front and a vocabulary head behind, in 64 bits beside the kernels.  Sequences join with
    prompts of their own, one is served in two pieces, then all step together; pages come from one pool in the order of need.
    Every step is compared on the same inputs: the reference reads the 16-bit cache that the kernels wrote."""
    hq, hkv, d, page, vocab, hid = 8, 2, 64, 16, 997, 256
    dt = torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(window + prefix)
    w_qkv = torch.randn((hq + 2 * hkv) * d, hid, generator=g, device="cuda") / math.sqrt(hid)
    w_head = 0.3 * torch.randn(vocab, hq * d, generator=g, device="cuda")
    emb = torch.randn(vocab, hid, generator=g, device="cuda")
    qn, kn = ((1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in range(2))
    ang = torch.arange(512, device="cuda", dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    cos, sin = (torch.cat([f(ang), f(ang)], 1).float() for f in (torch.cos, torch.sin))
    prompts = [torch.randint(0, vocab, (n,), generator=g, device="cuda") for n in (5, 150, 33, 1)]
    pool = torch.randperm(200, generator=torch.Generator().manual_seed(1)).tolist()
    k_pages = torch.full((200, hkv, page, d), float("nan"), dtype=dt, device="cuda")
    v_pages = k_pages.clone()
    b = len(prompts)
    table = torch.full((b, 24), -1, dtype=torch.int32)
    have = [0] * b
    plan = ttq.PagedAttention(ctx, hq, hkv, d, page, max_seqs=b, max_tokens=256, dtype=dt)
    shared = torch.randint(0, vocab, (prefix,), generator=g, device="cuda")
    prefix_table = torch.tensor([pool.pop() for _ in range(-(-prefix // page))], dtype=torch.int32)

    def serve(pieces, pre):
        """pieces: token ids of every sequence (maybe none) -> attention results of all rows."""
        for s, ids in enumerate(pieces):
            have[s] += len(ids)
            while int((table[s] >= 0).sum()) * page < have[s]:
                table[s, int((table[s] >= 0).sum())] = pool.pop()
        ids = torch.cat(list(pieces))
        start = torch.tensor(np.cumsum([0] + [len(p) for p in pieces]), dtype=torch.int32)
        kv_len = torch.tensor([pre + n for n in have], dtype=torch.int32)
        batch = ttq.PagedBatch(start.cuda(), kv_len.cuda(), table.cuda(), max_q=max(len(p) for p in pieces), prefix_len=pre,
                               prefix_table=prefix_table.cuda() if pre else None)
        qkv = (emb[ids] @ w_qkv.T).to(dt)
        q = plan.append(qkv, k_pages, v_pages, batch, cos, sin, q_norm=qn, k_norm=kn)
        out = plan.forward(q, k_pages, v_pages, batch, window=window, sinks=sinks)
        ctx.check_device_status()
        # the keys of every position as the kernels stored them, against their own definition and as the reference's cache
        row = 0
        for s, piece in enumerate(pieces):
            n, total = len(piece), pre + have[s]
            if n == 0:
                continue
            at = torch.arange(have[s])
            pages, slots = table[s][at // page].long().cuda(), (at % page).cuda()
            k, v = k_pages[pages, :, slots].double(), v_pages[pages, :, slots].double()
            x = qkv[row:row + n].double().view(n, hq + 2 * hkv, d)
            xk = x[:, hq:hq + hkv]
            xk = xk / ((xk ** 2).mean(-1, keepdim=True) + 1e-6).sqrt() * kn.double()
            pos = torch.arange(total - n, total, device="cuda")
            turned = xk * cos[pos].double()[:, None] + torch.cat([-xk[..., d // 2:], xk[..., :d // 2]], -1) * sin[pos].double()[:, None]
            # one rounding to bf16 (2^-8 of the value), 32-bit arithmetic on terms no larger than a few units
            assert ((k[-n:] - turned).abs() <= 2.0 ** -8 * turned.abs() + 2.0 ** -18).all()
            if pre:
                at = torch.arange(pre)
                pages, slots = prefix_table[at // page].long().cuda(), (at % page).cuda()
                k, v = torch.cat([k_pages[pages, :, slots].double(), k]), torch.cat([v_pages[pages, :, slots].double(), v])
            k, v = (t.repeat_interleave(hq // hkv, 1) for t in (k, v))
            score = torch.einsum("nhd,jhd->hnj", q[row:row + n].double(), k) / math.sqrt(d)
            j = torch.arange(total, device="cuda")[None]
            seen = j <= pos[:, None]
            if window:
                seen &= (j > pos[:, None] - window) | (j < sinks)
            p = torch.softmax(torch.where(seen, score, -math.inf), -1)
            want = torch.einsum("hnj,jhd->nhd", p, v)
            # the weights' and the result's rounding to bf16, and 2^-10 for 32-bit scores of magnitude 2^4 (d * 2^-23 * sum |q k| * 2)
            bound = (2.0 ** -8 + 2.0 ** -10) * torch.einsum("hnj,jhd->nhd", p, v.abs()) + 2.0 ** -8 * want.abs() + 1e-6
            assert ((out[row:row + n].double() - want).abs() <= bound).all()
            row += n
        return out, start

    def next_tokens(out, start, step):
        last = out[(start[1:] - 1).long().cuda()].reshape(b, -1).float()
        logits = last @ w_head.T
        u = torch.rand(b, generator=g, device="cuda")
        settings = [(0.8, 40, 0.95, 0.0), (1.2, 0, 0.9, 0.01), (0.0, 0, 1.0, 0.0), (1.0, 5, 1.0, 0.0)]
        t = torch.tensor(settings)
        ids = ttq.sample(ctx, logits, u, temperature=t[:, 0].contiguous().cuda(), top_k=t[:, 1].int().cuda(), top_p=t[:, 2].contiguous().cuda(),
                         min_p=t[:, 3].contiguous().cuda())
        x = logits.cpu().numpy()
        f = t.numpy()
        assert ids.tolist() == [sample64(x[r], float(u[r]), f[r, 0], settings[r][1], f[r, 2], f[r, 3]) for r in range(b)]
        return ids

    none = torch.empty(0, dtype=torch.long, device="cuda")
    if prefix:  # the shared prefix enters the cache through the same calls, as a sequence whose pages become the prefix
        batch = ttq.PagedBatch(torch.tensor([0, prefix], dtype=torch.int32).cuda(), torch.tensor([prefix], dtype=torch.int32).cuda(), prefix_table[None].cuda(), max_q=prefix)
        plan.append((emb[shared] @ w_qkv.T).to(dt), k_pages, v_pages, batch, cos, sin, q_norm=qn, k_norm=kn)
    serve([prompts[0], prompts[1][:70], none, none], prefix)
    out, start = serve([torch.randint(0, vocab, (1,), generator=g, device="cuda"), prompts[1][70:], prompts[2], prompts[3]], prefix)
    for step in range(20):
        ids = next_tokens(out, start, step)
        out, start = serve([ids[s:s + 1] for s in range(b)], prefix)


def test_decoder_stack_samples(ctx):
    """``DecoderStack.step`` with random numbers draws from the logits that its greedy form takes the largest of."""
    cfg = DecoderConfig(n_layers=1, hidden=1024, n_q_heads=8, n_kv_heads=2, head_dim=128, ffn=1024, vocab=2048, context=128)
    stack = DecoderStack(ctx, cfg, batch=3)
    ids = torch.tensor([1, 500, 2047], device="cuda")
    greedy = stack.step(ids)
    u = torch.tensor([0.2, 0.5, 0.9], device="cuda")
    assert torch.equal(stack.step(ids, u, temperature=0.0), greedy)
    assert torch.equal(stack.step(ids, u, top_k=1), greedy)
    logits = stack.lm_head.forward(stack._step_fused(ids), out_dtype=torch.float32)
    got = stack.step(ids, u, temperature=1.5, top_k=50, top_p=0.9)
    x = logits.cpu().numpy()
    assert got.tolist() == [sample64(x[r], float(u[r]), np.float32(1.5), 50, np.float32(0.9), np.float32(0.0)) for r in range(3)]
