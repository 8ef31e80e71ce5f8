"""Plain statements, in 64 bits, of the paged operators and the sampler, and batches to run them on."""
import math

import numpy as np
import torch

import tattletale_b200 as ttq


class Batch:
    """A ragged batch over randomly handed out pages.  ``lens``: (new tokens, own tokens cached before them) per sequence.  Everything
    that no token may see -- slots behind a sequence's end, pages of nobody -- is NaN."""

    def __init__(self, lens, hq, hkv, d, page, dtype, prefix=0, seed=0, layout="hnd", pad_rows=0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hq, self.hkv, self.d, self.page, self.dtype, self.prefix = lens, hq, hkv, d, page, dtype, prefix
        own = [-(-(n + p) // page) for n, p in lens]
        npre = -(-prefix // page)
        total = sum(own) + npre + spare
        order = torch.randperm(total, generator=g).to(torch.int32)
        table = torch.full((len(lens), max(own + [1])), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(own):
            table[b, :n] = order[at:at + n]
            at += n
        self.table_host, self.prefix_host = table, order[at:at + npre]
        self.n_pages = total
        shape = {"hnd": (total, hkv, page, d), "nhd": (total, page, hkv, d), "joint": (total, 2, hkv, page, d)}[layout]
        k = torch.randn(shape, generator=g)
        v = torch.randn(shape, generator=g)
        if layout == "nhd":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        elif layout == "joint":  # k and v of a page side by side in one allocation
            both = k.to(dtype).cuda()
            k, v = both[:, 0], both[:, 1]
        self.k, self.v = (k, v) if layout == "joint" else ((x.transpose(1, 2).to(dtype).cuda().transpose(1, 2) if layout == "nhd" else x.to(dtype).cuda()) for x in (k, v))
        valid = torch.zeros(total, page, dtype=torch.bool)
        for b, (n, p) in enumerate(lens):
            for i in range(n + p):
                valid[table[b, i // page], i % page] = True
        for i in range(prefix):
            valid[self.prefix_host[i // page], i % page] = True
        bad = ~valid.cuda()[:, None, :, None].expand(total, hkv, page, d)
        self.k[bad] = float("nan")
        self.v[bad] = float("nan")
        new = [n for n, _ in lens]
        self.rows = sum(new)
        self.q_start = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
        self.kv_len = torch.tensor([prefix + n + p for n, p in lens], dtype=torch.int32).cuda()
        self.q = torch.randn(self.rows + pad_rows, hq, d, generator=g).to(dtype).cuda()
        self.table = table.cuda()

    def batch(self, max_q=None):
        return ttq.PagedBatch(self.q_start, self.kv_len, self.table, max_q=max((n for n, _ in self.lens), default=0) if max_q is None else max_q,
                              prefix_len=self.prefix, prefix_table=self.prefix_host.cuda() if self.prefix else None)

    def plan(self, ctx, **more):
        return ttq.PagedAttention(ctx, self.hq, self.hkv, self.d, self.page, max_seqs=max(1, len(self.lens)), max_tokens=max(1, self.q.shape[0]),
                                  dtype=self.dtype, **more)

    def keys(self, b):
        """k and v of sequence b, in 64 bits: [kv heads, tokens, d]."""
        n, p = self.lens[b]
        pos = torch.arange(n + p)
        pages, slots = self.table_host[b][pos // self.page].long(), pos % self.page
        if self.prefix:
            pos = torch.arange(self.prefix)
            pages, slots = torch.cat([self.prefix_host[pos // self.page].long(), pages]), torch.cat([pos % self.page, slots])
        return tuple(x[pages.cuda(), :, slots.cuda()].double().transpose(0, 1) for x in (self.k, self.v))


def attention64(bt, window=0, sinks=0, scale=None):
    """The batch's result in 64 bits and a bound for the kernel's error, both [rows, hq, d].

    The bound: the softmax weights and the result are rounded to the 16-bit type (half a step u each, relative), and a score is
    a 32-bit sum of d products, off by at most d * 2^-23 * sum |q k| in units of its own (a truncating accumulator loses one step
    per addition), which moves every weight by that relative amount in numerator and denominator; 2^-18 stands for the
    exponentials (2 ulp), the running rescale and the 32-bit sums of the weights."""
    u = torch.finfo(bt.dtype).eps / 2
    scale = 1 / math.sqrt(bt.d) if scale is None else scale
    want = torch.zeros(bt.rows, bt.hq, bt.d, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    group, row = bt.hq // bt.hkv, 0
    for b, (n, p) in enumerate(bt.lens):
        if n == 0:
            continue
        total = bt.prefix + n + p
        k, v = bt.keys(b)
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        q = bt.q[row:row + n].double().transpose(0, 1)
        pos, j = torch.arange(total - n, total, device="cuda")[:, None], torch.arange(total, device="cuda")[None]
        seen = j <= pos
        if window:
            seen = seen & ((j > pos - window) | (j < sinks))
        s = torch.where(seen, q @ k.transpose(1, 2) * scale, -math.inf)
        w = torch.softmax(s, -1)
        o = (w @ v).transpose(0, 1)
        spread = (w @ v.abs()).transpose(0, 1)
        err_s = bt.d * 2.0 ** -23 * scale * torch.where(seen, q.abs() @ k.abs().transpose(1, 2), 0.0).amax(-1)
        want[row:row + n] = o
        bound[row:row + n] = spread * (u + 2 * err_s.transpose(0, 1)[..., None] + 2.0 ** -18) + o.abs() * u + 1e-7
        row += n
    return want, bound


def check_attention(got, bt, window=0, sinks=0, scale=None):
    want, bound = attention64(bt, window, sinks, scale)
    got = got[:bt.rows].double()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / bound).max().item()
    assert over <= 1, f"error {over:.2f} times the bound"


def sample64(x, u, temperature, top_k, top_p, min_p):
    """One row's token from the definition (numpy, 64 bits)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.argmax(x))
    w = np.where(x == top, 1.0, np.exp((x - top) / np.float64(temperature)) if np.isfinite(top) else 0.0)
    by = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        by = by[:top_k]
    if top_p < 1:
        cum = np.cumsum(w[by])
        by = by[:np.searchsorted(cum, np.float64(max(top_p, 0.0)) * cum[-1]) + 1]
    by = by[(w[by] >= np.float64(min_p)) | (w[by] == 1.0)]
    kept = np.zeros_like(w)
    kept[by] = w[by]
    return int(np.searchsorted(np.cumsum(kept), np.float64(u) * kept.sum(), side="right"))
