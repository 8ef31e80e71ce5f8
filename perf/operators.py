"""The measured cases of the operators around a paged key/value cache, and the operators in plain form.

What one pass runs, by the case's ``kind``:

  append  the rows that leave the fused qkv projection: per-head norm of q and k (where the model has one), the position
          rotation, k and v into the pages of their sequences, q out
  attend  causal attention of the batch's new tokens over their sequences' pages, optionally with a sliding window and a
          few first tokens that stay visible (sinks)
  prefix  the same for a batch whose sequences all start with one shared prefix, held once in the cache
  sample  the next token of every row of logits from given random numbers: temperature, top-k, top-p, min-p

A batch is ragged: sequence b brings ``q_start[b + 1] - q_start[b]`` new tokens, the last of its ``kv_len[b]`` tokens.  The
lengths of a case are spread over its ``[lo, hi]`` ranges by a fixed rule, pages are handed out in random order.  ``run``
computes the plain forms from elementary torch operations in 32 bits (the sampler, whose cuts lie between neighbouring
probabilities, in 64) or, where ``own`` is true, calls the framework.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
THETA = 500000.0

_context = None


def context():
    """One library context per process, as a serving process keeps."""
    global _context
    if _context is None:
        import tattletale_b200 as ttq
        _context = ttq.Context(0)
    return _context


def _batch(kind, seqs, new, past, heads, d, page, dtype, **more):
    return {"kind": kind, "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "hq": heads[0],
            "hkv": heads[1], "d": d, "page": page, "dtype": dtype, "window": more.get("window", 0), "sinks": more.get("sinks", 0),
            "prefix": more.get("prefix", 0), "norm": more.get("norm", False)}


def listed():
    cases = [
        # three users decoding: the append is a launch and little else
        ("append-step-3", _batch("append", 3, (1, 1), (100, 2000), (32, 8), 128, 16, "bf16")),
        # two prompts entering the cache of a model that normalises q and k per head
        ("append-prompt-2", _batch("append", 2, (3501, 4600), (0, 700), (32, 8), 128, 64, "f16", norm=True)),
        # one user decoding in a short chat
        ("attend-step-1", _batch("attend", 1, (1, 1), (1530, 1530), (32, 8), 128, 16, "bf16")),
        # a server's continuous batch with chats of all lengths
        ("attend-step-64", _batch("attend", 64, (1, 1), (17, 16000), (32, 8), 128, 16, "bf16")),
        # long chats through the windowed layers of a model that keeps its first tokens in sight
        ("attend-window-step-23", _batch("attend", 23, (1, 1), (900, 33000), (64, 8), 64, 32, "f16", window=4096, sinks=4)),
        # a few prompts, the longest of several thousand tokens
        ("attend-prompt-3", _batch("attend", 3, (1111, 4300), (0, 0), (32, 8), 128, 64, "bf16")),
        # a piece of a long prompt through a windowed layer, behind what is cached of it
        ("attend-window-chunk-2", _batch("attend", 2, (2000, 2049), (9000, 12000), (40, 8), 128, 16, "bf16", window=2048, sinks=8)),
        # many users behind one system prompt, decoding
        ("prefix-step-48", _batch("prefix", 48, (1, 1), (5, 700), (32, 8), 128, 16, "bf16", prefix=12345)),
        # questions of a sentence or two asked about one long document
        ("prefix-questions-9", _batch("prefix", 9, (11, 75), (0, 0), (28, 4), 128, 32, "f16", prefix=24000)),
        # the next token of one chat
        ("sample-1", {"kind": "sample", "rows": 1, "vocab": 128256, "dtype": "f32"}),
        # a continuous batch, every user with settings of their own, logits as a 16-bit vocabulary head leaves them
        ("sample-37", {"kind": "sample", "rows": 37, "vocab": 32001, "dtype": "bf16"}),
        # a large batch over a large vocabulary
        ("sample-256", {"kind": "sample", "rows": 256, "vocab": 128256, "dtype": "f32"}),
    ]
    return [{"name": name, **case} for name, case in cases]


# ---- drawn cases ---------------------------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _range(rng, lo, hi):
    a, b = _log(rng, lo, hi), _log(rng, lo, hi)
    return (min(a, b), max(a, b))


def draw(rng):
    """One more case: from a few rows to long prompts, lengths and batch sizes log-uniform."""
    kind = rng.choice(["append", "attend", "attend", "attend", "prefix", "prefix", "sample"])
    if kind == "sample":
        case = {"kind": kind, "rows": _log(rng, 1, 256), "vocab": _log(rng, 1000, 160000), "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}
    else:
        hkv = rng.choice([1, 2, 4, 8])
        heads = (hkv * rng.choice([1, 2, 3, 4, 5, 7, 8]), hkv)
        more = {"norm": kind == "append" and rng.random() < 0.5}
        if kind == "prefix":
            more["prefix"] = _log(rng, 200, 30000)
        if kind != "append" and rng.random() < 0.4:
            more.update(window=_log(rng, 30, 6000), sinks=rng.choice([0, 1, 4, 64]))
        if rng.random() < 0.5:  # a decode step
            seqs, new, past = _log(rng, 1, 200), (1, 1), _range(rng, 1, 20000 if kind != "prefix" else 2000)
        else:
            seqs, new, past = _log(rng, 1, 16), _range(rng, 2, 4000 if kind != "prefix" else 200), rng.choice([(0, 0), _range(rng, 1, 12000)])
        case = _batch(kind, seqs, new, past, heads, rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["bf16", "f16"]), **more)
    # no dearer than the dearest listed case of the kind, on the roofline and in plain form: fewer rows, then shorter ones
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while _cost(case) > most:
        if kind == "sample":
            case["rows"] = case["rows"] * 2 // 3
        elif case["seqs"] > 1:
            case["seqs"] = case["seqs"] * 2 // 3
        else:
            for key in ("new_lo", "new_hi"):
                case[key] = max(1, case[key] * 2 // 3)
            for key in ("past_lo", "past_hi", "prefix"):
                case[key] = case[key] * 2 // 3
    return case


def _cost(case):
    w = work(case)
    if case["kind"] in ("sample", "append"):
        return w["bytes"]
    new, past = _lengths(case)  # the plain form computes every score, masked ones too
    scores = sum(n * (n + p + case["prefix"]) for n, p in zip(new, past)) * case["hq"] * case["d"]
    return max(w["bytes"] / 6e12, w["flops"] / 6e14, scores / 1e14)


# ---- a case's lengths and its work ---------------------------------------------------------------------------------

def _spread(lo, hi, n, step):
    """n lengths over [lo, hi], both ends among them where n > 1, in no particular order."""
    if n == 1:
        return [hi]
    return [lo + round((hi - lo) * i / (n - 1)) for i in sorted(range(n), key=lambda i: i * step % 1.0)]


def _lengths(c):
    """New tokens and cached own tokens (behind any shared prefix) of every sequence."""
    return _spread(c["new_lo"], c["new_hi"], c["seqs"], 0.618034), _spread(c["past_lo"], c["past_hi"], c["seqs"], 0.754878)


def _visible(c, pos):
    """How many keys a token at position pos sees."""
    if not c["window"] or pos < c["window"]:
        return pos + 1
    return c["window"] + min(c["sinks"], pos + 1 - c["window"])


def work(case):
    c = case
    if c["kind"] == "sample":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["rows"] * (c["vocab"] * size + 4 * 5 + 8), "flops": 4 * c["rows"] * c["vocab"]}
    new, past = _lengths(c)
    hq, hkv, d, t = c["hq"], c["hkv"], c["d"], sum(new)
    if c["kind"] == "append":
        row = (hq + 2 * hkv) * d
        return {"bytes": 2 * 2 * t * row + 2 * 4 * d * t, "flops": 3 * t * (hq + hkv) * d}
    keys = own_keys = pairs = 0
    prefix_first = c["prefix"]  # first prefix position behind the sinks that any token sees
    for n, p in zip(new, past):
        first = p + c["prefix"]
        pairs += sum(_visible(c, pos) for pos in range(first, first + n))
        lo = max(0, first - c["window"] + 1) if c["window"] else 0
        prefix_first = min(prefix_first, lo)
        own_keys += first + n - max(c["prefix"], lo) + max(0, min(c["sinks"], lo) - c["prefix"])
    if c["prefix"]:
        keys = c["prefix"] - prefix_first + min(c["sinks"], prefix_first)
    keys += own_keys
    return {"bytes": 2 * (2 * keys * hkv * d + 2 * t * hq * d), "flops": 4 * pairs * hq * d}


# ---- states --------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": dict(c)}
    if c["kind"] == "sample":
        m, v = c["rows"], c["vocab"]
        # a broad bulk with a handful of likely tokens above it
        logits = 2.0 * randn(m, v)
        likely = torch.randint(0, v, (m, 40), generator=gen, device="cuda")
        logits.scatter_add_(1, likely, 6.0 + 3.0 * randn(m, 40))
        s["logits"] = logits.to(DTYPES[c["dtype"]])
        s["u"] = torch.rand(m, generator=gen, device="cuda")
        # every user's own settings: plain sampling, nucleus, short lists, greedy
        pick = torch.randint(0, 6, (m,), generator=gen, device="cuda")
        table = torch.tensor([[1.0, 0, 1.0, 0.0], [0.7, 0, 0.95, 0.0], [0.8, 50, 0.9, 0.0], [1.3, 1000, 1.0, 0.02], [0.0, 0, 1.0, 0.0],
                              [1.1, 0, 0.99, 0.001]], device="cuda")[pick]
        s["temperature"], s["top_p"], s["min_p"] = (table[:, i].contiguous() for i in (0, 2, 3))
        s["top_k"] = table[:, 1].to(torch.int32)
        return s
    dt = DTYPES[c["dtype"]]
    new, past = _lengths(c)
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    s["new"], s["kv"] = new, [c["prefix"] + p + n for n, p in zip(new, past)]
    own_pages = [-(-(p + n) // page) for n, p in zip(new, past)]
    prefix_pages = -(-c["prefix"] // page)
    total = sum(own_pages) + prefix_pages + 3  # a few pages belong to nobody
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    rows = torch.full((c["seqs"], max(own_pages)), -1, dtype=torch.int32)
    at = torch.cumsum(torch.tensor([0] + own_pages), 0).tolist()
    host = order.cpu()
    for b, n in enumerate(own_pages):
        rows[b, :n] = host[at[b]:at[b] + n]
    s["block_table"] = rows.cuda()
    s["prefix_table"] = order[at[-1]:at[-1] + prefix_pages].contiguous() if prefix_pages else None
    s["q_start"] = torch.cumsum(torch.tensor([0] + new), 0).to(torch.int32).cuda()
    s["kv_len"] = torch.tensor(s["kv"], dtype=torch.int32).cuda()
    s["k_pages"] = randn(total, hkv, page, d).to(dt)
    s["v_pages"] = randn(total, hkv, page, d).to(dt)
    t = sum(new)
    if c["kind"] == "append":
        spread = torch.exp(0.3 * randn((hq + 2 * hkv) * d))
        s["qkv"] = (randn(t, (hq + 2 * hkv) * d) * spread).to(dt)
        ang = torch.arange(max(s["kv"]), device="cuda", dtype=torch.float64)[:, None] / THETA ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        s["cos"], s["sin"] = (torch.cat([f(ang), f(ang)], 1).float() for f in (torch.cos, torch.sin))
        s["q_norm"], s["k_norm"] = ((1 + 0.1 * randn(d)).to(dt) if c["norm"] else None for _ in range(2))
    else:
        s["q"] = (1.5 * randn(t, hq, d)).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] != "sample":
        import tattletale_b200 as ttq
        c = case
        s["paged"] = ttq.PagedAttention(context(), c["hq"], c["hkv"], c["d"], c["page"], max_seqs=c["seqs"], max_tokens=sum(s["new"]),
                                        dtype=DTYPES[c["dtype"]])
        s["batch"] = ttq.PagedBatch(s["q_start"], s["kv_len"], s["block_table"], max_q=max(s["new"]), prefix_len=c["prefix"],
                                    prefix_table=s["prefix_table"])
    elif own:
        context()
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state, kind)
    return {"append": _append, "attend": _attend, "prefix": _attend, "sample": _sample}[kind](state)


def _run_own(s, kind):
    import tattletale_b200 as ttq
    c = s["case"]
    if kind == "sample":
        return ttq.sample(context(), s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    if kind == "append":
        q = s["paged"].append(s["qkv"], s["k_pages"], s["v_pages"], s["batch"], s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
        return [q, s["k_pages"], s["v_pages"]]
    return s["paged"].forward(s["q"], s["k_pages"], s["v_pages"], s["batch"], window=c["window"], sinks=c["sinks"])


def _append(s):
    c = s["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    t = s["qkv"].shape[0]
    token = torch.arange(t, device="cuda", dtype=torch.int32)
    seq = (token[:, None] >= s["q_start"][None, 1:]).sum(1)
    pos = (s["kv_len"][seq] - (s["q_start"][seq + 1] - token)).long()
    x = s["qkv"].float().view(t, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], s["qkv"].view(t, hq + 2 * hkv, d)[:, hq + hkv:]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def turned(h, weight):
        if weight is not None:
            h = h * torch.rsqrt((h * h).sum(-1, keepdim=True) / d + EPS) * weight.float()
        return (h * cos + torch.cat([-h[..., d // 2:], h[..., :d // 2]], -1) * sin).to(s["qkv"].dtype)

    own_pos = pos - c["prefix"]
    at = s["block_table"][seq, own_pos // page].long()
    s["k_pages"][at, :, own_pos % page] = turned(k, s["k_norm"])
    s["v_pages"][at, :, own_pos % page] = v
    return [turned(q, s["q_norm"]), s["k_pages"], s["v_pages"]]


def _attend(s):
    c = s["case"]
    hq, hkv, d, page, pre = c["hq"], c["hkv"], c["d"], c["page"], c["prefix"]
    out = torch.empty_like(s["q"])
    first = 0
    for b, (n, total) in enumerate(zip(s["new"], s["kv"])):
        keys = []
        for pages in (s["k_pages"], s["v_pages"]):
            table = s["block_table"][b, :-(-(total - pre) // page)]
            rows = pages[table.long()].transpose(0, 1).reshape(hkv, -1, d)[:, :total - pre]
            if pre:
                shared = pages[s["prefix_table"].long()].transpose(0, 1).reshape(hkv, -1, d)[:, :pre]
                rows = torch.cat([shared, rows], 1)
            keys.append(rows)
        pos = torch.arange(total - n, total, device="cuda")[:, None]
        j = torch.arange(total, device="cuda")[None]
        seen = j <= pos
        if c["window"]:
            seen = seen & ((j > pos - c["window"]) | (j < c["sinks"]))
        seen = seen.repeat_interleave(hq // hkv, 0)
        q = s["q"][first:first + n].view(n, hkv, hq // hkv, d)
        step = hkv if n * hq * total <= 1 << 28 else 1  # all kv heads at once where their scores stay small
        for h in range(0, hkv, step):
            qh = q[:, h:h + step].transpose(0, 1).reshape(step, -1, d).float()
            score = (qh @ keys[0][h:h + step].float().transpose(1, 2)) / math.sqrt(d)
            score = torch.where(seen, score, -math.inf)
            e = torch.exp(score - score.amax(-1, keepdim=True))
            o = (e @ keys[1][h:h + step].float()) / e.sum(-1, keepdim=True)
            out[first:first + n].view(n, hkv, hq // hkv, d)[:, h:h + step] = o.view(step, n, hq // hkv, d).transpose(0, 1).to(out.dtype)
        first += n
    return out


def _sample(s):
    t = s["temperature"].double()[:, None]
    x = s["logits"].double()
    m, v = x.shape
    order_x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    z = order_x / torch.where(t > 0, t, 1.0)
    e = torch.exp(z - z[:, :1])
    rank = torch.arange(v, device="cuda")[None]
    k = s["top_k"].long()[:, None]
    keep = (rank < k) | (k <= 0)
    mass = torch.cumsum(torch.where(keep, e, 0.0), -1)
    # the shortest run of the likeliest tokens that holds top_p of the mass: a token stays while those before it hold less
    keep = keep & ((mass - e < s["top_p"].double()[:, None] * mass[:, -1:]) | (s["top_p"][:, None] >= 1) | (rank == 0))
    keep = keep & (e >= s["min_p"].double()[:, None])
    keep = torch.where(t > 0, keep, rank == 0)
    weight = torch.zeros_like(x).scatter_(1, order, torch.where(keep, e, 0.0))
    cdf = torch.cumsum(weight, -1)
    # the first token, in the order of the vocabulary, whose cumulative weight exceeds u of the whole
    return (cdf <= s["u"].double()[:, None] * cdf[:, -1:]).sum(-1)


# ---- the results in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "prefix": _exact_attend, "sample": _exact_sample}[case["kind"]](s)


def _exact_append(s):
    c = s["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    qs, ks, vs = s["qkv"].double().split([hq * d, hkv * d, hkv * d], 1)
    kc, vc, out = s["k_pages"].double(), s["v_pages"].double(), torch.empty(qs.shape[0], hq, d, dtype=torch.float64, device="cuda")

    def rotate(x, weight, pos):
        if weight is not None:
            x = x / ((x ** 2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
        cos, sin = s["cos"].double()[pos][:, None, :], s["sin"].double()[pos][:, None, :]
        a, b = x.chunk(2, -1)
        ca, cb = cos.chunk(2, -1)
        sa, sb = sin.chunk(2, -1)
        return torch.cat([a * ca - b * sa, b * cb + a * sb], -1)

    first = 0
    for b, (n, total) in enumerate(zip(s["new"], s["kv"])):
        rows = slice(first, first + n)
        pos = torch.arange(total - n, total, device="cuda")
        slot = pos - c["prefix"]
        pages = s["block_table"][b][slot // page].long()
        out[rows] = rotate(qs[rows].view(n, hq, d), s["q_norm"], pos)
        kc[pages, :, slot % page] = rotate(ks[rows].view(n, hkv, d), s["k_norm"], pos)
        vc[pages, :, slot % page] = vs[rows].view(n, hkv, d)
        first += n
    return [out, kc, vc]


def _exact_attend(s):
    c = s["case"]
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    group = hq // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["seqs"]):
        total = s["kv"][b]
        where = torch.arange(total - c["prefix"], device="cuda")
        page_of, in_page = s["block_table"][b][where // page].long(), where % page
        if c["prefix"]:
            where = torch.arange(c["prefix"], device="cuda")
            page_of = torch.cat([s["prefix_table"][where // page].long(), page_of])
            in_page = torch.cat([where % page, in_page])
        end = sum(s["new"][:b + 1])
        for h in range(hkv):
            k, v = s["k_pages"][page_of, h, in_page].double(), s["v_pages"][page_of, h, in_page].double()
            for r in range(end - s["new"][b], end, 512):  # blocks of query tokens
                r1 = min(r + 512, end)
                pos = total - end + torch.arange(r, r1, device="cuda")
                dist = pos[:, None] - torch.arange(total, device="cuda")[None]
                hidden = dist < 0
                if c["window"]:
                    hidden |= (dist >= c["window"]) & (torch.arange(total, device="cuda")[None] >= c["sinks"])
                x = torch.einsum("tgd,jd->tgj", s["q"][r:r1, h * group:(h + 1) * group].double(), k) * d ** -0.5
                x.masked_fill_(hidden[:, None], -math.inf)
                lse = torch.logsumexp(x, -1, keepdim=True)
                out[r:r1, h * group:(h + 1) * group] = torch.einsum("tgj,jd->tgd", torch.exp(x - lse), v)
    return out


def _exact_sample(s):
    logits, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    temperature, top_p, min_p = (s[key].double().cpu().numpy() for key in ("temperature", "top_p", "min_p"))
    top_k = s["top_k"].cpu().numpy()
    ids = np.empty(len(u), dtype=np.int64)
    for r, x in enumerate(logits):
        if temperature[r] <= 0:
            ids[r] = np.argmax(x)
            continue
        w = np.exp((x - x.max()) / temperature[r])
        by = np.argsort(-x, kind="stable")
        if top_k[r] > 0:
            by = by[:top_k[r]]
        if top_p[r] < 1:
            by = by[:np.searchsorted(np.cumsum(w[by]), top_p[r] * w[by].sum()) + 1]
        by = by[w[by] >= min_p[r]]
        kept = np.zeros_like(w)
        kept[by] = w[by]
        ids[r] = np.searchsorted(np.cumsum(kept), u[r] * kept.sum(), side="right")
    return torch.from_numpy(ids)
