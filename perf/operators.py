"""Operators of a serving step that continues sequences held in the paged pool.

Three kinds of call:

* ``chunk``   attention of a chunk of new tokens over a paged cache: a long prompt prefilled
              piece by piece, a prompt whose beginning is cached already, the drafted tokens
              of speculative decoding; rows of a batch with their own lengths;
* ``scored``  the same with capped scores (``cap * tanh(s / cap)``), a distance bias per head,
              a sliding window and a prefix that every token sees, for chunks and for single
              tokens;
* ``norm``    the addition of a block's output to the residual stream and the RMSNorm of the
              sum, which gives both.

Query token t of row b stands at position ``start[b] + t``; it sees the positions up to its own
that are less than ``window`` before it, and those below ``prefix[b]``.  Tokens at or past the
row's length give zeros.  With ``own`` unset the operators run as elementary torch operations.
"""

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
LAYOUTS = [(24, 8, 128), (32, 8, 128), (8, 1, 128), (16, 16, 64), (14, 2, 64), (12, 4, 96)]
MOST_PAIRS = 2 * 2048 * 15360 * 24 * 128   # new tokens x context x heads x width of a case
MOST_CACHE = 2 * 16384 * 8 * 128 * 4       # cached tokens x heads x width of a case
MOST_NORM = 16384 * 5120                   # rows x width of a norm case


def listed():
    return [
        # drafted tokens of one conversation, verified at once: latency counts
        _chunk("chunk_verify_b1", 1, 4, 1024, 1024, (24, 8, 128), 64),
        # the same on a loaded server: odd draft length, a length per conversation, small blocks
        _chunk("chunk_verify_b24", 24, 5, 300, 4096, (24, 8, 128), 16),
        # the last piece of a long prompt that is prefilled in pieces of 512 tokens
        _chunk("chunk_512_of_8192", 1, 512, 8192, 8192, (24, 8, 128), 64),
        # continued conversations: rows with their own number of new tokens and contexts
        _chunk("chunk_ragged_b6", 6, 333, 500, 6000, (32, 8, 128), 32, ragged_new=True),
        # two long documents in large pieces: the largest call
        _chunk("chunk_2048_of_16384", 2, 2048, 16384, 16384, (24, 8, 128), 64),
        # one decode step of a model with capped scores, on a loaded server
        _chunk("scored_cap_decode_b32", 32, 1, 512, 4096, (24, 8, 128), 64, cap=50.0),
        # one decode step of a model with a distance bias and no shared heads, long context
        _chunk("scored_bias_decode_b2", 2, 1, 9001, 20011, (16, 16, 64), 64, bias=True),
        # a piece of a prompt in a layer with capped scores and a sliding window
        _chunk("scored_cap_window_b2", 2, 1000, 5000, 5000, (32, 8, 128), 64, cap=50.0, window=1024),
        # prompts whose image or instruction tokens see each other, with the distance bias
        _chunk("scored_prefix_b3", 3, 777, 777, 777, (14, 2, 64), 64, bias=True, prefix=256),
        # the residual stream of one token
        {"name": "norm_1x4096", "kind": "norm", "rows": 1, "width": 4096},
        # a decode batch beside a short prompt, odd rows
        {"name": "norm_777x2560", "kind": "norm", "rows": 777, "width": 2560},
        # the prompts of a prefill step
        {"name": "norm_16384x5120", "kind": "norm", "rows": 16384, "width": 5120},
    ]


def _chunk(name, batch, new, low, high, layout, block, ragged_new=False, cap=0.0, bias=False,
           window=0, prefix=0):
    hq, hkv, d = layout
    scored = cap > 0 or bias or window > 0 or prefix > 0
    return {"name": name, "kind": "scored" if scored else "chunk", "batch": batch, "new": new,
            "low": low, "high": high, "hq": hq, "hkv": hkv, "d": d, "block": block,
            "ragged_new": ragged_new, "cap": cap, "bias": bias, "window": window,
            "prefix": prefix}


def _log(rng, low, high):
    """An integer from low to high, spread evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "scored", "scored", "norm"])
    if kind == "norm":
        width = 8 * _log(rng, 32, 1024)
        return {"kind": kind, "rows": _log(rng, 1, min(16384, MOST_NORM // width)), "width": width}
    hq, hkv, d = layout = rng.choice(LAYOUTS)
    new = 1 if kind == "scored" and rng.random() < 0.4 else _log(rng, 2, 2048)
    high = _log(rng, max(new, 64), 20011 if new == 1 else 16384)
    low = _log(rng, max(new, min(64, high)), high) if rng.random() < 0.7 else high
    batch = _log(rng, 1, 32)
    while batch > 1 and (batch * new * high * hq * d > MOST_PAIRS
                         or batch * high * hkv * d > MOST_CACHE):
        batch -= 1
    c = _chunk("", batch, new, low, high, layout, rng.choice([8, 16, 24, 32, 64, 64, 128]),
               ragged_new=new > 1 and rng.random() < 0.5)
    if kind == "scored":
        while c["kind"] == "chunk":
            c = _chunk("", batch, new, low, high, layout, c["block"], c["ragged_new"],
                       cap=rng.choice([0.0, 20.0, 30.0, 50.0]), bias=rng.random() < 0.5,
                       window=rng.choice([0, _log(rng, 16, 4096)]),
                       prefix=rng.choice([0, 0, _log(rng, 1, low)]))
    del c["name"]
    return c


# -- inputs ------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g, dtype=torch.float16)


def _sizes(case):
    """(contexts, start positions, prefixes) of the rows: a property of the case, so that its
    work is the same for every seed."""
    batch, new, low, high = case["batch"], case["new"], case["low"], case["high"]
    r = torch.Generator().manual_seed(1000003 * batch + 1009 * high + 31 * low + new)
    lens = torch.randint(low, high + 1, (batch,), generator=r).tolist()
    lens[0] = high
    count = [new] * batch
    if case["ragged_new"]:
        count = torch.randint(1, new + 1, (batch,), generator=r).tolist()
        count[0] = new
    pre = [0] * batch
    if case["prefix"]:
        pre = torch.randint(0, case["prefix"] + 1, (batch,), generator=r).tolist()
        pre[0] = case["prefix"]
    return lens, [n - c for n, c in zip(lens, count)], pre


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "norm":
        m, n = case["rows"], case["width"]
        return {"kind": "norm", "x": _randn(g, m, n), "residual": _randn(g, m, n) * 3,
                "weight": 1 + 0.1 * _randn(g, n)}
    lens, starts, pre = _sizes(case)
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    counts = [-(-n // block) for n in lens]
    perm = torch.randperm(sum(counts), device=DEV, generator=g).int()
    table = torch.full((case["batch"], max(counts)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = perm[at:at + n]
        at += n
    i32 = dict(dtype=torch.int32, device=DEV)
    s = {"kind": case["kind"], "lens": lens, "starts": starts, "prefix": pre, "block": block,
         "table": table, "kc": _randn(g, at, block, hkv, d), "vc": _randn(g, at, block, hkv, d),
         # scores of a model that caps them spread wider
         "q": _randn(g, case["batch"], case["new"], hq, d) * (3 if case["cap"] else 1),
         "scale": d ** -0.5, "cap": case["cap"], "window": case["window"], "slopes": None,
         "d_starts": torch.tensor(starts, **i32), "d_lens": torch.tensor(lens, **i32),
         "d_prefix": torch.tensor(pre, **i32) if case["prefix"] else None}
    if case["bias"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV, dtype=torch.float32) / hq)
    if own:
        import fast_infer_amd as fi

        s["ws"] = fi.paged_chunk_attention_workspace(case["batch"], case["new"], hq, hkv, max(lens),
                                                     d, DEV)
    return s


# -- one pass ------------------------------------------------------------------------------

def run(state):
    s = state
    if own:
        import fast_infer_amd as fi

        if s["kind"] == "norm":
            return fi.add_rms_norm(s["x"], s["residual"], s["weight"], EPS)
        return fi.paged_chunk_attention(
            s["q"], s["kc"], s["vc"], s["table"], s["block"], max(s["lens"]), s["scale"],
            start_positions=s["d_starts"], context_lens=s["d_lens"], softcap=s["cap"] or None,
            alibi_slopes=s["slopes"], window=s["window"] or None, prefix_lens=s["d_prefix"],
            workspace=s["ws"])
    if s["kind"] == "norm":
        h = (s["x"].float() + s["residual"].float()).half()
        f = h.float()
        r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
        return (f * r * s["weight"].float()).half(), h
    q, block = s["q"], s["block"]
    batch, new, hq, d = q.shape
    hkv = s["kc"].shape[2]
    out = torch.zeros_like(q)
    for b in range(batch):
        n, start, pre = s["lens"][b], s["starts"][b], s["prefix"][b]
        cnt = n - start
        pos = torch.arange(n, device=DEV)
        slot = s["table"][b, pos // block].long() * block + pos % block
        k = s["kc"].view(-1, hkv, d)[slot].float().permute(1, 2, 0).contiguous()   # [hkv, d, n]
        v = s["vc"].view(-1, hkv, d)[slot].float().transpose(0, 1).contiguous()    # [hkv, n, d]
        qb = q[b, :cnt].float().view(cnt, hkv, hq // hkv, d).permute(1, 2, 0, 3)
        x = torch.bmm(qb.reshape(hkv, -1, d), k).view(hq, cnt, n) * s["scale"]
        if s["cap"]:
            x = s["cap"] * torch.tanh(x / s["cap"])
        dist = (start + torch.arange(cnt, device=DEV)).view(-1, 1) - pos           # [cnt, n]
        if s["slopes"] is not None:
            x = x - s["slopes"].view(-1, 1, 1) * dist.abs().float()
        see = dist >= 0
        if s["window"]:
            see = see & (dist < s["window"])
        if pre:
            see = see | (pos < pre)
        x = torch.where(see, x, torch.full_like(x, -math.inf))
        p = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.bmm(p.view(hkv, -1, n), v).view(hq, cnt, d) / p.sum(-1, keepdim=True)
        out[b, :cnt] = o.transpose(0, 1).half()
    return out


# -- what a pass cannot do without ---------------------------------------------------------

def work(case):
    if case["kind"] == "norm":
        m, n = case["rows"], case["width"]
        return {"bytes": 2 * (4 * m * n + n), "flops": 5 * m * n}
    lens, starts, pre = _sizes(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    pairs = keys = tokens = 0
    for n, start, p in zip(lens, starts, pre):
        w = case["window"] or n
        pairs += sum(max(0, min(w, t + 1, t + 1 - p)) + p for t in range(start, n))
        first = max(0, start - w + 1)
        keys += n - first + min(first, p)
        tokens += n - start
    size = 2 * d * hkv * 2 * keys + 2 * d * hq * (tokens + case["batch"] * case["new"])
    size += 4 * -(-keys // case["block"])
    if case["bias"]:
        size += 4 * hq
    return {"bytes": size, "flops": 4 * d * hq * pairs}


# -- the definition in 64 bits -------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        h = s["x"].double().add(s["residual"].double()).to(torch.float16)
        total = h.double().square().sum(dim=1)
        factor = (total / case["width"] + EPS).pow(-0.5)
        return s["weight"].double() * h.double() * factor.unsqueeze(1), h.double()
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    group = hq // hkv
    out = torch.zeros(case["batch"], case["new"], hq, d, dtype=torch.float64, device=DEV)
    for b, (n, start, pre) in enumerate(zip(*_sizes(case))):
        blocks = s["table"][b, :-(-n // block)].long()
        keys = s["kc"][blocks].flatten(0, 1)[:n].double()
        values = s["vc"][blocks].flatten(0, 1)[:n].double()
        at = torch.arange(start, n, device=DEV).unsqueeze(1)
        key_at = torch.arange(n, device=DEV).unsqueeze(0)
        hidden = key_at > at
        if case["window"]:
            hidden |= key_at <= at - case["window"]
        hidden &= key_at >= pre
        for h in range(hq):
            score = torch.mm(s["q"][b, :n - start, h].double(), keys[:, h // group].t().contiguous())
            score.mul_(s["scale"])
            if case["cap"]:
                score.div_(case["cap"]).tanh_().mul_(case["cap"])
            if case["bias"]:
                score.sub_((at - key_at).abs().double() * s["slopes"][h].double())
            score.masked_fill_(hidden, -math.inf)
            weight = (score - torch.logsumexp(score, dim=1, keepdim=True)).exp_()
            out[b, :n - start, h] = torch.mm(weight, values[:, h // group].contiguous())
    return out
