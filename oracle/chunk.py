"""Attention of a chunk of new tokens over a paged pool, and the residual norm, in 64 bits.

``chunk_attention`` follows the definition token by token set: scores, cap, distance bias and
visibility as ``fi_paged_chunk_attention_fwd`` states them, a softmax over the visible keys only
(what a masked key holds never enters a sum).  With it come error bounds for the kernel's fp16
results, from the roundings that it makes.
"""

import math

import torch


def gather(pool, table_row, n, bs):
    """The first n tokens of a row as [n, heads, dim], and which of them lie in the pool."""
    pos = torch.arange(n, device=pool.device)
    entry = torch.full((n,), -1, dtype=torch.long, device=pool.device)
    blk = pos // bs
    known = blk < table_row.numel()
    entry[known] = table_row[blk[known]].long()
    ok = (entry >= 0) & (entry < pool.shape[0])
    rows = pool[entry.clamp(0, pool.shape[0] - 1), pos % bs]
    return rows, ok


def chunk_attention(q, kc, vc, table, bs, lens, starts=None, scale=None, cap=0.0, slopes=None,
                    window=0, prefix=None):
    """(o, bound): float64 [batch, new, heads, dim] and the largest |error| of the fp16 kernel.

    Bound: each weight is rounded to fp16 (relative 2^-11, the sum takes the same rounded
    weights, so an output moves by at most twice that of the weighted |v|), weights below the
    type's normal range by 2^-25 absolutely next to a largest weight of at least 1, and scores
    are off by their fp32 arithmetic (eta); the output is rounded once (2^-11 of itself)."""
    batch, new, hq, d = q.shape
    hkv = kc.shape[2]
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(batch, new, hq, d, dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, 2.0 ** -25)
    for b in range(batch):
        n = max(min(lens[b], table.shape[1] * bs), 0)
        start = n - new if starts is None else starts[b]
        k, ok = gather(kc, table[b], n, bs)
        v, _ = gather(vc, table[b], n, bs)
        key = torch.arange(n, device=q.device)
        for t in range(new):
            pos = start + t
            if pos < 0 or pos >= n:
                continue
            see = key <= pos
            if window:
                see &= key > pos - window
            if prefix is not None:
                see |= key < prefix[b]
            idx = torch.nonzero(see & ok).flatten()
            if not idx.numel():
                continue
            ks = k[idx].double().transpose(0, 1).contiguous()  # [hkv, m, d]
            vs = v[idx].double().transpose(0, 1).contiguous()
            qs = q[b, t].double().view(hkv, hq // hkv, d)
            x = torch.bmm(qs, ks.transpose(1, 2).contiguous()).view(hq, -1) * scale
            mag = torch.bmm(qs.abs(), ks.abs().transpose(1, 2).contiguous()).max() * abs(scale)
            eta = (d + 8) * 2.0 ** -24 * float(mag) + 2.0 ** -20
            if cap:
                x = cap * torch.tanh(x / cap)
                eta += 4e-7 * min(cap, 500.0) + 2.0 ** -21 * min(cap, float(mag))
            if slopes is not None:
                x = x - slopes.double().view(-1, 1) * (pos - key[idx]).abs().double()
                eta += 2.0 ** -20
            w = torch.softmax(x, -1)
            o = torch.bmm(w.view(hkv, hq // hkv, -1), vs).view(hq, d)
            near = torch.bmm(w.view(hkv, hq // hkv, -1), vs.abs()).view(hq, d)
            out[b, t] = o
            bound[b, t] += (2.0 ** -11 * o.abs() + (2.0 ** -10 + 2 * eta) * near
                            + idx.numel() * 2.0 ** -24 * vs.abs().amax(1).repeat_interleave(hq // hkv, 0))
    return out, bound


def add_rms_norm(x, residual, weight, eps):
    """(out, h) in 64 bits from the fp16-rounded h, and the bound of the fp16 kernel's out: one
    rounding (2^-11), and the fp32 sum and scaling."""
    h = (x.double() + residual.double()).to(torch.float16)
    f = h.double()
    out = f / torch.sqrt((f * f).mean(-1, keepdim=True) + eps) * weight.double()
    return out, h, out.abs() * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -25


def is_close(got, exact, bound):
    """Every element within its bound; where not, the worst one for the message."""
    err = (got.double() - exact).abs()
    bad = ~(err <= bound)
    if not bool(bad.any()):
        return True, ""
    i = int(torch.where(bad, err / bound, torch.zeros_like(err)).nan_to_num(math.inf).argmax())
    at = [int(c) for c in torch.unravel_index(torch.tensor(i), err.shape)]
    return False, (f"{int(bad.sum())} of {bad.numel()} off, worst at {at}: got "
                   f"{float(got.flatten()[i])}, exact {float(exact.flatten()[i])}, bound "
                   f"{float(bound.flatten()[i])}")
