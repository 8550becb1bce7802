"""GPU parity of paged_chunk_attention against the 64-bit form (oracle/chunk.py), marked ``gpu``.

Covered: head layouts (shared heads of any group, one kv head, none shared), head widths, block
sizes that end inside a tile, chunks of one token to several row tiles, contexts from nothing to
many parts, padded rows, the score options alone and together, table entries that are missing,
infinities and NaN where a token does not look, strides, offsets past 32 bits, other streams,
graphs, and agreement with flash_attention and paged_attention where those apply.  Bounds are
the oracle's, from the kernel's roundings.
"""

import math

import pytest
import torch

from conftest import banner
from oracle import chunk as OC

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _slopes(hq):
    return 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV, dtype=torch.float32) / hq)


def _case(seed, lens, new, hq, hkv, d, bs, spare=3, spread=1.0):
    """Random q and pools, and a shuffled table with -1 past each row's blocks."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    counts = [-(-n // bs) for n in lens]
    total = sum(counts) + spare
    perm = torch.randperm(total, device=DEV, generator=g).int()
    table = torch.full((len(lens), max(counts + [1])), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = perm[at:at + n]
        at += n
    r = dict(device=DEV, generator=g)
    q = (torch.randn(len(lens), new, hq, d, **r) * spread).half()
    kc = torch.randn(total, bs, hkv, d, **r).half()
    vc = torch.randn(total, bs, hkv, d, **r).half()
    return q, kc, vc, table


def _i32(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device=DEV)


def _check(q, kc, vc, table, bs, lens, starts=None, bound_tokens=None, **kw):
    import fast_infer_amd as fi

    opts = dict(scale=kw.get("sm_scale"), cap=kw.get("softcap") or 0.0, slopes=kw.get("alibi_slopes"),
                window=kw.get("window") or 0, prefix=kw.get("prefix"))
    call = {k: v for k, v in kw.items() if k != "prefix"}
    out = fi.paged_chunk_attention(q, kc, vc, table, bs, bound_tokens or max(max(lens), 1),
                                   start_positions=_i32(starts), context_lens=_i32(lens),
                                   prefix_lens=_i32(kw.get("prefix")), **call)
    torch.cuda.synchronize()
    assert out.shape == q.shape and out.stride() == torch.empty_like(q).stride()
    exact, bound = OC.chunk_attention(q, kc, vc, table, bs, lens, starts, **opts)
    ok, msg = OC.is_close(out, exact, bound)
    assert ok, msg
    return out


LAYOUTS = [(24, 8, 128), (4, 4, 128), (32, 8, 64), (7, 1, 128), (32, 1, 40), (10, 2, 80), (3, 3, 8),
           (12, 4, 96), (40, 2, 128)]


@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
@pytest.mark.parametrize("new", [1, 2, 5, 17, 64, 131])
def test_layouts(hip, hq, hkv, d, new):
    banner(f"chunk attention {hq}/{hkv} heads x {d}, {new} new tokens")
    bs = [64, 16, 8, 24, 128, 1][new % 6]
    lens = [new, new + 1, new + 63, new + 200, new + 700]
    _check(*_case(new + hq, lens, new, hq, hkv, d, bs), bs, lens)


@pytest.mark.parametrize("bs", [1, 3, 8, 16, 24, 48, 64, 100, 128, 256, 1000])
def test_block_sizes(hip, bs):
    banner(f"chunk attention block size {bs}")
    lens = [70, 333, 1290]
    _check(*_case(bs, lens, 33, 6, 2, 64, bs), bs, lens)


OPTIONS = {
    "cap": dict(softcap=30.0),
    "bias": dict(alibi=True),
    "window": dict(window=50),
    "window1": dict(window=1),
    "prefix": dict(prefix=[10, 0, 150, 500]),
    "cap_bias": dict(softcap=20.0, alibi=True),
    "bias_window": dict(alibi=True, window=129),
    "sinks": dict(window=65, prefix=[4, 4, 1, 70]),
    "all": dict(softcap=50.0, alibi=True, window=77, prefix=[3, 64, 200, 65]),
}


@pytest.mark.parametrize("name", sorted(OPTIONS))
@pytest.mark.parametrize("new", [1, 4, 40, 200])
def test_options(hip, name, new):
    banner(f"chunk attention option {name}, {new} new tokens")
    opts = dict(OPTIONS[name])
    hq, hkv, d, bs = 6, 2, 128, 32
    lens = [new, new + 130, new + 301, new + 900]
    if opts.pop("alibi", False):
        opts["alibi_slopes"] = _slopes(hq)
    case = _case(new, lens, new, hq, hkv, d, bs, spread=4.0 if "softcap" in opts else 1.0)
    _check(*case, bs, lens, **opts)


@pytest.mark.parametrize("opts", [{}, dict(softcap=25.0, window=100), dict(window=33, prefix=[0, 70, 5, 40, 9, 9])])
def test_padded_batch(hip, opts):
    """Rows with their own number of new tokens (none included), empty rows, starts past the
    length and before the sequence: tokens that are not there give zeros."""
    banner(f"chunk attention padded batch {opts}")
    lens = [200, 90, 77, 0, 40, 64]
    starts = [160, 90, 70, 0, -9, 500]
    out = _check(*_case(3, lens, 40, 12, 4, 128, 16), 16, lens, starts, **opts)
    assert not out[1].any() and not out[3].any() and not out[5].any()
    assert not out[2, 7:].any() and not out[4, :9].any() and out[4, 9:].any()


@pytest.mark.parametrize("new", [1, 30])
def test_loose_bounds(hip, new):
    """A bound far above the lengths (a serving loop passes its maximum), lengths above the
    bound, and lengths past the table's width."""
    banner(f"chunk attention loose bounds, {new} new")
    lens = [100, 300, 2000]
    q, kc, vc, table = _case(9, lens, new, 6, 2, 128, 64)
    _check(q, kc, vc, table, 64, lens, bound_tokens=100000)
    import fast_infer_amd as fi

    exact, bound = OC.chunk_attention(q, kc, vc, table, 64, [100, 256, 256])
    out = fi.paged_chunk_attention(q, kc, vc, table, 64, 256, context_lens=_i32(lens))
    assert OC.is_close(out, exact, bound)[0]
    exact, bound = OC.chunk_attention(q, kc, vc, table[:, :3], 64, lens)
    out = fi.paged_chunk_attention(q, kc, vc, table[:, :3], 64, _i32(lens))
    assert OC.is_close(out, exact, bound)[0]


def test_one_shared_length_and_empty(hip):
    banner("chunk attention shared length")
    import fast_infer_amd as fi

    q, kc, vc, table = _case(10, [500, 500], 6, 6, 2, 128, 64)
    out = fi.paged_chunk_attention(q, kc, vc, table, 64, 500)
    exact, bound = OC.chunk_attention(q, kc, vc, table, 64, [500, 500])
    assert OC.is_close(out, exact, bound)[0]
    assert not fi.paged_chunk_attention(q, kc, vc, table, 64, 0).any()
    for shape in ((0, 6, 6, 128), (2, 0, 6, 128)):
        assert fi.paged_chunk_attention(q.new_empty(shape), kc, vc, table, 64, 500).shape == shape


@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("opts", [{}, dict(window=40)])
def test_missing_table_entries(hip, new, opts):
    """-1 and out-of-pool entries drop out of the softmax; rows left with no key give zeros."""
    banner(f"chunk attention missing entries, {new} new {opts}")
    lens = [200, 700, 90]
    q, kc, vc, table = _case(11, lens, new, 6, 2, 128, 16)
    table[0, 2], table[0, 7], table[1, 30:] = -1, 10 ** 6, -7
    table[2] = -1
    out = _check(q, kc, vc, table, 16, lens, **opts)
    assert not out[2].any()
    if opts:  # row 1's last blocks are gone: so is all that a window of 40 shows its last token
        assert not out[1, -1].any()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 128), (24, 2, 64), (2, 2, 128)])
@pytest.mark.parametrize("new", [1, 5, 100])
def test_infinities_where_no_token_looks(hip, bad, hq, hkv, d, new):
    """Unused pool slots, slots past a row's length, keys behind a token and before its window."""
    banner(f"chunk attention {bad} in masked places, {hq}/{hkv} x {d}, {new} new")
    import fast_infer_amd as fi

    lens, bs, window = [new + 190, new + 3], 16, 64
    q, kc, vc, table = _case(12, lens, new, hq, hkv, d, bs)
    want, bound = OC.chunk_attention(q, kc, vc, table, bs, lens, window=window)
    owner = torch.full((kc.shape[0], bs), -1, device=DEV)
    for b, n in enumerate(lens):
        pos = torch.arange(n, device=DEV)
        owner[table[b, pos // bs].long(), pos % bs] = b
    kc[owner < 0], vc[owner < 0] = bad, bad  # unused and past the lengths
    pos = torch.arange(max(lens[0] - new - window, 0), device=DEV)  # before every window of row 0
    for c in (kc, vc):
        c[table[0, pos // bs].long(), pos % bs] = bad
    out = fi.paged_chunk_attention(q, kc, vc, table, bs, max(lens), context_lens=_i32(lens),
                                   window=window)
    ok, msg = OC.is_close(out, want, bound)
    assert ok, msg
    if new > 1:  # and in the chunk's own last token: the tokens before it do not see it
        last = lens[0] - 1
        for c in (kc, vc):
            c[table[0, last // bs].long(), last % bs] = bad
        out = fi.paged_chunk_attention(q, kc, vc, table, bs, max(lens), context_lens=_i32(lens),
                                       window=window)
        ok, msg = OC.is_close(out[:, :-1], want[:, :-1], bound[:, :-1])
        assert ok, msg
        assert not torch.isfinite(out[0, -1]).any()


def test_infinite_values_that_are_seen(hip):
    """An infinity in V reaches exactly the tokens that see it, in its columns and with its sign;
    both signs or a NaN give NaN."""
    banner("chunk attention visible infinities")
    import fast_infer_amd as fi

    lens, bs, new = [160], 16, 50
    q, kc, vc, table = _case(13, lens, new, 6, 2, 128, bs)
    want, bound = OC.chunk_attention(q, kc, vc, table, bs, lens)
    spots = {(120, 0, 5): math.inf, (130, 1, 7): -math.inf, (140, 0, 5): -math.inf, (150, 1, 100): math.nan}
    for (pos, h, c), x in spots.items():
        vc[table[0, pos // bs].long(), pos % bs, h, c] = x
    out = fi.paged_chunk_attention(q, kc, vc, table, bs, 160)[0].float()
    touched = torch.zeros_like(out, dtype=torch.bool)
    for (pos, h, c), x in spots.items():
        t = pos - (lens[0] - new)
        touched[t:, 3 * h:3 * h + 3, c] = True
        seen = out[t:, 3 * h:3 * h + 3, c]
        if (pos, h, c) == (120, 0, 5):
            assert (seen[:20] == math.inf).all() and seen[20:].isnan().all()
        elif (pos, h, c) == (130, 1, 7):
            assert (seen == x).all()
        else:
            assert seen.isnan().all()
    assert ((out.double() - want[0]).abs() <= bound[0])[~touched].all()


@pytest.mark.parametrize("scale", [0.0, -0.1, 2.0, 1e-6, 1e-19, -1e-21, 1e-40])
@pytest.mark.parametrize("opts", [{}, dict(softcap=10.0), dict(alibi=True), dict(softcap=3000.0, alibi=True)])
def test_scales(hip, scale, opts):
    banner(f"chunk attention scale {scale} {opts}")
    opts = dict(opts)
    if opts.pop("alibi", False):
        opts["alibi_slopes"] = _slopes(6)
    lens = [90, 400]
    _check(*_case(14, lens, 21, 6, 2, 64, 32), 32, lens, sm_scale=scale, window=70, **opts)


@pytest.mark.parametrize("cap", [1e-40, 1e-19, 1e-3, 0.5, 500.0, 501.0, 1e5, 1e7])
def test_caps(hip, cap):
    """Caps below the scores and far above them (where the plain form of tanh loses digits)."""
    banner(f"chunk attention cap {cap}")
    lens = [300]
    _check(*_case(15, lens, 9, 6, 2, 128, 64, spread=8.0), 64, lens, softcap=cap)


def test_strides_and_alignment(hip):
    """Views of a fused projection, transposed heads, rows the kernel cannot read directly."""
    banner("chunk attention strides")
    import fast_infer_amd as fi

    lens = [150, 260]
    q, kc, vc, table = _case(16, lens, 11, 6, 2, 128, 64)
    exact, bound = OC.chunk_attention(q, kc, vc, table, 64, lens)
    qkv = torch.randn(2, 11, 10, 128, device=DEV).half()
    qkv[:, :, :6] = q
    wide = torch.zeros(2, 11, 6, 136, dtype=torch.float16, device=DEV)
    wide[..., 4:132] = q
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    table2 = torch.zeros(2, table.shape[1], 2, dtype=torch.int32, device=DEV)
    table2[..., 0] = table
    cols = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    cols[:, 0] = _i32(lens)
    for view in (qkv[:, :, :6], wide[..., 4:132], heads_first):
        out = fi.paged_chunk_attention(view, kc, vc, table2[..., 0], 64, 260, context_lens=cols[:, 0].long())
        ok, msg = OC.is_close(out, exact, bound)
        assert ok, msg
        assert out.stride() == torch.empty_like(view).stride()


def test_long_context_and_parts(hip):
    """One conversation of 100000 tokens; the same call without a workspace, with a small one and
    again; bounds and bits."""
    banner("chunk attention long context")
    import fast_infer_amd as fi

    n, new = 100_003, 3
    q, kc, vc, table = _case(17, [n], new, 6, 2, 128, 64)
    out = _check(q, kc, vc, table, 64, [n])
    again = fi.paged_chunk_attention(q, kc, vc, table, 64, n)
    assert torch.equal(out, again)
    exact, bound = OC.chunk_attention(q, kc, vc, table, 64, [n])
    from fast_infer_amd import _lib

    lib = _lib.load()
    full = lib.fi_paged_chunk_attention_workspace_size(1, new, 6, 2, n, 128)
    assert full > 0
    for size in (0, 1000, full - 1, full):
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
        o = torch.empty_like(q)
        rc = lib.fi_paged_chunk_attention_fwd(
            q.data_ptr(), *q.stride()[:3], kc.data_ptr(), vc.data_ptr(), kc.shape[0], 64, 2,
            table.data_ptr(), table.stride(0), table.shape[1], None, None, n, o.data_ptr(), *o.stride()[:3],
            1, new, 6, 128, 128 ** -0.5, 0.0, None, 0, None, ws.data_ptr() if size else None, size,
            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        ok, msg = OC.is_close(o, exact, bound)
        assert ok, (size, msg)


def test_offsets_past_32_bits(hip):
    """Pools of 4.5 GB: the same rows at the pools' far end."""
    banner("chunk attention pools past 4 GiB")
    import fast_infer_amd as fi

    lens, new, bs, hq, hkv, d = [300, 90], 7, 64, 12, 4, 128
    q, kc, vc, table = _case(18, lens, new, hq, hkv, d, bs)
    want = fi.paged_chunk_attention(q, kc, vc, table, bs, 300, context_lens=_i32(lens))
    blocks = 4_500_000_000 // (bs * hkv * d * 2)
    far = blocks - kc.shape[0]
    pools = []
    for c in (kc, vc):
        big = torch.empty(blocks, bs, hkv, d, dtype=torch.float16, device=DEV)
        big[far:] = c
        pools.append(big)
    moved = torch.where(table >= 0, table + far, table)
    out = fi.paged_chunk_attention(q, *pools, moved, bs, 300, context_lens=_i32(lens))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_agrees_with_prefill_and_decode(hip):
    """A whole prompt as one chunk against flash_attention, its last token against
    paged_attention, and the prompt in pieces against the whole (each within both bounds)."""
    banner("chunk attention against prefill and decode")
    import fast_infer_amd as fi

    n, hq, hkv, d, bs = 700, 24, 8, 128, 64
    q, kc, vc, table = _case(19, [n, n], n, hq, hkv, d, bs)
    exact, bound = OC.chunk_attention(q[:, -40:], kc, vc, table, bs, [n, n])
    whole = fi.paged_chunk_attention(q, kc, vc, table, bs, n)
    rows = lambda c: torch.stack([c[table[b].long()].flatten(0, 1)[:n] for b in range(2)])
    flash = fi.flash_attention(q.transpose(1, 2), rows(kc).transpose(1, 2), rows(vc).transpose(1, 2))
    assert (whole.float() - flash.transpose(1, 2).float()).abs().max() <= 4e-3  # 2e-3 each
    decode = fi.paged_attention(q[:, -1].contiguous(), kc, vc, table, bs, n)
    one = fi.paged_chunk_attention(q[:, -1:], kc, vc, table, bs, n)
    for out in (whole[:, -40:], flash.transpose(1, 2)[:, -40:]):
        assert OC.is_close(out, exact, bound)[0]
    for out in (decode, one[:, 0]):
        assert OC.is_close(out, exact[:, -1], bound[:, -1])[0]
    at = 0
    for size in (1, 200, 333, 166):
        piece = fi.paged_chunk_attention(q[:, at:at + size], kc, vc, table, bs, at + size)
        assert (piece.float() - whole[:, at:at + size].float()).abs().max() <= 4e-3
        at += size
    assert at == n


def test_other_stream_and_two_at_once(hip):
    banner("chunk attention on two streams")
    import fast_infer_amd as fi

    lens = [3000, 1000]
    a = _case(20, lens, 8, 24, 8, 128, 64)
    b = _case(21, lens, 8, 24, 8, 128, 64)
    want = [fi.paged_chunk_attention(*x, 64, 3000, context_lens=_i32(lens)) for x in (a, b)]
    lens_t = _i32(lens)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, (s, x) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append(fi.paged_chunk_attention(*x, 64, 3000, context_lens=lens_t))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_graph_replay(hip):
    """Captured with the workspace of the call's own; replayed with new inputs and lengths in the
    same tensors, with eager calls between."""
    banner("chunk attention graph replay")
    import fast_infer_amd as fi

    q, kc, vc, table = _case(22, [900, 400], 6, 24, 8, 128, 64)
    lens, starts = _i32([900, 400]), _i32([894, 396])
    call = lambda: fi.paged_chunk_attention(q, kc, vc, table, 64, 960, start_positions=starts,
                                            context_lens=lens, softcap=30.0, window=500)
    call()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(4):
        q.copy_(torch.randn_like(q))
        lens.copy_(_i32([900 - step, 400 - 50 * step]))
        starts.copy_(_i32([894 - step, 396 - 50 * step]))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call()), step


def test_wrapper_refusals(hip):
    import fast_infer_amd as fi

    q, kc, vc, table = _case(23, [64], 4, 6, 2, 128, 64)
    call = lambda **kw: fi.paged_chunk_attention(q, kc, vc, table, 64, 64, **kw)
    for kw in (dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=math.nan), dict(window=0),
               dict(alibi_slopes=torch.ones(5, device=DEV)), dict(context_lens=_i32([])),
               dict(start_positions=_i32([])), dict(prefix_lens=_i32([]))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(fi._lib.FastInferError):
        call(softcap=math.inf)
    with pytest.raises(fi._lib.FastInferError):
        fi.paged_chunk_attention(q, kc, vc, table, 64, 64, math.nan)
    with pytest.raises(fi._lib.FastInferError):
        fi.paged_chunk_attention(q, kc, vc, table, 64, -1)
    for ws in (torch.empty(1 << 24, dtype=torch.uint8), torch.empty(1 << 24, 2, dtype=torch.uint8, device=DEV)[:, 0]):
        with pytest.raises(ValueError):
            call(workspace=ws)
    with pytest.raises(ValueError):
        fi.paged_chunk_attention(q, kc, vc, table, 32, 64)
    with pytest.raises(ValueError):
        fi.paged_chunk_attention(q[:, :, :5], kc, vc, table, 64, 64)
    with pytest.raises(ValueError):
        fi.paged_chunk_attention(q, kc.transpose(0, 1), vc.transpose(0, 1), table, 64, 64)
    with pytest.raises(ValueError):
        fi.paged_chunk_attention(q, kc, vc, table, 64, _i32([64]), context_lens=_i32([64]))
    with pytest.raises(TypeError):
        fi.paged_chunk_attention(q, kc, vc, table.long(), 64, 64)
    with pytest.raises(RuntimeError):
        fi.paged_chunk_attention(q, kc.cpu(), vc.cpu(), table, 64, 64)


def test_many_rows_share_the_work_list(hip):
    """More batch rows than a wave has lanes, most without new tokens, lengths far apart."""
    banner("chunk attention 150 rows")
    batch, new = 150, 3
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(0, 400, (batch,), generator=g).tolist()
    lens[70], lens[149] = 5000, 3000
    starts = [n - int(c) for n, c in zip(lens, torch.randint(0, new + 1, (batch,), generator=g))]
    q, kc, vc, table = _case(24, lens, new, 3, 1, 64, 16)
    _check(q, kc, vc, table, 16, lens, starts)


@pytest.mark.parametrize("new", [1, 5, 9, 60])
def test_infinite_values_per_column_padding_and_parts(hip, new):
    """Single infinite columns in the chunk, in the prefix and past the window, on a padded batch
    whose context is cut into parts: rows that see them, and padding, which stays zero."""
    banner(f"chunk attention infinite columns, {new} new")
    import fast_infer_amd as fi

    lens, bs, window, prefix = [2000, 700], 16, 100, [70, 3]
    starts = [2000 - new, 700 - (new + 1) // 2]
    q, kc, vc, table = _case(25, lens, new, 6, 2, 128, bs)
    want, bound = OC.chunk_attention(q, kc, vc, table, bs, lens, starts, window=window, prefix=prefix)
    spots = [(0, 69, 0, 3), (0, 70, 0, 4), (0, 1999, 1, 127), (0, 1900 - new, 1, 64), (1, 2, 0, 9), (1, 699, 1, 31)]
    for b, pos, h, c in spots:
        vc[table[b, pos // bs].long(), pos % bs, h, c] = math.inf if pos % 2 else -math.inf
    out = fi.paged_chunk_attention(q, kc, vc, table, bs, 2000, start_positions=_i32(starts),
                                   context_lens=_i32(lens), window=window, prefix_lens=_i32(prefix))
    for b, pos, h, c in spots:
        for t in range(new):
            at = starts[b] + t
            if at < lens[b] and (pos < prefix[b] or at - window < pos <= at):
                want[b, t, 3 * h:3 * h + 3, c] = math.inf if pos % 2 else -math.inf
    finite = torch.isfinite(want)
    assert torch.equal(out.double()[~finite], want[~finite])
    assert ((out.double() - want).abs() <= bound)[finite].all()
    assert not out[1, (new + 1) // 2:].any()


@pytest.mark.parametrize("bs", [8, 16, 24])
@pytest.mark.parametrize("new", [2, 50])
def test_long_parts(hip, bs, new):
    """Parts of far more than 64 key tiles (no workspace): entries in the pool and missing ones
    throughout, block sizes with one entry per 16 keys and with several."""
    banner(f"chunk attention long parts, block size {bs}, {new} new")
    from fast_infer_amd import _lib

    n = 17_003
    q, kc, vc, table = _case(26, [n], new, 6, 2, 64, bs)
    gone = torch.randperm(table.shape[1], generator=torch.Generator().manual_seed(1))[:40]
    table[0, gone.to(DEV)] = -1
    exact, bound = OC.chunk_attention(q, kc, vc, table, bs, [n])
    o = torch.empty_like(q)
    rc = _lib.load().fi_paged_chunk_attention_fwd(
        q.data_ptr(), *q.stride()[:3], kc.data_ptr(), vc.data_ptr(), kc.shape[0], bs, 2,
        table.data_ptr(), table.stride(0), table.shape[1], None, None, n, o.data_ptr(), *o.stride()[:3],
        1, new, 6, 64, 0.125, 0.0, None, 0, None, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    ok, msg = OC.is_close(o, exact, bound)
    assert ok, msg


# (batch, kv heads, group, new tokens, longest row, head_dim, block size): row tiles that fill the
# device, with two and three row blocks a wave, and fewer of them over longer rows, cut into parts
MANY_ROWS = [(4, 8, 8, 193, 242, 128, 16), (4, 8, 8, 260, 367, 128, 64), (4, 8, 8, 193, 220, 64, 24),
             (4, 8, 8, 274, 379, 64, 16), (2, 8, 1, 582, 3619, 128, 64), (4, 8, 3, 174, 3747, 128, 32),
             (1, 4, 6, 534, 3085, 120, 48), (2, 8, 2, 291, 3600, 64, 16), (4, 8, 1, 524, 3737, 64, 40)]


@pytest.mark.parametrize("opts", [{}, {"softcap": 20.0}, {"alibi": 1, "prefix": 150},
                                  {"softcap": 900.0, "alibi": 1, "window": 100, "prefix": 70}],
                         ids=["plain", "cap", "bias", "all"])
@pytest.mark.parametrize("shape", MANY_ROWS, ids=lambda s: "x".join(map(str, s)))
def test_many_query_rows(hip, shape, opts):
    """Chunks of many query rows, the rows of the batch at different lengths and padded but for one."""
    banner(f"chunk attention many rows {shape} {opts}")
    batch, hkv, group, new, longest, d, bs = shape
    lens = [longest - 37 * b * (longest // 150) for b in range(batch)]
    starts = [n - new + 11 * b for b, n in enumerate(lens)]
    kw = dict(opts)
    if kw.pop("alibi", None):
        kw["alibi_slopes"] = _slopes(group * hkv)
    if "prefix" in kw:
        kw["prefix"] = [kw["prefix"] >> b for b in range(batch)]
    q, kc, vc, table = _case(27, lens, new, group * hkv, hkv, d, bs, spread=3.0 if "softcap" in kw else 1.0)
    out = _check(q, kc, vc, table, bs, lens, starts, **kw)
    for b in range(1, batch):
        assert not out[b, new - 11 * b:].any()


@pytest.mark.parametrize("shape", MANY_ROWS[1:4] + MANY_ROWS[5:8], ids=lambda s: "x".join(map(str, s)))
def test_infinite_values_of_many_query_rows(hip, shape):
    """Infinite values of V at the chunk's own positions reach the tokens that see them and no others."""
    banner(f"chunk attention infinities many rows {shape}")
    import fast_infer_amd as fi

    batch, hkv, group, new, longest, d, bs = shape
    lens = [longest - 20 * b for b in range(batch)]
    starts = [n - new + b for b, n in enumerate(lens)]
    q, kc, vc, table = _case(28, lens, new, group * hkv, hkv, d, bs)
    want, bound = OC.chunk_attention(q, kc, vc, table, bs, lens, starts, window=90)
    spots = [(b, starts[b] + t, (3 * t) % hkv, (17 * t) % d) for b in range(batch) for t in (5, new // 2, new - 9)]
    # (the third and fourth rows of the shorter chunks begin before position 0: their first spot is an
    # index from the table's end, of a slot that may be another row's.  So what each row holds is read back.)
    for b, pos, h, c in spots:
        vc[table[b, pos // bs].long(), pos % bs, h, c] = math.inf
    for b in range(batch):
        pos = torch.arange(lens[b], device=DEV)
        rows = vc[table[b, pos // bs].long(), pos % bs]
        for at, h, c in torch.isinf(rows).nonzero().tolist():
            t0, t1 = max(at - starts[b], -starts[b], 0), min(at - starts[b] + 90, lens[b] - starts[b])
            want[b, t0:max(t1, t0), group * h:group * h + group, c] = math.inf
    out = fi.paged_chunk_attention(q, kc, vc, table, bs, longest, start_positions=_i32(starts),
                                   context_lens=_i32(lens), window=90)
    finite = torch.isfinite(want)
    assert torch.equal(out.double()[~finite], want[~finite])
    assert ((out.double() - want).abs() <= bound)[finite].all()
