"""add_rms_norm against the 64-bit form, and the operators of a step that continues cached
sequences together (block manager, residual norm, INT4 projections, RoPE with the pool write,
chunk attention), marked ``gpu``."""

import pytest
import torch

from conftest import banner
from oracle import chunk as OC

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _rows(seed, m, n, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = dict(device=DEV, generator=g)
    return (torch.randn(m, n, **r).half(), (torch.randn(m, n, **r) * spread).half(),
            (1 + 0.2 * torch.randn(n, **r)).half())


def _check_norm(out, h, x, res, w, eps=1e-5):
    exact, want_h, bound = OC.add_rms_norm(x, res, w, eps)
    assert torch.equal(h, want_h)
    ok, msg = OC.is_close(out, exact, bound)
    assert ok, msg


@pytest.mark.parametrize("m", [1, 3, 64, 1000])
@pytest.mark.parametrize("n", [8, 64, 504, 512, 520, 2040, 2048, 2056, 4096, 5120, 8192, 8200, 20000])
def test_add_rms_norm(hip, m, n):
    banner(f"add_rms_norm {m} x {n}")
    from fast_infer_amd import add_rms_norm

    x, res, w = _rows(m + n, m, n)
    out, h = add_rms_norm(x, res, w, 1e-5)
    torch.cuda.synchronize()
    _check_norm(out, h, x, res, w)


def test_add_rms_norm_many_rows(hip):
    banner("add_rms_norm 70001 x 256")
    from fast_infer_amd import add_rms_norm

    x, res, w = _rows(5, 70001, 256)
    out, h = add_rms_norm(x, res, w, 1e-6)
    _check_norm(out, h, x, res, w, 1e-6)


@pytest.mark.parametrize("n", [1000, 9000])
def test_add_rms_norm_strides_and_in_place(hip, n):
    banner(f"add_rms_norm strides {n}")
    from fast_infer_amd import add_rms_norm

    x, res, w = _rows(6, 24, n)
    wide = torch.zeros(24, n + 64, dtype=torch.float16, device=DEV)
    wide[:, 32:32 + n] = x
    odd = torch.zeros(24, n + 1, dtype=torch.float16, device=DEV)
    odd[:, 1:] = res
    out, h = add_rms_norm(wide[:, 32:32 + n], odd[:, 1:], w)
    _check_norm(out, h, x, res, w)
    out3, h3 = add_rms_norm(x.view(2, 3, 4, n), res.view(2, 3, 4, n), w)
    assert out3.shape == h3.shape == (2, 3, 4, n)
    assert torch.equal(out3.view(24, n), out) and torch.equal(h3.view(24, n), h)
    # in place: the residual's own rows, padding around them untouched
    stream = torch.full((24, n + 64), 7.0, dtype=torch.float16, device=DEV)
    stream[:, 16:16 + n] = res
    view = stream[:, 16:16 + n]
    out2, h2 = add_rms_norm(x, view, w, inplace=True)
    assert h2 is view and torch.equal(view, h) and torch.equal(out2, out)
    assert (stream[:, :16] == 7).all() and (stream[:, 16 + n:] == 7).all()
    with pytest.raises(ValueError):
        add_rms_norm(x, odd[:, 1:], w, inplace=True)
    # the residual added to itself, and a weight of another type
    out, h = add_rms_norm(res, res, w.float())
    _check_norm(out, h, res, res, w)


def test_add_rms_norm_extremes(hip):
    """Sums that overflow, rows of zeros, the smallest values, one row's NaN beside others."""
    banner("add_rms_norm extremes")
    from fast_infer_amd import add_rms_norm

    x, res, w = _rows(7, 6, 768)
    x[0], res[0] = 0, 0
    x[1], res[1] = 6e-8, 0
    x[2], res[2] = 60000, 5000
    x[3, 5] = float("nan")
    out, h = add_rms_norm(x, res, w)
    # 60000 + 5000 is below the type's 65504: row 2 rounds to 64992 and stays finite
    assert not out[0].any() and (h[2] == 64992).all() and out[3].isnan().all()
    keep = [0, 1, 2, 4, 5]
    _check_norm(out[keep], h[keep], x[keep], res[keep], w)
    x[4], res[4] = 60000, 6000  # 66000 is past it
    out, h = add_rms_norm(x, res, w)
    assert torch.isinf(h[4]).all() and out[4].isnan().all()
    keep = [0, 1, 2, 5]
    _check_norm(out[keep], h[keep], x[keep], res[keep], w)


def test_add_rms_norm_equals_its_parts_and_graph(hip):
    """The addition and rms_norm apart give the same h and, up to one last bit, the same rows;
    captured, it replays on new inputs."""
    banner("add_rms_norm against its parts")
    from fast_infer_amd import add_rms_norm, rms_norm

    x, res, w = _rows(8, 300, 4096)
    out, h = add_rms_norm(x, res, w)
    assert torch.equal(h, x + res)
    parts = rms_norm(x + res, w).float()
    assert ((out.float() - parts).abs() <= parts.abs() * 2.0 ** -10 + 2.0 ** -24).all()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = add_rms_norm(x, res, w)
    for step in range(3):
        x.copy_(torch.randn_like(x))
        res.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        eager = add_rms_norm(x, res, w)
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1])
    with pytest.raises(ValueError):
        add_rms_norm(x, res[:5], w)
    with pytest.raises(ValueError):
        add_rms_norm(x, res, w[:8])
    with pytest.raises(TypeError):
        add_rms_norm(x, res.float(), w)
    with pytest.raises(RuntimeError):
        add_rms_norm(x, res.cpu(), w)


HQ, HKV, D, HIDDEN, LAYERS, BS = 8, 2, 64, 512, 2, 16


def _model(seed):
    from fast_infer_amd import precompute_freqs, quantize_int4_groupwise

    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=g)
    layers = []
    for _ in range(LAYERS):
        layers.append(dict(norm=(1 + 0.1 * rand(HIDDEN)).half(),
                           qkv=quantize_int4_groupwise((rand((HQ + 2 * HKV) * D, HIDDEN) * 0.05).half()),
                           o=quantize_int4_groupwise((rand(HIDDEN, HQ * D) * 0.05).half())))
    cos, sin = precompute_freqs(D, 512, device=DEV)
    return layers, cos.half(), sin.half()


def _step(model, cache, x, count, **opts):
    """One pass over new tokens x [batch, new, hidden], `count` of them real in each row."""
    from fast_infer_amd import add_rms_norm, int4_matmul, paged_chunk_attention, rope_store_kv

    layers, cos, sin = model
    batch, new, _ = x.shape
    starts, lens = cache.append(torch.tensor(count, dtype=torch.int32, device=DEV))
    block, stream = x, torch.zeros_like(x)
    for i, layer in enumerate(layers):
        normed, stream = add_rms_norm(block, stream, layer["norm"])
        qkv = int4_matmul(normed, layer["qkv"]).view(batch, new, HQ + 2 * HKV, D)
        q, k, v = qkv.split([HQ, HKV, HKV], 2)
        q, _ = rope_store_kv(q, k, v, cos, sin, 0, cache.k[i], cache.v[i], cache.block_table,
                             start_positions=starts, return_k=False)
        attn = paged_chunk_attention(q, cache.k[i], cache.v[i], cache.block_table, BS, 256,
                                     start_positions=starts, context_lens=lens, **opts)
        block = int4_matmul(attn.view(batch, new, HQ * D), layer["o"])
    normed, _ = add_rms_norm(block, stream, layers[0]["norm"])
    return normed


@pytest.mark.parametrize("opts", [{}, dict(softcap=20.0), dict(window=24)])
def test_prompts_in_pieces(hip, opts):
    """Three prompts of different lengths given whole, and in ragged pieces with padding: the
    same hidden states.  Every fp16 rounding on the way (about six a layer, each 2^-11 of values
    of order 1, through two layers and a norm) may differ between the two; 2^-5 is more than 24
    such steps of values up to 2.5 and far below what one wrong key does."""
    banner(f"prompts in pieces {opts}")
    from fast_infer_amd import PagedKVCache

    model = _model(31)
    lens = [100, 37, 64]
    g = torch.Generator(device=DEV).manual_seed(32)
    x = torch.randn(3, max(lens), HIDDEN, device=DEV, generator=g).half()
    fresh = lambda: PagedKVCache(LAYERS, HKV, D, 256, BS, DEV, 3)
    cache = fresh()
    whole = _step(model, cache, x, lens, **opts)
    cache.check()
    cache = fresh()
    at = [0, 0, 0]
    plan = [[60, 1, 30], [1, 20, 33], [0, 16, 1], [39, 0, 0]]
    for counts in plan:
        new = max(counts)
        part = torch.randn(3, new, HIDDEN, device=DEV, generator=g).half()  # noise as padding
        for b, c in enumerate(counts):
            part[b, :c] = x[b, at[b]:at[b] + c]
        out = _step(model, cache, part, counts, **opts)
        for b, c in enumerate(counts):
            diff = (out[b, :c].float() - whole[b, at[b]:at[b] + c].float()).abs()
            assert c == 0 or diff.max() <= 2.0 ** -5, (counts, b, float(diff.max()))
            at[b] += c
    cache.check()
    assert at == lens and cache.seq_lens.tolist() == lens


def test_drafted_tokens_rejected(hip):
    """Four drafted tokens verified at once, two rejected: the row goes on from its accepted
    length, over the stale rows that the rejected ones left in the pool."""
    banner("drafted tokens")
    from fast_infer_amd import PagedKVCache

    model = _model(33)
    g = torch.Generator(device=DEV).manual_seed(34)
    x = torch.randn(1, 60, HIDDEN, device=DEV, generator=g).half()
    cache = PagedKVCache(LAYERS, HKV, D, 256, BS, DEV, 1)
    whole = _step(model, cache, x, [60])
    cache.reset()
    _step(model, cache, x[:, :50], [50])
    draft = torch.cat([x[:, 50:52], torch.randn(1, 2, HIDDEN, device=DEV, generator=g).half()], 1)
    out = _step(model, cache, draft, [4])
    assert (out[:, :2].float() - whole[:, 50:52].float()).abs().max() <= 2.0 ** -5
    cache.seq_lens.sub_(2)
    out = _step(model, cache, x[:, 52:60].contiguous(), [8])
    assert (out.float() - whole[:, 52:60].float()).abs().max() <= 2.0 ** -5
