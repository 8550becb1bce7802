"""Host-side checks of paged_chunk_attention and add_rms_norm on the CPU: refusals of the C
entry points and of the wrappers, workspace sizes, the native call path, and the M0 use of the
compiled kernels (no kernel runs)."""

import math
import random
import re

import pytest
import torch

import fast_infer_amd as fi
from fast_infer_amd import _lib
from oracle import chunk as OC
from test_device_code import _device_asm

A = 1 << 40  # an aligned address that no call here dereferences


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _chunk(**kw):
    """fi_paged_chunk_attention_fwd's arguments, valid for an empty batch, with overrides."""
    a = dict(q=A, q_sb=8, q_st=8, q_sh=8, kc=A, vc=A, blocks=4, bs=64, hkv=8, table=A, bt_stride=4,
             max_blocks=4, starts=None, lens=None, tokens=256, o=A, o_sb=8, o_st=8, o_sh=8, batch=0,
             new=4, hq=24, d=128, scale=0.1, cap=0.0, slopes=None, window=0, prefix=None, ws=None,
             ws_bytes=0, stream=None)
    a.update(kw)
    return list(a.values())


def _norm(**kw):
    a = dict(x=A, xs=256, r=A + 4096, rs=256, M=0, hidden=256, w=A, eps=1e-5, h=A + 8192, hs=256,
             o=A + 16384, os=256, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad,rc,text", [
    (dict(d=60), _lib.FI_ERR_UNSUPPORTED, b"head_dim 60"),
    (dict(d=136), _lib.FI_ERR_UNSUPPORTED, b"head_dim 136"),
    (dict(hq=20), _lib.FI_ERR_INVALID, b"heads 20/8"),
    (dict(hkv=0), _lib.FI_ERR_INVALID, b"invalid sizes"),
    (dict(new=-1), _lib.FI_ERR_INVALID, b"invalid sizes"),
    (dict(batch=-1), _lib.FI_ERR_INVALID, b"invalid sizes"),
    (dict(tokens=-1), _lib.FI_ERR_INVALID, b"invalid sizes"),
    (dict(blocks=-1), _lib.FI_ERR_INVALID, b"invalid sizes"),
    (dict(max_blocks=-1), _lib.FI_ERR_INVALID, b"invalid sizes"),
    (dict(bs=0), _lib.FI_ERR_INVALID, b"block_size 0"),
    (dict(batch=1, bs=1 << 32, blocks=0), _lib.FI_ERR_INVALID, b"block_size 4294967296"),
    (dict(window=-5), _lib.FI_ERR_INVALID, b"window -5"),
    (dict(cap=-1.0), _lib.FI_ERR_INVALID, b"softcap -1"),
    (dict(cap=math.inf), _lib.FI_ERR_INVALID, b"softcap inf"),
    (dict(cap=math.nan), _lib.FI_ERR_INVALID, b"softcap"),
    (dict(scale=math.nan), _lib.FI_ERR_INVALID, b"sm_scale"),
    (dict(scale=math.inf), _lib.FI_ERR_INVALID, b"sm_scale"),
    (dict(cap=1.1e7), _lib.FI_ERR_INVALID, b"softcap"),
    (dict(scale=-1.1e7), _lib.FI_ERR_INVALID, b"sm_scale"),
    (dict(batch=1, tokens=(1 << 22) + 1), _lib.FI_ERR_UNSUPPORTED, b"too large"),
    (dict(batch=1, blocks=1 << 26), _lib.FI_ERR_UNSUPPORTED, b"too large"),
    (dict(batch=1, new=1 << 27), _lib.FI_ERR_UNSUPPORTED, b"too large"),
    (dict(batch=1 << 20, new=1 << 13), _lib.FI_ERR_UNSUPPORTED, b"new tokens"),
    (dict(batch=1, q=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(batch=1, o=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(batch=1, vc=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(batch=1, table=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(batch=1, q=A + 2), _lib.FI_ERR_INVALID, b"aligned"),
    (dict(batch=1, o=A + 8), _lib.FI_ERR_INVALID, b"aligned"),
    (dict(batch=1, kc=A + 8), _lib.FI_ERR_INVALID, b"aligned"),
    (dict(batch=1, q_st=12), _lib.FI_ERR_INVALID, b"aligned"),
    (dict(batch=1, o_sb=4), _lib.FI_ERR_INVALID, b"aligned"),
    (dict(batch=1, ws=A + 8, ws_bytes=1 << 30), _lib.FI_ERR_INVALID, b"workspace"),
])
def test_chunk_refusals(lib, bad, rc, text):
    # a workspace is looked at only by calls that are cut into parts
    more = dict(tokens=1 << 16, max_blocks=1 << 10) if "ws" in bad else {}
    assert lib.fi_paged_chunk_attention_fwd(*_chunk(**{**more, **bad})) == rc
    assert text in lib.fi_last_error()


def test_chunk_empty_calls(lib):
    assert lib.fi_paged_chunk_attention_fwd(*_chunk()) == _lib.FI_OK
    assert lib.fi_paged_chunk_attention_fwd(*_chunk(batch=3, new=0, q=None, o=None)) == _lib.FI_OK


def test_chunk_workspace_size(lib):
    size = lib.fi_paged_chunk_attention_workspace_size
    assert size(1, 4, 24, 8, 512, 128) == 0         # a few tiles of keys: not cut
    assert size(64, 512, 24, 8, 4096, 128) == 0     # query tiles alone fill the device
    assert size(1, 4, 24, 8, 4096, 128) > 0
    for bad in ((0, 4, 24, 8, 4096, 128), (1, 0, 24, 8, 4096, 128), (1, 4, 20, 8, 4096, 128),
                (1, 4, 24, 8, 0, 128), (1, 4, 24, 8, 4096, 60), (1, 4, 24, 8, (1 << 22) + 1, 128)):
        assert size(*bad) == 0
    # a window may choose other row blocks: 106 rows of 16 keys or more a wave, parts of one round
    # of 512 workgroups, 128 columns, a maximum and a sum
    assert size(1, 106, 1, 1, 17117, 128) >= (512 + 1) * 106 * 130 * 4 + 8
    # bounded whatever the sizes
    rng = random.Random(3)
    for _ in range(200):
        batch, new = rng.randint(1, 64), rng.randint(1, 600)
        group, hkv = rng.randint(1, 16), rng.randint(1, 16)
        sizes = [size(batch, new, group * hkv, hkv, n, 128) for n in (64, 300, 1000, 5000, 1 << 17, 1 << 22)]
        assert max(sizes) <= 1536 * min(192, new * group) * 130 * 4 + 8 * batch


@pytest.mark.parametrize("bad,rc,text", [
    (dict(hidden=100), _lib.FI_ERR_UNSUPPORTED, b"multiple of 8"),
    (dict(hidden=0), _lib.FI_ERR_UNSUPPORTED, b"multiple of 8"),
    (dict(hidden=(1 << 24) + 8), _lib.FI_ERR_UNSUPPORTED, b"multiple of 8"),
    (dict(M=-1), _lib.FI_ERR_UNSUPPORTED, b"-1 rows"),
    (dict(M=1 << 24), _lib.FI_ERR_UNSUPPORTED, b"too many rows"),
    (dict(M=2, x=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(M=2, r=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(M=2, w=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(M=2, h=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(M=2, o=None), _lib.FI_ERR_INVALID, b"null"),
    (dict(M=2, x=A + 2), _lib.FI_ERR_INVALID, b"aligned"),
    (dict(M=2, w=A + 8), _lib.FI_ERR_INVALID, b"aligned"),
    (dict(M=2, rs=260), _lib.FI_ERR_INVALID, b"aligned"),
    (dict(M=2, h=A, o=A), _lib.FI_ERR_INVALID, b"overlap"),
    (dict(M=2, os=128), _lib.FI_ERR_INVALID, b"overlap"),
    (dict(M=2, hs=0), _lib.FI_ERR_INVALID, b"overlap"),
])
def test_norm_refusals(lib, bad, rc, text):
    assert lib.fi_add_rmsnorm(*_norm(**bad)) == rc
    assert text in lib.fi_last_error()
    assert lib.fi_add_rmsnorm(*_norm()) == _lib.FI_OK


@pytest.mark.parametrize("name,args,sizes", [
    ("fi_paged_chunk_attention_fwd", _chunk(), (6, 7, 8, 11, 14, 19, 20, 21, 22)),
    ("fi_add_rmsnorm", _norm(), (4, 5)),
])
def test_native_calls_agree_with_the_library(lib, name, args, sizes):
    calls = _lib.calls()
    native, reference = getattr(calls, name), getattr(lib, name)
    assert native is not reference, "the call module is not built"
    assert len(args) == len(_lib.SIGNATURES[name][1])
    assert native(*args) == reference(*args) == _lib.FI_OK
    for i in sizes:
        bad = list(args)
        bad[i] = -3 - i
        assert native(*bad) == reference(*bad)
        native(*bad)
        said = lib.fi_last_error()
        reference(*bad)
        assert said == lib.fi_last_error(), i
    with pytest.raises(TypeError, match="arguments"):
        native(*args[:-1])
    assert set(_lib.FAST_CHUNK) == {"fi_paged_chunk_attention_fwd", "fi_add_rmsnorm"}


def test_native_call_hands_on_both_floats(lib):
    bad = _chunk(cap=-2.5, scale=0.75)
    assert _lib.calls().fi_paged_chunk_attention_fwd(*bad) == _lib.FI_ERR_INVALID
    assert b"sm_scale 0.75 and softcap -2.5" in lib.fi_last_error()


def _cpu(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def test_wrappers_reject_cpu_and_dtype():
    q, pool = _cpu(1, 2, 3, 128), _cpu(4, 64, 1, 128)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP device"):
        fi.paged_chunk_attention(q, pool, pool, table, 64, 100)
    with pytest.raises(TypeError, match="float16"):
        fi.paged_chunk_attention(q.float(), pool, pool, table, 64, 100)
    x, w = _cpu(2, 256), _cpu(256)
    with pytest.raises(RuntimeError, match="HIP device"):
        fi.add_rms_norm(x, x, w)
    assert fi.paged_chunk_attention_workspace(1, 4, 24, 8, 64, 128, "cpu") is None
    assert fi.paged_chunk_attention_workspace(1, 4, 24, 8, 4096, 128, "cpu").numel() > 0


def test_m0_is_only_set_by_the_copy_helper(tmp_path):
    """As for the other kernels that copy to LDS through inline asm: every M0 write is the
    helper's, followed by one idle slot and its copy, and nothing else names M0."""
    lines = [ln.split(";")[0].strip() for ln in _device_asm("paged_chunk.hip", tmp_path).splitlines()]
    lines = [ln for ln in lines if ln and not ln.startswith((".", "#"))]
    copies = 0
    for i, ln in enumerate(lines):
        if re.search(r"\bm0\b", ln):
            assert re.fullmatch(r"s_mov_b32 m0, s\d+", ln), ln
            assert lines[i + 1] == "s_nop 0" and lines[i + 2].startswith("global_load_lds_dword"), ln
            copies += 1
    assert copies == sum(ln.startswith("global_load_lds") for ln in lines) > 0


def test_oracle_of_whole_prompts():
    """The 64-bit form equals plain causal attention for a whole prompt, and single tokens of it."""
    g = torch.Generator().manual_seed(5)
    bs, n, hq, hkv, d = 8, 37, 6, 2, 16
    kc, vc = (torch.randn(9, bs, hkv, d, generator=g).half() for _ in range(2))
    table = torch.randperm(9, generator=g)[:5].int().view(1, 5)
    q = torch.randn(1, n, hq, d, generator=g).half()
    o, bound = OC.chunk_attention(q, kc, vc, table, bs, [n])
    k = kc[table[0].long()].flatten(0, 1)[:n].double().repeat_interleave(3, 1).transpose(0, 1)
    v = vc[table[0].long()].flatten(0, 1)[:n].double().repeat_interleave(3, 1).transpose(0, 1)
    s = q[0].double().transpose(0, 1) @ k.transpose(1, 2) * d ** -0.5
    s.masked_fill_(torch.ones(n, n).triu(1).bool(), -math.inf)
    ref = (torch.softmax(s, -1) @ v).transpose(0, 1)
    assert (o[0] - ref).abs().max() < 1e-12 and bound.max() < 0.02
    one, _ = OC.chunk_attention(q[:, 20:21], kc, vc, table, bs, [21])
    assert (one[0, 0] - ref[20]).abs().max() < 1e-12
