"""Calls of causal self-attention that have no right answer, on the CPU: each is refused, and says why, before anything looks
for a device; and the C-ABI's own refusals."""
import os
import subprocess

import pytest
import torch
from torch.autograd import forward_ad

from lingbot_world_v2_realtime_amd import KV4Cache, Rotary, _lib, kernels, norm_rotary_embed, packed_attention
from test_abi import E_ALIGN, E_DEVICE, E_NULL, E_SHAPE, FAKE, declared_functions

HEADER = os.path.join(os.path.dirname(__file__), "..", "include", "lbw_causal.h")
BF16, I32 = torch.bfloat16, torch.int32


def test_header_declarations_are_bound_and_exported(lib):
    decl = declared_functions(HEADER)
    assert set(decl) == set(_lib.CAUSAL_SIGNATURES)
    for name, n in decl.items():
        assert len(_lib.CAUSAL_SIGNATURES[name][1]) == n and hasattr(lib, name), name
    nm = subprocess.run(["nm", "-D", "--defined-only", _lib.LIB_PATH], capture_output=True, text=True).stdout
    assert set(decl) <= {line.split()[-1] for line in nm.splitlines() if " T " in line}


# ---------------------------------------------------------------- norm and rotation


def _norm(**kw):
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=BF16), k=torch.zeros(2, 3, 2, 64, dtype=BF16), positions=0, rope=Rotary.build(64, "cpu"),
             q_weight=torch.ones(64, dtype=BF16), k_weight=torch.ones(64, dtype=BF16))
    return lambda: norm_rotary_embed(**{**a, **kw})


@pytest.mark.parametrize("kw,error,said", [
    (dict(), ValueError, "device tensor"),
    (dict(k=None), ValueError, "k_weight without k"),
    (dict(q_weight=torch.ones(64, dtype=torch.float16), k_weight=None), TypeError, "q_weight must be"),
    (dict(q_weight=torch.ones(64)), TypeError, "one dtype"),
    (dict(q_weight=torch.ones(32, dtype=BF16)), ValueError, r"q_weight must be contiguous \(64,\)"),
    (dict(k_weight=torch.ones(64, 1, dtype=BF16)), ValueError, "k_weight must be contiguous"),
    (dict(q_weight=torch.ones(128, dtype=BF16)[::2]), ValueError, "contiguous"),
    (dict(q_weight=1.0), TypeError, "must be a tensor"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    (dict(eps=torch.tensor(1.0)), TypeError, "eps"),
    (dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.float64)), TypeError, "bfloat16, float16 or float32"),
    (dict(q=torch.zeros(3, 4, 64, dtype=BF16)), ValueError, "4-d"),
    (dict(k=torch.zeros(2, 4, 2, 64, dtype=BF16)), ValueError, "do not match"),
    (dict(k=torch.zeros(2, 3, 2, 64)), TypeError, "one dtype"),
    (dict(rope=Rotary.build(66, "cpu")), ValueError, "do not fit"),
    (dict(tensor_layout="BHD"), ValueError, "tensor_layout"),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), ValueError, "positions"),
    (dict(q=torch.zeros(2, 3, 64, 4, dtype=BF16).transpose(2, 3)), ValueError, "contiguous channels"),
])
def test_norm_rotary_refusals(kw, error, said):
    with pytest.raises(error, match=said):
        _norm(**kw)()


def test_norm_rotary_refuses_what_loses_a_derivative():
    rope = Rotary.build(64, "cpu")
    rope.freq.requires_grad_()
    with pytest.raises(ValueError, match="freq has no gradient"):
        _norm(rope=rope)()
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(2, 3, 4, 64, dtype=BF16), torch.ones(2, 3, 4, 64, dtype=BF16))
        with pytest.raises(Exception):
            _norm(q=x)()
    with pytest.raises(ValueError, match="negated"):
        _norm(q=torch._neg_view(torch.zeros(2, 3, 4, 64, dtype=BF16)))()


# ---------------------------------------------------------------- packed attention


def _starts(*x):
    return torch.tensor(x, dtype=I32)


def _attn(**kw):
    a = dict(q=torch.zeros(9, 4, 64, dtype=BF16), k=torch.zeros(9, 2, 64, dtype=BF16), v=torch.zeros(9, 2, 64, dtype=BF16),
             starts=_starts(0, 4, 9))
    return lambda: packed_attention(**{**a, **kw})


@pytest.mark.parametrize("kw,error,said", [
    (dict(), ValueError, "device tensor"),
    (dict(q=torch.zeros(9, 4, 64)), TypeError, "bfloat16 or float16"),
    (dict(q=torch.zeros(9, 4, 64, dtype=torch.float16)), TypeError, "one dtype"),
    (dict(q=torch.zeros(1, 9, 4, 64, dtype=BF16)), ValueError, "rows, heads, channels"),
    (dict(q=torch.zeros(9, 4, 96, dtype=BF16)), ValueError, "64 or 128"),
    (dict(q=torch.zeros(9, 4, 128, dtype=BF16)), ValueError, "do not match"),
    (dict(q=torch.zeros(9, 3, 64, dtype=BF16)), ValueError, "evenly"),
    (dict(q=torch.zeros(9, 0, 64, dtype=BF16)), ValueError, "heads"),
    (dict(v=torch.zeros(8, 2, 64, dtype=BF16)), ValueError, "do not match"),
    (dict(q=torch.zeros(7, 4, 64, dtype=BF16)), ValueError, "give k_starts"),
    (dict(starts=torch.tensor([0, 4, 9])), TypeError, "int32"),
    (dict(starts=[0, 4, 9]), TypeError, "must be a tensor"),
    (dict(starts=_starts(0)), ValueError, "starts must be contiguous"),
    (dict(starts=_starts(0, 1, 4, 5, 9)[::2]), ValueError, "starts must be contiguous"),
    (dict(k_starts=_starts(0, 9)), ValueError, "k_starts"),
    (dict(sm_scale=0.0), ValueError, "sm_scale"),
    (dict(sm_scale=float("inf")), ValueError, "sm_scale"),
    (dict(sm_scale=1e-60), ValueError, "sm_scale"),
    (dict(sm_scale=torch.tensor(0.1)), TypeError, "sm_scale"),
    (dict(v=torch._neg_view(torch.zeros(9, 2, 64, dtype=BF16))), ValueError, "negated"),
    (dict(k=None), TypeError, "must be a tensor"),
])
def test_packed_attention_refusals(kw, error, said):
    with pytest.raises(error, match=said):
        _attn(**kw)()
    with pytest.raises(error, match=said):   # the same where a gradient would be recorded
        kw = {n: x.clone().requires_grad_() if n in "qkv" and isinstance(x, torch.Tensor) and not x.is_neg() else x for n, x in kw.items()}
        _attn(**kw)()


# ---------------------------------------------------------------- the cache


CACHE = KV4Cache.empty(2, 3, 2, 64, "cpu")


def _cache(method, cache=None, **kw):
    rows = torch.zeros(2, 2, 64, dtype=BF16)
    a = dict(layer=1, table=torch.zeros(2, 4, dtype=I32), lens=_starts(5, 200), starts=None)
    a.update({"write": dict(k=rows, v=rows), "read": {}, "attend": dict(q=torch.zeros(2, 4, 64, dtype=BF16))}[method])
    return lambda: getattr(cache or CACHE, method)(**{**a, **kw})


def _with(**kw):
    import dataclasses
    return dataclasses.replace(CACHE, **kw)


@pytest.mark.parametrize("method", ["write", "read", "attend"])
@pytest.mark.parametrize("kw,error,said", [
    (dict(), ValueError, "on a device"),
    (dict(layer=2), ValueError, "layer 2"),
    (dict(layer=-1), ValueError, "layer -1"),
    (dict(layer=0.0), TypeError, "layer"),
    (dict(table=torch.zeros(2, 4, dtype=torch.int64)), TypeError, "table must be int32"),
    (dict(table=torch.zeros(3, 4, dtype=I32)), ValueError, "table must be"),
    (dict(table=torch.zeros(2, 0, dtype=I32)), ValueError, "table must be"),
    (dict(table=torch.zeros(4, 2, dtype=I32).t()), ValueError, "table must be"),
    (dict(lens=torch.zeros(2)), TypeError, "lens must be int32"),
    (dict(lens=torch.zeros(4, dtype=I32)[::2]), ValueError, "lens must be"),
    (dict(starts=_starts(0, 2)), ValueError, "starts"),
    (dict(starts=torch.zeros(3)), TypeError, "starts must be int32"),
    (dict(cache=_with(k=CACHE.k[0])), ValueError, "cache's k must be"),
    (dict(cache=_with(k_scale=CACHE.k_scale[:1])), ValueError, "cache's k_scale must be"),
    (dict(cache=_with(v=CACHE.v.float())), TypeError, "cache's v must be uint8"),
    (dict(cache=_with(v_scale=CACHE.v_scale.transpose(0, 1))), ValueError, "cache's v_scale must be"),
])
def test_cache_refusals(method, kw, error, said):
    with pytest.raises(error, match=said):
        _cache(method, **kw)()


@pytest.mark.parametrize("method,kw,error,said", [
    ("write", dict(k=torch.zeros(2, 2, 64)), TypeError, "bfloat16 or float16"),
    ("write", dict(k=torch.zeros(2, 3, 64, dtype=BF16), v=torch.zeros(2, 3, 64, dtype=BF16)), ValueError, "must be"),
    ("write", dict(k=torch.zeros(2, 2, 128, dtype=BF16), v=torch.zeros(2, 2, 128, dtype=BF16)), ValueError, "cache's 64"),
    ("write", dict(v=torch.zeros(2, 2, 64, dtype=torch.float16)), TypeError, "one dtype"),
    ("write", dict(k=torch.zeros(3, 2, 64, dtype=BF16), v=torch.zeros(3, 2, 64, dtype=BF16)), ValueError, "give starts"),
    ("write", dict(k=torch.zeros(2, 2, 64, dtype=BF16, requires_grad=True)), RuntimeError, "gradient"),
    ("attend", dict(q=torch.zeros(2, 3, 64, dtype=BF16)), ValueError, "evenly"),
    ("attend", dict(q=torch.zeros(2, 4, 128, dtype=BF16)), ValueError, "cache's 64"),
    ("attend", dict(q=torch.zeros(3, 4, 64, dtype=BF16)), ValueError, "give starts"),
    ("attend", dict(q=torch.zeros(2, 4, 64, dtype=BF16, requires_grad=True)), RuntimeError, "gradient"),
    ("attend", dict(sm_scale=-1.0), ValueError, "sm_scale"),
    ("read", dict(starts=_starts(0, 1, 2)), ValueError, "how many tokens"),
    ("read", dict(tokens=5), ValueError, "give starts"),
    ("read", dict(tokens=-1, starts=_starts(0, 1, 2)), ValueError, "tokens"),
])
def test_cache_refusals_of_each_call(method, kw, error, said):
    with pytest.raises(error, match=said):
        _cache(method, **kw)()


def test_cache_sizes():
    for bad in (dict(head_dim=96), dict(layers=0), dict(pages=0), dict(heads=-1)):
        with pytest.raises(ValueError):
            KV4Cache.empty(**{**dict(layers=1, pages=1, heads=1, device="cpu"), **bad})
    c = KV4Cache.empty(3, 5, 2, 128, "cpu")
    bytes_ = sum(x.numel() for x in (c.k, c.k_scale, c.v, c.v_scale))
    assert bytes_ * 8 == 4.25 * 3 * 5 * 64 * 2 * 128 * 2


# ---------------------------------------------------------------- the C-ABI


def _call(lib, name, **kw):
    base = {
        "lbw_norm_rotary": dict(q=FAKE, k=FAKE, dtype=0, vec=0, batch=1, len=4, qh=2, kh=1, dim=64, pairs=32, s=(512, 128, 64, 256, 64, 64),
                                qw=FAKE, kw=FAKE, eps=1e-6, pos=FAKE, i64=1, p=(4, 1, 0), start=0, freq=FAKE, axis=None, axes=1, inter=1,
                                factor=1.0, qo=FAKE, ko=FAKE, o=(512, 128, 64, 256, 64, 64), stream=None),
        "lbw_packed_attn_fwd": dict(q=FAKE, k=FAKE, v=FAKE, dtype=0, seqs=2, qr=9, kr=9, qh=4, kh=2, dim=64, s=(256, 64, 128, 64, 128, 64),
                                    st=FAKE, ks=FAKE, causal=1, scale=0.1, out=FAKE, rest=None, lse=None, stream=None),
        "lbw_packed_attn_bwd": dict(do=FAKE, out=FAKE, rest=FAKE, lse=FAKE, q=FAKE, k=FAKE, v=FAKE, dtype=0, seqs=2, qr=9, kr=9, qh=4, kh=2,
                                    dim=64, s=(256, 64, 256, 64, 128, 64, 128, 64), st=FAKE, ks=FAKE, causal=1, scale=0.1, dq=FAKE, dk=FAKE,
                                    dv=FAKE, ws=FAKE, stream=None),
        "lbw_kv4_write": dict(k=FAKE, v=FAKE, dtype=0, seqs=2, rows=2, heads=2, dim=64, s=(128, 64, 128, 64), st=None, lens=FAKE, table=FAKE,
                              t=4, width=4, pages=3, k4=FAKE, ks=FAKE, v4=FAKE, vs=FAKE, stream=None),
        "lbw_kv4_read": dict(seqs=2, rows=2, heads=2, dim=64, st=None, lens=FAKE, table=FAKE, t=4, width=4, pages=3, k4=FAKE, ks=FAKE, v4=FAKE,
                             vs=FAKE, k=FAKE, v=FAKE, stream=None),
        "lbw_kv4_attn": dict(q=FAKE, dtype=0, seqs=2, rows=2, qh=4, heads=2, dim=64, s=(256, 64), st=None, lens=FAKE, table=FAKE, t=4, width=4,
                             pages=3, k4=FAKE, ks=FAKE, v4=FAKE, vs=FAKE, scale=0.1, out=FAKE, ws=FAKE, stream=None),
    }[name]
    args = []
    for v in {**base, **kw}.values():
        args += v if isinstance(v, tuple) else [v]
    return getattr(lib, name)(*args)


@pytest.mark.parametrize("name,kw,status", [
    ("lbw_norm_rotary", dict(q=None), E_NULL), ("lbw_norm_rotary", dict(ko=None), E_NULL), ("lbw_norm_rotary", dict(dim=513), E_SHAPE),
    ("lbw_norm_rotary", dict(pairs=33), E_SHAPE), ("lbw_norm_rotary", dict(vec=1), E_SHAPE), ("lbw_norm_rotary", dict(eps=-1.0), E_SHAPE),
    ("lbw_norm_rotary", dict(q=FAKE + 1), E_ALIGN), ("lbw_norm_rotary", dict(qw=FAKE + 1), E_ALIGN), ("lbw_norm_rotary", dict(), E_DEVICE),
    ("lbw_packed_attn_fwd", dict(q=None), E_NULL), ("lbw_packed_attn_fwd", dict(st=None), E_NULL), ("lbw_packed_attn_fwd", dict(dtype=2), E_SHAPE),
    ("lbw_packed_attn_fwd", dict(dim=96), E_SHAPE), ("lbw_packed_attn_fwd", dict(qh=3), E_SHAPE), ("lbw_packed_attn_fwd", dict(scale=0.0), E_SHAPE),
    ("lbw_packed_attn_fwd", dict(seqs=0), E_SHAPE), ("lbw_packed_attn_fwd", dict(s=(256, 64, 0, 64, 128, 64)), E_ALIGN),
    ("lbw_packed_attn_fwd", dict(s=(256, 64, 128, 60, 128, 64)), E_ALIGN), ("lbw_packed_attn_fwd", dict(s=(256, 64, 1 << 24, 64, 128, 64)), E_ALIGN),
    ("lbw_packed_attn_fwd", dict(k=FAKE + 8), E_ALIGN), ("lbw_packed_attn_fwd", dict(rest=FAKE + 8), E_ALIGN), ("lbw_packed_attn_fwd", dict(), E_DEVICE),
    ("lbw_packed_attn_bwd", dict(ws=None), E_NULL), ("lbw_packed_attn_bwd", dict(dv=None), E_NULL), ("lbw_packed_attn_bwd", dict(kr=0), E_SHAPE),
    ("lbw_packed_attn_bwd", dict(lse=FAKE + 2), E_ALIGN), ("lbw_packed_attn_bwd", dict(ws=FAKE + 4), E_ALIGN), ("lbw_packed_attn_bwd", dict(), E_DEVICE),
    ("lbw_packed_attn_bwd", dict(dk=None, dv=None), E_DEVICE),
    ("lbw_kv4_write", dict(lens=None), E_NULL), ("lbw_kv4_write", dict(rows=3), E_SHAPE), ("lbw_kv4_write", dict(dtype=2), E_SHAPE),
    ("lbw_kv4_write", dict(pages=0), E_SHAPE), ("lbw_kv4_write", dict(s=(128, 63, 128, 64)), E_ALIGN), ("lbw_kv4_write", dict(v4=FAKE + 8), E_ALIGN),
    ("lbw_kv4_write", dict(), E_DEVICE), ("lbw_kv4_read", dict(k=None), E_NULL), ("lbw_kv4_read", dict(width=0), E_SHAPE),
    ("lbw_kv4_read", dict(), E_DEVICE), ("lbw_kv4_attn", dict(out=None), E_NULL), ("lbw_kv4_attn", dict(qh=3), E_SHAPE),
    ("lbw_kv4_attn", dict(ws=None, width=40000), E_NULL), ("lbw_kv4_attn", dict(scale=-0.1), E_SHAPE), ("lbw_kv4_attn", dict(), E_DEVICE),
])
def test_c_abi_statuses(lib, name, kw, status):
    if status == E_DEVICE and torch.cuda.is_available():
        pytest.skip("the call would go on")
    assert _call(lib, name, **kw) == status


def test_workspaces_hold_every_part(lib):
    for seqs, rows, qh, h, width, single in ((1, 1, 12, 4, 24, 1), (61, 61, 32, 8, 95, 1), (7, 35, 12, 12, 377, 0), (64, 64, 96, 12, 1, 1), (1, 16, 8, 1, 400, 0)):
        n = lib.lbw_kv4_attn_workspace_bytes(seqs, rows, qh, h, 128, width, single)
        # a part of each row and head at least, of 128 sums and two statistics; none where a sequence is one unit of keys
        assert n % 8 == 0 and (n == 0 if width == 1 else n >= rows * qh * 130 * 4)
    assert lib.lbw_packed_attn_bwd_workspace_bytes(100, 200, 4, 2) >= 100 * 4 * 4
    assert lib.lbw_norm_rotary_bwd_workspace_bytes(128) > 0
    assert kernels.block_binding() is not None
